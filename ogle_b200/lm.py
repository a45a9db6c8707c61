"""The operators of a language model's decoding step (include/ogle_cuda.h): keys and values appended to a paged cache held
in 8 bits, attention over that cache or over pages of it that a score chooses, the adjustment of logits before a token is chosen, the step of
a beam search and the pages' management behind it. One function per entry point, on torch CUDA tensors; torch is used for device
memory and the current stream only.

The cache is four tensors (k, v, k_scale, v_scale): k and v float8_e4m3fn [pages, kv heads, page tokens, head dim] (any strides
that keep a token's elements side by side and 16-byte boundaries), one float32 scale for each page and kv head, a power of two, or 0
where append has met nothing but zeros in the page. `new_cache` makes one; a page may be anywhere in it. Sequence b's token j lies in
page block_table[b, j // page tokens].

Rows are the new tokens of all sequences, one sequence behind the other: sequence b has rows row_start[b]..row_start[b + 1], the
last of the kv_len[b] tokens that it has once they are appended. Without row_start every sequence has one row. max_kv_len and
max_rows are the host's bounds of what kv_len and row_start hold on the device: nothing here waits for the device. Rows of a sequence
behind its first max_rows, rows that no sequence has (a padded batch), and tokens from max_kv_len on are ignored: a result made here
holds what was in memory there.

Pages are managed on the device: refs, int32 [pages], counts the table entries that name each page, 0 where it is free. advance_pages makes
the block table of the texts that go on from another one (forked, grown, cut, ended, new), copy_pages copies what two of them would
write to, compact_pages moves used pages to the front. None of them changes its inputs but the caches.

Attention over few pages: page_bounds keeps bounds of every page's keys (new_bounds), choose_pages picks for each row and kv head the pages
whose keys can have the largest products with its queries, sparse_attention attends those.
"""
import torch

from . import _lib
from ._lib import check
from .ops import _stream

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_PAGED_BATCH, _APPEND = _lib.packer(_lib.PagedBatch).pack, _lib.packer(_lib.AppendParams).pack
_ATTENTION, _LOGITS = _lib.packer(_lib.AttentionParams).pack, _lib.packer(_lib.LogitsParams).pack
_BEAM, _ADVANCE = _lib.packer(_lib.BeamParams).pack, _lib.packer(_lib.AdvanceParams).pack
_COMPACT, _COPY_PAGES = _lib.packer(_lib.CompactParams).pack, _lib.packer(_lib.CopyPagesParams).pack
_CHOOSE, _CHOSEN = _lib.packer(_lib.ChooseParams).pack, _lib.packer(_lib.ChosenPages).pack
_PAGE_TENSORS = _lib.packer(_lib.PageTensors).pack
_I32, _F32, _E4M3 = torch.int32, torch.float32, torch.float8_e4m3fn


def new_cache(pages, kv_heads, page_tokens, head_dim, device="cuda"):
    """Empty cache of so many pages: (k, v, k_scale, v_scale)."""
    k, v = (torch.zeros(pages, kv_heads, page_tokens, head_dim, dtype=_E4M3, device=device) for _ in range(2))
    k_scale, v_scale = (torch.ones(pages, kv_heads, dtype=_F32, device=device) for _ in range(2))
    return k, v, k_scale, v_scale


def rotary_table(positions, rotary_dim, base=10000.0, device="cuda"):
    """float32 [positions, rotary_dim]: the cosines of position * base^(-2 i / rotary_dim), then the sines."""
    half = rotary_dim // 2
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([angle.cos(), angle.sin()], 1).to(_F32).to(device)


def _vector(t, dtype, n, name, here=None):
    """Address of a contiguous vector of n values (any number, n None), on device `here` (any, None)."""
    if t is None:
        return 0
    if t.dtype != dtype or (not t.is_cuda if here is None else t.get_device() != here) or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name}: expected a contiguous {dtype} CUDA tensor" + (f" of {n} values" if n is not None else "") + (f" on device {here}" if here is not None else ""))
    return t.data_ptr()


def _rows(t, dtype, rows, heads, dim, name, here=None):
    """(address, row stride, head stride) of activations [rows, heads, dim]."""
    if t.dtype != dtype or (not t.is_cuda if here is None else t.get_device() != here) or t.dim() != 3:
        raise ValueError(f"{name}: expected a {dtype} CUDA tensor [rows, heads, head dim]" + (f" on device {here}" if here is not None else ""))
    shape, stride = t.shape, t.stride()
    if shape[0] != rows or shape[2] != dim or (heads is not None and shape[1] != heads) or (stride[2] != 1 and dim > 1):
        raise ValueError(f"{name}: expected [{rows}, {heads if heads is not None else 'heads'}, {dim}] with the elements of a head side by side, "
                         f"got {tuple(shape)} with strides {stride}")
    return t.data_ptr(), stride[0], stride[1]


def _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, q_heads, dtype, here=None):
    k, v, k_scale, v_scale = cache
    shape, stride = k.shape, k.stride()
    if k.dtype != _E4M3 or v.dtype != _E4M3 or not k.is_cuda or not v.is_cuda or len(shape) != 4 or shape != v.shape:
        raise ValueError("cache: expected float8_e4m3fn CUDA tensors [pages, kv heads, page tokens, head dim] for keys and values")
    pages, kv_heads, page_tokens, dim = shape
    if stride != v.stride() or stride[3] != 1:
        raise ValueError("cache: keys and values need the same strides, the elements of a token side by side")
    if dtype not in _DTYPE:
        raise ValueError(f"activations are float32, float16 or bfloat16, not {dtype}")
    if here is not None and (k.get_device() != here or v.get_device() != here or block_table.get_device() != here):
        raise ValueError(f"cache and block_table: expected on device {here}")
    table_shape, table_strides = block_table.shape, block_table.stride()
    if block_table.dtype != _I32 or not block_table.is_cuda or len(table_shape) != 2 or table_strides[1] != 1 and table_shape[1] > 1:
        raise ValueError("block_table: expected an int32 CUDA tensor [sequences, blocks]")
    seqs, blocks = table_shape
    table_stride = table_strides[0] if seqs > 1 else blocks
    if table_stride < blocks or max_kv_len > blocks * page_tokens:
        raise ValueError(f"block_table: {blocks} blocks of {page_tokens} tokens are fewer than max_kv_len = {max_kv_len}")
    if row_start is None and rows != seqs:
        raise ValueError(f"{rows} rows for {seqs} sequences need row_start")
    return _PAGED_BATCH(seqs, rows, 1 if row_start is None else max_rows, max_kv_len, q_heads, kv_heads, dim, page_tokens, pages,
                        table_stride, _DTYPE[dtype], 0, stride[0], stride[1], stride[2],
                        _vector(row_start, _I32, seqs + 1, "row_start", here), _vector(kv_len, _I32, seqs, "kv_len", here), block_table.data_ptr(),
                        k.data_ptr(), v.data_ptr(), _vector(k_scale, _F32, pages * kv_heads, "k_scale", here),
                        _vector(v_scale, _F32, pages * kv_heads, "v_scale", here))


def append(k, v, cache, block_table, kv_len, max_kv_len, row_start=None, max_rows=1, q=None, rotary=None, interleaved=False, out=None):
    """Stores the rows' keys and values k, v [rows, kv heads, head dim] in the cache, quantised to e4m3 with a power-of-two
    scale for each page and head (ogle_cuda_kv_append). rotary [positions, rotary dim] (see rotary_table; None: no rotation)
    rotates k and q by the rows' positions on the way, in pairs half the rotary dim apart or, interleaved, of neighbours.
    Returns the rotated q (into `out`, which may be q itself; 0 for rows that stand before the text), or None without q."""
    rows, dtype = k.shape[0], k.dtype
    heads, dim = cache[0].shape[1], cache[0].shape[3]
    q_heads = heads if q is None else q.shape[1]
    b = _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, q_heads, dtype)
    pk, pv = _rows(k, dtype, rows, heads, dim, "k"), _rows(v, dtype, rows, heads, dim, "v")
    pq = po = (0, 0, 0)
    if q is not None:
        pq = _rows(q, dtype, rows, None, dim, "q")
        if out is None:
            out = q.new_empty(rows, q_heads, dim)
            po = out.data_ptr(), q_heads * dim, dim
        else:
            po = _rows(out, dtype, rows, q_heads, dim, "out")
    table = n = d = 0
    if rotary is not None:
        if rotary.dim() != 2:
            raise ValueError("rotary: expected [positions, rotary dim]")
        n, d = rotary.shape
        table = _vector(rotary, _F32, None, "rotary")
    p = _APPEND(pk[0], pv[0], pq[0], po[0], pk[1], pk[2], pv[1], pv[2], pq[1], pq[2], po[1], po[2], table, d, n, bool(interleaved), 0)
    check(_lib.cuda_lib().ogle_cuda_kv_append(b, p, _stream()), "kv_append")
    return out if q is not None else None


def attention(q, cache, block_table, kv_len, max_kv_len, row_start=None, max_rows=1, scale=None, causal=True, window=0, out=None):
    """Softmax attention of q [rows, heads, head dim] over the cached keys and values (ogle_cuda_paged_attention): of each row
    over the tokens up to its own (causal; else all of its sequence), with a window over the last `window` of them. scale: of the
    products, 1 / sqrt(head dim) where None. Returns (out, lse): lse float32 [rows, heads], the logarithm of the sum of
    exponentials; a row without a token has out 0 and lse -inf."""
    dtype = q.dtype
    if q.dim() != 3:
        raise ValueError("q: expected [rows, heads, head dim]")
    rows, heads, dim = q.shape
    b = _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, heads, dtype)
    pq = _rows(q, dtype, rows, heads, cache[0].shape[3], "q")
    if out is None:
        out = q.new_empty(rows, heads, dim)
        po = out.data_ptr(), heads * dim, dim
    else:
        po = _rows(out, dtype, rows, heads, dim, "out")
    lse = q.new_empty(rows, heads, dtype=_F32)
    p = _ATTENTION(pq[0], po[0], lse.data_ptr(), pq[1], pq[2], po[1], po[2], dim ** -0.5 if scale is None else scale, bool(causal), window, 0)
    lib = _lib.cuda_lib()
    # a workspace of this call's own: its memory goes back to the stream that the call runs on. Where the call only asks for a nominal
    # one, which it does not touch, the results' address stands for it (an allocation is 1.6 us of a call that takes 15).
    n = lib.ogle_cuda_paged_attention_workspace_bytes(b, p)
    if n > _lib.ATTENTION_NO_WORKSPACE:
        workspace = q.new_empty(n, dtype=torch.uint8)
        check(lib.ogle_cuda_paged_attention(b, p, workspace.data_ptr(), n, _stream()), "paged_attention")
    else:
        check(lib.ogle_cuda_paged_attention(b, p, po[0], n, _stream()), "paged_attention")
    return out, lse


def adjust_logits(logits, tokens=None, token_start=None, prompt_len=None, repetition=None, presence=None, frequency=None,
                  bias_token=None, bias_value=None, bias_start=None, allowed=None, out_dtype=None, out=None):
    """Logits [rows, vocab] with the repeated-token penalties, biases and grammar mask of each row applied
    (ogle_cuda_adjust_logits). tokens (int32) token_start[r]..token_start[r + 1] are row r's text so far, the first prompt_len[r] of
    them its prompt; repetition (of every token of the text), presence and frequency (of those behind the prompt) are float32
    [rows]; biases are given as lists like the tokens, the last one of a token counting; allowed int32 [rows, words]: bit t % 32 of word
    t // 32 is 0 where token t must not follow (or [words] for all rows). out_dtype: the logits' own, or float32. `out` may be logits."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DTYPE or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits: expected a CUDA tensor [rows, vocab] in float32, float16 or bfloat16, a row's elements side by side")
    rows, vocab = logits.shape
    if out is None:
        out = logits.new_empty(rows, vocab, dtype=out_dtype or logits.dtype)
    elif out.shape != logits.shape or not out.is_cuda or out.dtype != (out_dtype or out.dtype) or out.stride(1) != 1 and vocab > 1:
        raise ValueError("out: expected a CUDA tensor of the logits' shape")
    if out.dtype != logits.dtype and out.dtype != _F32:
        raise ValueError("out: the logits' type or float32")
    if (tokens is None) != (token_start is None):
        raise ValueError("tokens and token_start go together")
    if not (bias_token is None) == (bias_value is None) == (bias_start is None):
        raise ValueError("bias_token, bias_value and bias_start go together")
    n_tokens = tokens.numel() if tokens is not None else 0
    n_biases = bias_token.numel() if bias_token is not None else 0
    mask_stride = 0
    if allowed is not None:
        if allowed.dtype != _I32 or not allowed.is_cuda or allowed.shape[-1] < (vocab + 31) // 32 or allowed.stride(-1) != 1 and vocab > 32 or \
                allowed.dim() not in (1, 2) or allowed.dim() == 2 and allowed.shape[0] != rows:
            raise ValueError("allowed: expected an int32 CUDA tensor [rows, ceil(vocab / 32)] or [ceil(vocab / 32)]")
        mask_stride = allowed.stride(0) if allowed.dim() == 2 else 0
    p = _LOGITS(rows, vocab, _DTYPE[logits.dtype], _DTYPE[out.dtype], n_tokens, n_biases, logits.stride(0) if rows > 1 else vocab,
                out.stride(0) if rows > 1 else vocab, mask_stride, logits.data_ptr(), out.data_ptr(),
                _vector(tokens, _I32, None, "tokens"), _vector(token_start, _I32, rows + 1, "token_start"),
                _vector(prompt_len, _I32, rows, "prompt_len"), _vector(repetition, _F32, rows, "repetition"),
                _vector(presence, _F32, rows, "presence"), _vector(frequency, _F32, rows, "frequency"),
                _vector(bias_token, _I32, None, "bias_token"), _vector(bias_value, _F32, n_biases, "bias_value"),
                _vector(bias_start, _I32, rows + 1, "bias_start"), allowed.data_ptr() if allowed is not None else 0)
    check(_lib.cuda_lib().ogle_cuda_adjust_logits(p, _stream()), "adjust_logits")
    return out


def _device(t, name):
    """Number of the device that a call's first tensor lies on: the others have to, too."""
    here = t.get_device()
    if here < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    return here


def _here(device):
    """The current stream, which is one of the call's device: a call does not go to another."""
    if device != torch.cuda.current_device():
        raise ValueError(f"tensors of device {device}, but the current one is {torch.cuda.current_device()}")
    return torch._C._cuda_getCurrentRawStream(device)


#: A workspace of up to so many bytes lies behind a call's results, in their allocation; a larger one goes back when the call is made.
_SMALL = 1 << 16


def _results(like, ints, workspace):
    """int32 results of a call and its workspace: (tensor of the results and what is behind them, their address, the workspace's, what holds it)."""
    if workspace <= _SMALL:
        first = (ints + 3) // 4 * 4
        out = like.new_empty(first + (workspace + 3) // 4, dtype=_I32)
        at = out.data_ptr()
        return out, at, at + 4 * first, out
    out, held = like.new_empty(ints, dtype=_I32), like.new_empty(workspace, dtype=torch.uint8)
    return out, out.data_ptr(), held.data_ptr(), held


def _table(t, name, here):
    """(sequences, blocks, row stride) of a block table."""
    shape, stride = t.shape, t.stride()
    if t.dtype != _I32 or t.get_device() != here or len(shape) != 2 or stride[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: expected an int32 CUDA tensor [sequences, blocks] on device {here}")
    return shape[0], shape[1], stride[0] if shape[0] > 1 else shape[1]


def beam_step(logits, scores, beams, count, ends=None):
    """The best continuations of each group of `beams` rows of logits [groups * beams, vocab] (ogle_cuda_beam_step): by the rows' scores
    (float32 [groups * beams]: the logarithm of what each text has come to; not finite: no such text; None: 0) plus the logarithm of the
    token's probability. Returns (score, beam, token) of the `count` best, [groups, count], in falling order, equal ones by beam,
    logit and token, behind the last -inf, -1, -1; and (next_row, next_token, next_score) [groups * beams]: the first `beams` of these whose token is not
    among `ends` (int32), as advance_pages takes them - the row that each goes on from, or -1."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DTYPE or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits: expected a CUDA tensor [rows, vocab] in float32, float16 or bfloat16, a row's elements side by side")
    rows, vocab = logits.shape
    here = _device(logits, "logits")
    if beams < 1 or rows % beams != 0:
        raise ValueError(f"{rows} rows are no whole groups of {beams} beams")
    groups = rows // beams
    # one allocation for all six (a view is 1.1 us, an allocation 1.5)
    n = groups * count
    lib = _lib.cuda_lib()
    given = (groups, beams, vocab, count, _DTYPE[logits.dtype], ends.numel() if ends is not None else 0, logits.stride(0) if rows > 1 else vocab,
             logits.data_ptr(), _vector(scores, _F32, rows, "scores", here), _vector(ends, _I32, None, "ends", here))
    size = lib.ogle_cuda_beam_step_workspace_bytes(_BEAM(*given, 0, 0, 0, 0, 0, 0))
    out, at, workspace, held = _results(logits, 3 * (n + max(rows, 1)), size)
    p = _BEAM(*given, at, at + 4 * n, at + 8 * n, at + 12 * n, at + 12 * n + 4 * rows, at + 12 * n + 8 * rows)
    check(lib.ogle_cuda_beam_step(p, workspace, size, _here(here)), "beam_step")
    shape, stride, out32 = (groups, count), (count, 1), out.view(_F32)
    return (out32.as_strided(shape, stride), out.as_strided(shape, stride, n), out.as_strided(shape, stride, 2 * n),
            out.as_strided((rows,), (1,), 3 * n), out.as_strided((rows,), (1,), 3 * n + rows), out32.as_strided((rows,), (1,), 3 * n + 2 * rows))


def advance_pages(block_table, kv_len, parent, new, refs, page_tokens, blocks=None):
    """Block table of the texts that go on (ogle_cuda_advance_pages). Text i goes on from sequence parent[i] of block_table and kv_len (-1: from
    nothing) and is about to have new[i] more tokens (int32, or one number for all): it shares the parent's full pages, keeps or copies the last
    one and gets what else its tokens need. refs int32 [pages]: how many table entries name each page. Sequences that no text goes on from
    are gone. Nothing is changed in place. Returns (table [texts, blocks], kv_len with the new tokens, refs, copies int32 [texts, 3] for
    copy_pages, state): state[0] pages are free for the next call, state[1] requests found none (an entry of -1: take the old table
    again, with fewer texts). blocks: columns of the new table, as the old one where None."""
    here = _device(refs, "refs")
    seqs, old_blocks, stride = _table(block_table, "block_table", here)
    n, pages = parent.numel(), refs.numel()
    blocks = old_blocks if blocks is None else blocks
    tokens = new if isinstance(new, torch.Tensor) else None
    lib = _lib.cuda_lib()
    given = (seqs, n, old_blocks, blocks, page_tokens, pages, 0 if tokens is not None else new, 0, stride, blocks, block_table.data_ptr(),
             _vector(kv_len, _I32, seqs, "kv_len", here), _vector(parent, _I32, n, "parent", here), _vector(tokens, _I32, n, "new", here),
             _vector(refs, _I32, pages, "refs", here))
    size = lib.ogle_cuda_advance_pages_workspace_bytes(_ADVANCE(*given, 0, 0, 0, 0, 0))
    out, at, workspace, held = _results(refs, n * (blocks + 4) + pages + 2, size)      # one allocation for all five
    p = _ADVANCE(*given, at, at + 4 * n * blocks, at + 4 * n * (blocks + 4), at + 4 * n * (blocks + 1), at + 4 * (n * (blocks + 4) + pages))
    check(lib.ogle_cuda_advance_pages(p, workspace, size, _here(here)), "advance_pages")
    at = n * blocks
    return (out.as_strided((n, blocks), (blocks, 1)), out.as_strided((n,), (1,), at), out.as_strided((pages,), (1,), at + 4 * n),
            out.as_strided((n, 3), (3, 1), at + n), out.as_strided((2,), (1,), at + 4 * n + pages))


def compact_pages(block_table, refs, most, page_tokens):
    """Moves used pages to the front of the pool (ogle_cuda_compact_pages), `most` of them at most. Nothing is changed in place. Returns
    (table, refs, copies int32 [most, 3] for copy_pages, state): state[0] pages are in use, state[1] moves are left for another call."""
    here = _device(refs, "refs")
    seqs, blocks, stride = _table(block_table, "block_table", here)
    pages = refs.numel()
    lib = _lib.cuda_lib()
    given = (seqs, blocks, page_tokens, pages, most, 0, stride, blocks, block_table.data_ptr(), _vector(refs, _I32, pages, "refs", here))
    size = lib.ogle_cuda_compact_pages_workspace_bytes(_COMPACT(*given, 0, 0, 0, 0))
    out, at, workspace, held = _results(refs, seqs * blocks + pages + 3 * max(most, 0) + 2, size)
    p = _COMPACT(*given, at, at + 4 * seqs * blocks, at + 4 * (seqs * blocks + pages), at + 4 * (seqs * blocks + pages + 3 * most))
    check(lib.ogle_cuda_compact_pages(p, workspace, size, _here(here)), "compact_pages")
    at = seqs * blocks
    return (out.as_strided((seqs, blocks), (blocks, 1)), out.as_strided((pages,), (1,), at), out.as_strided((most, 3), (3, 1), at + pages),
            out.as_strided((2,), (1,), at + pages + 3 * most))


def copy_pages(caches, copies, bounds=None):
    """For each (page, new page, tokens) of copies, int32 [n, 3], the first tokens of the page's keys and values and its scales in each of
    the caches (ogle_cuda_copy_pages), in place; bounds, where there are some, go along: one pair (see new_bounds) for each cache."""
    if not caches:
        return
    k0 = caches[0][0]
    shape, stride = k0.shape, k0.stride()
    if len(shape) != 4 or stride[3] != 1:
        raise ValueError("caches: expected keys and values [pages, kv heads, page tokens, head dim], the elements of a token side by side")
    pages, heads, page_tokens, dim = shape
    here = _device(k0, "caches")
    layers = []
    for i, (k, v, k_scale, v_scale) in enumerate(caches):
        if k.dtype != _E4M3 or v.dtype != _E4M3 or k.get_device() != here or v.get_device() != here or k.shape != shape or v.shape != shape or k.stride() != stride or v.stride() != stride:
            raise ValueError(f"caches: expected float8_e4m3fn CUDA tensors of the same shape and strides for all keys and values, on device {here}")
        b = (0, 0) if bounds is None else _bounds(bounds[i], pages, heads, dim, here)
        layers.append(_PAGE_TENSORS(k.data_ptr(), v.data_ptr(), _vector(k_scale, _F32, pages * heads, "k_scale", here),
                                    _vector(v_scale, _F32, pages * heads, "v_scale", here), *b))
    if copies.dim() != 2 or copies.shape[1] != 3:
        raise ValueError("copies: expected [n, 3]")
    p = _COPY_PAGES(copies.shape[0], len(layers), heads, dim, page_tokens, pages, stride[0], stride[1], stride[2], _vector(copies, _I32, None, "copies", here))
    check(_lib.cuda_lib().ogle_cuda_copy_pages(p, b"".join(layers), _here(here)), "copy_pages")


def _bounds(bounds, pages, heads, dim, here):
    """Addresses of a cache's bounds."""
    lo_hi, scale = bounds
    if lo_hi.shape != (pages, heads, 2, dim):
        raise ValueError(f"bounds: expected int8 [{pages}, {heads}, 2, {dim}]")
    return _vector(lo_hi, torch.int8, None, "bounds", here), _vector(scale, _F32, pages * heads, "the bounds' scale", here)


def new_bounds(cache):
    """Room for the bounds of a cache's pages: (int8 [pages, kv heads, 2, head dim], float32 [pages, kv heads])."""
    pages, heads, _, dim = cache[0].shape
    return (torch.zeros(pages, heads, 2, dim, dtype=torch.int8, device=cache[0].device), torch.zeros(pages, heads, dtype=_F32, device=cache[0].device))


def page_bounds(cache, bounds, block_table, kv_len, max_kv_len, row_start=None, max_rows=1):
    """Bounds of the keys in every page that the batch's rows were appended to (ogle_cuda_page_bounds), in place: behind `append`, with its
    batch. choose_pages needs them of all pages that a row may choose."""
    pages, heads, _, dim = cache[0].shape
    # rows are not looked at, but row_start is cut to their number: any that a batch could have, and any type
    rows = block_table.shape[0] if row_start is None else (1 << 30) // heads
    here = _device(cache[0], "cache")
    b = _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, heads, torch.bfloat16, here)
    check(_lib.cuda_lib().ogle_cuda_page_bounds(b, *_bounds(bounds, pages, heads, dim, here), _here(here)), "page_bounds")


def choose_pages(q, cache, bounds, block_table, kv_len, max_kv_len, row_start=None, max_rows=1, count=16, first=1, last=1):
    """The `count` pages that each row of q [rows, heads, head dim] attends (ogle_cuda_choose_pages), for each kv head as blocks of the row's
    sequence: the `first` ones, the row's own with the last - 1 before it, and of the others those whose keys, going by their bounds, can have
    the largest product with one of the head's queries, in 8 bits. Returns int32 [rows, kv heads, count], rising, filled up with -1."""
    if q.dim() != 3:
        raise ValueError("q: expected [rows, heads, head dim]")
    pages, kv_heads, _, dim = cache[0].shape
    rows, heads, _ = q.shape
    here = _device(q, "q")
    b = _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, heads, q.dtype, here)
    chosen = q.new_empty(rows, kv_heads, max(count, 0), dtype=_I32)
    p = _CHOOSE(*_rows(q, q.dtype, rows, heads, dim, "q", here), *_bounds(bounds, pages, kv_heads, dim, here), chosen.data_ptr(), kv_heads * count, count,
                count, first, last, 0)
    lib = _lib.cuda_lib()
    n = lib.ogle_cuda_choose_pages_workspace_bytes(b, p)
    workspace = q.new_empty(n, dtype=torch.uint8) if n else None
    check(lib.ogle_cuda_choose_pages(b, p, workspace.data_ptr() if n else 0, n, _here(here)), "choose_pages")
    return chosen


def sparse_attention(q, cache, chosen, block_table, kv_len, max_kv_len, row_start=None, max_rows=1, scale=None, out=None):
    """Softmax attention of q [rows, heads, head dim] over the tokens, up to the row's own, of the pages that choose_pages has chosen for the
    row and kv head (ogle_cuda_sparse_attention). chosen: int32 [rows, kv heads, count], rising, filled up with -1. Returns (out, lse) as
    `attention` does."""
    dtype = q.dtype
    if q.dim() != 3:
        raise ValueError("q: expected [rows, heads, head dim]")
    rows, heads, dim = q.shape
    kv_heads = cache[0].shape[1]
    here = _device(q, "q")
    b = _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, heads, dtype, here)
    pq = _rows(q, dtype, rows, heads, cache[0].shape[3], "q", here)
    if chosen.dim() != 3 or chosen.dtype != _I32 or chosen.get_device() != here or chosen.shape[0] != rows or chosen.shape[1] != kv_heads or chosen.stride(2) != 1 and chosen.shape[2] > 1:
        raise ValueError(f"chosen: expected an int32 CUDA tensor [{rows}, {kv_heads}, count], a choice's entries side by side")
    if out is None:
        out = q.new_empty(rows, heads, dim)
        po = out.data_ptr(), heads * dim, dim
    else:
        po = _rows(out, dtype, rows, heads, dim, "out", here)
    lse = q.new_empty(rows, heads, dtype=_F32)
    p = _ATTENTION(pq[0], po[0], lse.data_ptr(), pq[1], pq[2], po[1], po[2], dim ** -0.5 if scale is None else scale, 1, 0, 0)
    count = chosen.shape[2]
    c = _CHOSEN(chosen.data_ptr(), chosen.stride(0) if rows > 1 else kv_heads * count, chosen.stride(1) if kv_heads > 1 else count, count, 0)
    lib = _lib.cuda_lib()
    n = lib.ogle_cuda_sparse_attention_workspace_bytes(b, p, c) if row_start is not None and max_rows > 1 else 0       # of single rows none
    workspace = q.new_empty(n, dtype=torch.uint8) if n else None
    check(lib.ogle_cuda_sparse_attention(b, p, c, workspace.data_ptr() if n else 0, n, _here(here)), "sparse_attention")
    return out, lse
