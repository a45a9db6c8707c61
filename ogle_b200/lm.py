"""The operators of a language model's decoding step (include/ogle_cuda.h): keys and values appended to a paged cache held
in 8 bits, attention over that cache, and the adjustment of logits before a token is chosen. One function per entry point,
on torch CUDA tensors; torch is used for device memory and the current stream only.

The cache is four tensors (k, v, k_scale, v_scale): k and v float8_e4m3fn [pages, kv heads, page tokens, head dim] (any strides
that keep a token's elements side by side and 16-byte boundaries), one float32 scale for each page and kv head, a power of two, or 0
where append has met nothing but zeros in the page. `new_cache` makes one; a page may be anywhere in it. Sequence b's token j lies in
page block_table[b, j // page tokens].

Rows are the new tokens of all sequences, one sequence behind the other: sequence b has rows row_start[b]..row_start[b + 1], the
last of the kv_len[b] tokens that it has once they are appended. Without row_start every sequence has one row. max_kv_len and
max_rows are the host's bounds of what kv_len and row_start hold on the device: nothing here waits for the device. Rows of a sequence
behind its first max_rows, rows that no sequence has (a padded batch), and tokens from max_kv_len on are ignored: a result made here
holds what was in memory there.
"""
import torch

from . import _lib
from ._lib import check
from .ops import _stream

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_PAGED_BATCH, _APPEND = _lib.packer(_lib.PagedBatch).pack, _lib.packer(_lib.AppendParams).pack
_ATTENTION, _LOGITS = _lib.packer(_lib.AttentionParams).pack, _lib.packer(_lib.LogitsParams).pack
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


def _vector(t, dtype, n, name):
    """Address of a contiguous vector of n values (any number, n None)."""
    if t is None:
        return 0
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name}: expected a contiguous {dtype} CUDA tensor" + (f" of {n} values" if n is not None else ""))
    return t.data_ptr()


def _rows(t, dtype, rows, heads, dim, name):
    """(address, row stride, head stride) of activations [rows, heads, dim]."""
    if t.dtype != dtype or not t.is_cuda or t.dim() != 3:
        raise ValueError(f"{name}: expected a {dtype} CUDA tensor [rows, heads, head dim]")
    shape, stride = t.shape, t.stride()
    if shape[0] != rows or shape[2] != dim or (heads is not None and shape[1] != heads) or (stride[2] != 1 and dim > 1):
        raise ValueError(f"{name}: expected [{rows}, {heads if heads is not None else 'heads'}, {dim}] with the elements of a head side by side, "
                         f"got {tuple(shape)} with strides {stride}")
    return t.data_ptr(), stride[0], stride[1]


def _batch(cache, block_table, kv_len, max_kv_len, row_start, max_rows, rows, q_heads, dtype):
    k, v, k_scale, v_scale = cache
    shape, stride = k.shape, k.stride()
    if k.dtype != _E4M3 or v.dtype != _E4M3 or not k.is_cuda or not v.is_cuda or len(shape) != 4 or shape != v.shape:
        raise ValueError("cache: expected float8_e4m3fn CUDA tensors [pages, kv heads, page tokens, head dim] for keys and values")
    pages, kv_heads, page_tokens, dim = shape
    if stride != v.stride() or stride[3] != 1:
        raise ValueError("cache: keys and values need the same strides, the elements of a token side by side")
    if dtype not in _DTYPE:
        raise ValueError(f"activations are float32, float16 or bfloat16, not {dtype}")
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
                        _vector(row_start, _I32, seqs + 1, "row_start"), _vector(kv_len, _I32, seqs, "kv_len"), block_table.data_ptr(),
                        k.data_ptr(), v.data_ptr(), _vector(k_scale, _F32, pages * kv_heads, "k_scale"),
                        _vector(v_scale, _F32, pages * kv_heads, "v_scale"))


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
