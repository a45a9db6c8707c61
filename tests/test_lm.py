"""The language-model operators' checks of their arguments: no GPU needed."""
import ctypes as C
import os

import pytest
import torch

from ogle_b200 import _lib, lm

OK, INVALID, UNSUPPORTED, ALIGNMENT = 0, -1, -2, -4


def batch(**more):
    b = _lib.PagedBatch()
    b.n_seqs, b.n_rows, b.max_rows, b.max_kv_len = 2, 2, 1, 100
    b.q_heads, b.kv_heads, b.head_dim, b.page_tokens, b.n_pages, b.table_stride, b.dtype = 8, 2, 64, 16, 20, 7, _lib.DTYPE_BF16
    b.page_stride, b.head_stride, b.token_stride = 2048, 1024, 64
    b.kv_len = b.block_table = b.k_cache = b.v_cache = b.k_scale = b.v_scale = 1 << 20      # never read: the calls are refused
    for k, v in more.items():
        setattr(b, k, v)
    return b


def attend(b, workspace=1 << 20, size=1 << 40, **more):
    p = _lib.AttentionParams()
    p.q = p.out = p.lse = 1 << 20
    p.q_row = p.out_row = 512
    p.q_head = p.out_head = 64
    p.scale, p.causal = 0.125, 1
    for k, v in more.items():
        setattr(p, k, v)
    return _lib.cuda_lib().ogle_cuda_paged_attention(C.byref(b), C.byref(p), workspace, size, None)


def kv_append(b, **more):
    p = _lib.AppendParams()
    p.k = p.v = p.q = p.q_out = 1 << 20
    p.k_row = p.v_row = 128
    p.k_head = p.v_head = p.q_head = p.q_out_head = 64
    p.q_row = p.q_out_row = 512
    for k, v in more.items():
        setattr(p, k, v)
    return _lib.cuda_lib().ogle_cuda_kv_append(C.byref(b), C.byref(p), None)


@pytest.mark.parametrize("field,value,status", [
    ("n_seqs", -1, INVALID), ("n_rows", -1, INVALID), ("max_kv_len", -1, INVALID), ("max_kv_len", 113, INVALID), ("dtype", 3, INVALID),
    ("q_heads", 7, INVALID), ("kv_heads", 0, INVALID), ("head_dim", 0, INVALID), ("head_dim", 72, INVALID), ("head_dim", 272, UNSUPPORTED),
    ("page_tokens", 8, INVALID), ("page_tokens", 48, INVALID), ("page_tokens", 2048, INVALID), ("n_pages", -1, INVALID),
    ("page_stride", 2047, ALIGNMENT), ("head_stride", 8, ALIGNMENT), ("token_stride", 48, INVALID), ("token_stride", 72, ALIGNMENT),
    ("n_rows", 3, INVALID), ("kv_len", None, INVALID), ("block_table", None, INVALID), ("k_cache", None, INVALID), ("v_scale", None, INVALID),
    ("k_cache", 8, ALIGNMENT), ("n_rows", 1 << 30, UNSUPPORTED)])
def test_batches_that_are_refused(field, value, status):
    assert attend(batch(**{field: value})) == status
    assert kv_append(batch(**{field: value})) == status
    p = _lib.AttentionParams()
    assert _lib.cuda_lib().ogle_cuda_paged_attention_workspace_bytes(C.byref(batch(**{field: value})), C.byref(p)) == 0


def test_nothing_to_do_is_no_error():
    assert attend(batch(n_seqs=0, n_rows=0)) == OK
    assert kv_append(batch(n_seqs=0, n_rows=0)) == OK
    lib = _lib.cuda_lib()
    p = _lib.LogitsParams()
    assert lib.ogle_cuda_adjust_logits(C.byref(p), None) == OK


def test_attention_refusals():
    assert attend(batch(), q=None) == INVALID
    assert attend(batch(), out=None) == INVALID
    assert attend(batch(), window=-1) == INVALID
    assert attend(batch(), q=(1 << 20) + 2) == ALIGNMENT
    assert attend(batch(), q_row=513) == ALIGNMENT
    assert attend(batch(), workspace=None) == INVALID
    assert attend(batch(), workspace=(1 << 20) + 4) == ALIGNMENT
    assert attend(batch(), size=16) == INVALID
    lib = _lib.cuda_lib()
    assert lib.ogle_cuda_paged_attention(None, None, None, 0, None) == INVALID
    p = _lib.AttentionParams()
    assert lib.ogle_cuda_paged_attention_workspace_bytes(C.byref(batch()), C.byref(p)) > 0


def test_append_refusals():
    assert kv_append(batch(), k=None) == INVALID
    assert kv_append(batch(), q_out=None) == INVALID
    assert kv_append(batch(), k_head=65) == ALIGNMENT
    assert kv_append(batch(), v=(1 << 20) + 8) == ALIGNMENT
    for more in (dict(rotary_dim=12), dict(rotary_dim=0), dict(rotary_dim=72), dict(rotary_dim=64, rotary_rows=99)):
        assert kv_append(batch(), rotary=1 << 20, **{"rotary_rows": 100, **more}) == INVALID
    assert kv_append(batch(), rotary=(1 << 20) + 4, rotary_dim=64, rotary_rows=100) == ALIGNMENT
    assert _lib.cuda_lib().ogle_cuda_kv_append(None, None, None) == INVALID


def logits(**more):
    p = _lib.LogitsParams()
    p.rows, p.vocab, p.logits_stride, p.out_stride = 2, 100, 100, 100
    p.logits = p.out = 1 << 20
    for k, v in more.items():
        setattr(p, k, v)
    return _lib.cuda_lib().ogle_cuda_adjust_logits(C.byref(p), None)


def test_logits_refusals():
    assert logits(rows=-1) == INVALID
    assert logits(dtype=5) == INVALID
    assert logits(dtype=_lib.DTYPE_F16, out_dtype=_lib.DTYPE_BF16) == INVALID
    assert logits(logits=None) == INVALID
    assert logits(tokens=1 << 20) == INVALID                    # without token_start
    assert logits(bias_token=1 << 20, bias_start=1 << 20) == INVALID
    assert logits(logits_stride=99) == INVALID
    assert logits(allowed=1 << 20, allowed_stride=3) == INVALID
    assert logits(dtype=_lib.DTYPE_F16, out_dtype=_lib.DTYPE_F32) == INVALID     # in place, of another type
    assert logits(rows=1 << 17) == UNSUPPORTED
    assert _lib.cuda_lib().ogle_cuda_adjust_logits(None, None) == INVALID


def test_front_end_refuses_host_tensors_and_wrong_shapes():
    cache = lm.new_cache(4, 2, 16, 64, device="cpu")
    assert cache[0].shape == (4, 2, 16, 64) and cache[2].shape == (4, 2)
    x, table, n = torch.zeros(1, 2, 64), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        lm.attention(x, cache, table, n, 1)
    with pytest.raises(ValueError):
        lm.append(x, x, cache, table, n, 1)
    with pytest.raises(ValueError):
        lm.adjust_logits(torch.zeros(2, 10))


def test_rotary_table():
    t = lm.rotary_table(50, 16, base=100.0, device="cpu")
    assert t.shape == (50, 16) and t.dtype == torch.float32
    i = torch.arange(8, dtype=torch.float64)
    angle = 7 * 100.0 ** (-i / 8)
    assert torch.allclose(t[7].double(), torch.cat([angle.cos(), angle.sin()]), atol=1e-7)
    assert torch.equal(t[0], torch.cat([torch.ones(8), torch.zeros(8)]))


def test_structures_lie_as_the_header_says(tmp_path):
    """Offsets and sizes of the ctypes mirrors, and so of the packed bytes, against the compiler's."""
    import shutil
    import subprocess
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no g++")
    mirrors = {"OglePagedBatch": _lib.PagedBatch, "OgleAppendParams": _lib.AppendParams, "OgleAttentionParams": _lib.AttentionParams,
               "OgleLogitsParams": _lib.LogitsParams}
    lines = ["#include <cstddef>", '#include "ogle_cuda.h"']
    for name, mirror in mirrors.items():
        lines.append(f"static_assert(sizeof({name}) == {C.sizeof(mirror)}, \"\");")
        lines += [f"static_assert(offsetof({name}, {f}) == {getattr(mirror, f).offset}, \"\");" for f, _ in mirror._fields_]
    source = tmp_path / "layout.cc"
    source.write_text("\n".join(lines) + "\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    done = subprocess.run([compiler, "-std=c++17", "-fsyntax-only", "-I", include, str(source)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    packed = _lib.packer(_lib.AttentionParams).pack(1, 2, 3, 4, 5, 6, 7, 0.5, 1, 9, 0)
    back = _lib.AttentionParams.from_buffer_copy(packed)
    assert (back.q, back.out, back.lse, back.q_row, back.out_head, back.scale, back.causal, back.window) == (1, 2, 3, 4, 7, 0.5, 1, 9)
