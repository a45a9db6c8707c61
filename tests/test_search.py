"""Checks of the arguments of the operators that search and choose over the paged cache: no GPU needed."""
import ctypes as C
import os

import pytest
import torch

from ogle_b200 import _lib, lm
from test_lm import batch

OK, INVALID, UNSUPPORTED, ALIGNMENT = 0, -1, -2, -4
SOMEWHERE = 1 << 20                              # never read: the calls are refused


def filled(structure, **more):
    p = structure()
    for name, kind in structure._fields_:
        if kind is C.c_void_p:
            setattr(p, name, SOMEWHERE)
    for k, v in more.items():
        setattr(p, k, v)
    return p


def beam(workspace=SOMEWHERE, size=1 << 40, **more):
    p = filled(_lib.BeamParams, **{**dict(n_groups=2, beams=3, vocab=100, count=6, logits_stride=100, n_ends=1), **more})
    return _lib.cuda_lib().ogle_cuda_beam_step(C.byref(p), workspace, size, None)


@pytest.mark.parametrize("more,status", [
    (dict(n_groups=-1), INVALID), (dict(beams=0), INVALID), (dict(vocab=-1), INVALID), (dict(count=0), INVALID), (dict(dtype=3), INVALID),
    (dict(n_ends=-1), INVALID), (dict(logits_stride=99), INVALID), (dict(count=129), UNSUPPORTED), (dict(beams=1025), UNSUPPORTED),
    (dict(n_groups=30000), UNSUPPORTED), (dict(n_ends=1025), UNSUPPORTED), (dict(logits=None), INVALID), (dict(ends=None), INVALID),
    (dict(out_score=None), INVALID), (dict(next_token=None), INVALID), (dict(workspace=None), INVALID), (dict(size=16), INVALID),
    (dict(workspace=SOMEWHERE + 8), ALIGNMENT), (dict(logits=SOMEWHERE + 2), ALIGNMENT), (dict(n_groups=0), OK)])
def test_beam_step_refusals(more, status):
    assert beam(**more) == status


def test_workspaces_are_asked_for():
    lib = _lib.cuda_lib()
    assert lib.ogle_cuda_beam_step_workspace_bytes(C.byref(filled(_lib.BeamParams, n_groups=2, beams=3, vocab=100, count=6, logits_stride=100))) > 0
    assert lib.ogle_cuda_beam_step_workspace_bytes(C.byref(filled(_lib.BeamParams))) == 0
    assert lib.ogle_cuda_advance_pages_workspace_bytes(C.byref(filled(_lib.AdvanceParams, page_tokens=16))) > 0
    assert lib.ogle_cuda_compact_pages_workspace_bytes(C.byref(filled(_lib.CompactParams, page_tokens=16))) > 0
    many = batch(max_kv_len=16000, table_stride=1000)
    assert lib.ogle_cuda_choose_pages_workspace_bytes(C.byref(many), C.byref(filled(_lib.ChooseParams, count=4))) >= 2 * 2 * 1000 * 4
    for call in ("beam_step", "advance_pages", "compact_pages"):
        assert getattr(lib, f"ogle_cuda_{call}")(None, None, 0, None) == INVALID


ADVANCE = dict(n_old=2, n_new=3, old_blocks=4, new_blocks=4, page_tokens=16, n_pages=10, old_stride=4, new_stride=4,
               new_table=2 * SOMEWHERE, new_len=2 * SOMEWHERE, new_refs=2 * SOMEWHERE)


def advance(workspace=SOMEWHERE, size=1 << 40, **more):
    p = filled(_lib.AdvanceParams, **{**ADVANCE, **more})
    return _lib.cuda_lib().ogle_cuda_advance_pages(C.byref(p), workspace, size, None)


@pytest.mark.parametrize("more,status", [
    (dict(n_old=-1), INVALID), (dict(n_new=-1), INVALID), (dict(old_blocks=-1), INVALID), (dict(n_pages=-1), INVALID), (dict(page_tokens=24), INVALID),
    (dict(page_tokens=8), INVALID), (dict(page_tokens=2048), INVALID), (dict(old_stride=3), INVALID), (dict(new_stride=3), INVALID),
    (dict(n_pages=(1 << 26) + 1), UNSUPPORTED), (dict(n_new=1 << 20, new_blocks=1 << 12, new_stride=1 << 12), UNSUPPORTED), (dict(table=None), INVALID),
    (dict(kv_len=None), INVALID), (dict(parent=None), INVALID), (dict(refs=None), INVALID), (dict(state=None), INVALID), (dict(copies=None), INVALID),
    (dict(new_refs=SOMEWHERE), INVALID), (dict(new_table=SOMEWHERE), INVALID), (dict(new_len=SOMEWHERE), INVALID), (dict(workspace=None), INVALID),
    (dict(size=8), INVALID), (dict(workspace=SOMEWHERE + 2), ALIGNMENT)])
def test_advance_refusals(more, status):
    assert advance(**more) == status


@pytest.mark.parametrize("more,status", [
    (dict(n_seqs=-1), INVALID), (dict(n_copies=-1), INVALID), (dict(page_tokens=0), INVALID), (dict(table_stride=3), INVALID), (dict(refs=None), INVALID),
    (dict(copies=None), INVALID), (dict(new_table=None), INVALID), (dict(state=None), INVALID), (dict(new_refs=SOMEWHERE), INVALID),
    (dict(n_pages=(1 << 26) + 1), UNSUPPORTED), (dict(n_copies=(1 << 28) + 1), UNSUPPORTED)])
def test_compact_refusals(more, status):
    p = filled(_lib.CompactParams, **{**dict(n_seqs=2, blocks=4, page_tokens=16, n_pages=10, n_copies=5, table_stride=4, new_stride=4, new_refs=2 * SOMEWHERE), **more})
    lib = _lib.cuda_lib()
    assert lib.ogle_cuda_compact_pages(C.byref(p), SOMEWHERE, 1 << 40, None) == status
    if status == INVALID and "refs" not in more:
        assert lib.ogle_cuda_compact_pages(C.byref(p), SOMEWHERE, 0, None) == INVALID


COPY = dict(n_copies=3, n_layers=1, kv_heads=2, head_dim=64, page_tokens=16, n_pages=10, page_stride=2048, head_stride=1024, token_stride=64)


@pytest.mark.parametrize("more,layer,status", [
    (dict(n_copies=-1), {}, INVALID), (dict(n_layers=-1), {}, INVALID), (dict(kv_heads=0), {}, INVALID), (dict(head_dim=24), {}, INVALID),
    (dict(head_dim=272), {}, UNSUPPORTED), (dict(page_tokens=17), {}, INVALID), (dict(page_stride=2056), {}, ALIGNMENT), (dict(token_stride=48), {}, INVALID),
    (dict(head_stride=1 << 37), {}, UNSUPPORTED), (dict(copies=None), {}, INVALID), ({}, dict(k=None), INVALID), ({}, dict(v_scale=None), INVALID), ({}, dict(bounds_scale=None), INVALID),
    ({}, dict(v=SOMEWHERE + 4), ALIGNMENT), ({}, dict(bounds=SOMEWHERE + 8), ALIGNMENT), (dict(n_copies=0), {}, OK), (dict(n_layers=0), {}, OK)])
def test_copy_refusals(more, layer, status):
    p, t = filled(_lib.CopyPagesParams, **{**COPY, **more}), filled(_lib.PageTensors, **layer)
    assert _lib.cuda_lib().ogle_cuda_copy_pages(C.byref(p), C.byref(t), None) == status


def choose(b=None, workspace=SOMEWHERE, size=1 << 40, **more):
    p = filled(_lib.ChooseParams, **{**dict(q_row=512, q_head=64, chosen_row=16, chosen_head=8, count=8, first=1, last=1), **more})
    return _lib.cuda_lib().ogle_cuda_choose_pages(C.byref(b or batch()), C.byref(p), workspace, size, None)


@pytest.mark.parametrize("more,status", [
    (dict(count=0), INVALID), (dict(first=-1), INVALID), (dict(last=0), INVALID), (dict(first=8), INVALID), (dict(first=9), INVALID),
    (dict(last=2 ** 31 - 1), INVALID), (dict(q=None), INVALID), (dict(bounds=None), INVALID), (dict(bounds_scale=None), INVALID), (dict(chosen=None), INVALID),
    (dict(chosen_head=7), INVALID), (dict(chosen_row=7), INVALID), (dict(q_row=513), ALIGNMENT), (dict(bounds=SOMEWHERE + 8), ALIGNMENT),
    (dict(workspace=None), INVALID), (dict(size=100), INVALID), (dict(workspace=SOMEWHERE + 2), ALIGNMENT)])
def test_choose_refusals(more, status):
    many = batch(max_kv_len=16000, table_stride=1000)
    assert choose(many, **more) == status
    if "workspace" not in more and "size" not in more:
        assert choose(**more) == status
    assert choose(batch(n_seqs=-1)) == INVALID
    assert choose(batch(q_heads=514, kv_heads=2)) == UNSUPPORTED


def sparse(b=None, workspace=SOMEWHERE, size=1 << 40, choice={}, **more):
    p = filled(_lib.AttentionParams, **{**dict(q_row=512, out_row=512, q_head=64, out_head=64, scale=0.1, causal=1), **more})
    c = filled(_lib.ChosenPages, **{**dict(chosen_row=16, chosen_head=8, count=8), **choice})
    return _lib.cuda_lib().ogle_cuda_sparse_attention(C.byref(b or batch()), C.byref(p), C.byref(c), workspace, size, None)


@pytest.mark.parametrize("more,status", [
    (dict(causal=0), INVALID), (dict(window=5), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(choice=dict(chosen=None)), INVALID),
    (dict(choice=dict(count=0)), INVALID), (dict(choice=dict(chosen_head=7)), INVALID), (dict(q_row=513), ALIGNMENT), (dict(out=SOMEWHERE + 2), ALIGNMENT),
    (dict(workspace=SOMEWHERE + 2), ALIGNMENT), (dict(choice=dict(count=1 << 23, chosen_row=1 << 24, chosen_head=1 << 23)), UNSUPPORTED)])
def test_sparse_refusals(more, status):
    assert sparse(**more) == status
    # several rows to a tile: lists
    many = batch(n_rows=8000, max_rows=4000, row_start=SOMEWHERE)
    assert sparse(many, workspace=None) == INVALID
    assert sparse(many, size=64) == INVALID
    lib = _lib.cuda_lib()
    assert lib.ogle_cuda_sparse_attention(None, None, None, None, 0, None) == INVALID
    assert lib.ogle_cuda_page_bounds(C.byref(batch()), None, SOMEWHERE, None) == INVALID
    assert lib.ogle_cuda_page_bounds(C.byref(batch()), SOMEWHERE + 8, SOMEWHERE, None) == ALIGNMENT


def test_nothing_to_do_is_no_error():
    empty = batch(n_seqs=0, n_rows=0)
    assert choose(empty) == OK and sparse(empty) == OK
    assert _lib.cuda_lib().ogle_cuda_page_bounds(C.byref(empty), SOMEWHERE, SOMEWHERE, None) == OK


def test_front_end_refuses_host_tensors_and_wrong_shapes():
    cache = lm.new_cache(4, 2, 16, 64, device="cpu")
    bounds = lm.new_bounds(cache)
    assert bounds[0].shape == (4, 2, 2, 64) and bounds[0].dtype == torch.int8 and bounds[1].shape == (4, 2)
    x, table, n = torch.zeros(1, 2, 64), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: lm.beam_step(torch.zeros(4, 10), None, 2, 4), lambda: lm.beam_step(torch.zeros(4, 10), None, 3, 4),
                 lambda: lm.advance_pages(table, n, n, 1, n, 16), lambda: lm.compact_pages(table, n, 4, 16), lambda: lm.copy_pages([cache], torch.zeros(1, 3, dtype=torch.int32)),
                 lambda: lm.page_bounds(cache, bounds, table, n, 1), lambda: lm.choose_pages(x, cache, bounds, table, n, 1),
                 lambda: lm.sparse_attention(x, cache, torch.zeros(1, 2, 4, dtype=torch.int32), table, n, 1)):
        with pytest.raises(ValueError):
            call()


def test_structures_lie_as_the_header_says(tmp_path):
    """Offsets and sizes of the ctypes mirrors, and so of the packed bytes, against the compiler's."""
    import shutil
    import subprocess
    compiler = shutil.which("g++")
    if not compiler:
        pytest.skip("no g++")
    mirrors = {"OgleBeamParams": _lib.BeamParams, "OgleAdvanceParams": _lib.AdvanceParams, "OgleCompactParams": _lib.CompactParams,
               "OglePageTensors": _lib.PageTensors, "OgleCopyPagesParams": _lib.CopyPagesParams, "OgleChooseParams": _lib.ChooseParams,
               "OgleChosenPages": _lib.ChosenPages}
    lines = ["#include <cstddef>", '#include "ogle_cuda.h"']
    for name, mirror in mirrors.items():
        lines.append(f"static_assert(sizeof({name}) == {C.sizeof(mirror)}, \"\");")
        lines += [f"static_assert(offsetof({name}, {f}) == {getattr(mirror, f).offset}, \"\");" for f, _ in mirror._fields_]
        _lib.packer(mirror)
    source = tmp_path / "layout.cc"
    source.write_text("\n".join(lines) + "\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    done = subprocess.run([compiler, "-std=c++17", "-fsyntax-only", "-I", include, str(source)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


def test_a_search_refuses_empty_prompts():
    from ogle_b200 import lm_example
    with pytest.raises(ValueError):
        lm_example.Search(None, [[3, 4], []], 2)
