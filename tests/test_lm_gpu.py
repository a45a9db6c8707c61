"""The language-model operators (ogle_b200/lm.py) against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

import lm_checks as ref
from ogle_b200 import _lib, lm

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rows_of(rows, heads, dim, dtype, seed=1, amplitude=1.5):
    return (amplitude * torch.randn(rows, heads, dim, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


# ------------------------------------------------------------------------------------------------------ attention
CASES = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, window
    ([1], [0], 16, 1, 1, 16, 0),                                # a first token: one key
    ([1], [700], 64, 32, 8, 128, 0),
    ([1, 1, 1, 1], [0, 15, 16, 1000], 16, 8, 2, 64, 0),         # ends on and around a page's
    ([1] * 9, [3, 63, 64, 65, 127, 511, 2047, 0, 300], 64, 8, 8, 128, 0),    # one query head to a kv head
    ([1, 1], [130, 4000], 128, 16, 1, 128, 0),                  # sixteen query heads to one
    ([1, 1, 1], [77, 300, 5], 32, 15, 5, 80, 0),                # three to one, 80 elements
    ([1, 1], [260, 1029], 256, 6, 2, 256, 0),
    ([1, 1], [40, 500], 32, 12, 2, 48, 0),
    ([1, 1, 1], [5, 200, 3000], 64, 8, 2, 128, 100),            # windows shorter and longer than what there is
    ([1, 1], [31, 2000], 16, 4, 4, 64, 1),                      # a window of the row alone
    ([5, 5, 5], [0, 62, 1500], 32, 8, 4, 256, 64),              # drafts in a window
    ([3, 1, 7, 2], [10, 900, 61, 0], 16, 8, 2, 64, 0),
    ([40, 1, 17], [0, 333, 100], 64, 8, 2, 128, 0),             # prompts and single tokens together
    ([70], [0], 16, 4, 4, 96, 20),
    ([129, 64], [5, 0], 128, 4, 1, 64, 0),
    ([33], [50], 32, 16, 1, 256, 0),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, dtype):
    new, past, page, heads, kv_heads, dim, window = CASES[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=case)
    q = rows_of(sum(new), heads, dim, dtype)
    got = lm.attention(q, window=window, **batch)
    ref.check_attention(got, ref.attention64(q, batch, total, new, window=window), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_all_tokens(dtype):
    """Not causal: every row attends every token of its sequence; with a window, none before it."""
    new, past = [4, 1, 20], [60, 9, 0]
    batch, total = ref.make_batch(new, past, 16, 2, 64)
    q = rows_of(sum(new), 6, 64, dtype)
    for window in (0, 7):
        got = lm.attention(q, causal=False, window=window, scale=0.3, **batch)
        ref.check_attention(got, ref.attention64(q, batch, total, new, scale=0.3, causal=False, window=window), dtype)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_attention_with_negative_and_vanishing_scales(scale, dtype):
    new, past = [1, 3], [300, 20]
    batch, total = ref.make_batch(new, past, 16, 2, 128)
    q = rows_of(4, 8, 128, dtype)
    got = lm.attention(q, scale=scale, **batch)
    ref.check_attention(got, ref.attention64(q, batch, total, new, scale=scale), dtype)


def test_sequences_without_tokens_or_rows():
    new, past = [1, 0, 1, 3, 0], [10, 5, 0, 100, 0]
    batch, total = ref.make_batch(new, past, 16, 2, 128)
    q = rows_of(5, 8, 128, F32)
    ref.check_attention(lm.attention(q, **batch), ref.attention64(q, batch, total, new), F32)
    # the device says that a sequence has no token: its rows have no key
    batch["kv_len"][0] = 0
    batch["kv_len"][3] = 2                                       # of three rows the first stands before the text
    out, lse = lm.attention(q, **batch)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())
    assert bool(torch.isfinite(lse[1]).all()) and bool(torch.isfinite(lse[3:]).all())
    assert lm.attention(q[:0], **{**batch, "block_table": batch["block_table"][:0], "kv_len": batch["kv_len"][:0],
                                  "row_start": batch["row_start"][:1]})[0].shape == (0, 8, 128)
    none = {**batch, "kv_len": torch.zeros_like(batch["kv_len"]), "max_kv_len": 0}
    out, lse = lm.attention(q, **none)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_without_row_start_every_sequence_has_a_row():
    new, past = [1] * 5, [3, 100, 0, 64, 500]
    batch, total = ref.make_batch(new, past, 64, 2, 128)
    q = rows_of(5, 8, 128, BF16)
    with_it = lm.attention(q, **batch)
    del batch["row_start"], batch["max_rows"]
    without = lm.attention(q, **batch)
    assert torch.equal(with_it[0], without[0]) and torch.equal(with_it[1], without[1])


@pytest.mark.parametrize("dtype", [F32, F16])
def test_strides_of_queries_cache_and_results(dtype):
    """Queries that are a slice of a joint projection, a token-major cache, results into a slice."""
    new, past = [1, 4], [200, 30]
    batch, total = ref.make_batch(new, past, 32, 2, 64, token_major=True)
    assert not batch["cache"][0].is_contiguous()
    wide = rows_of(5, 12, 64, dtype)
    q, out = wide[:, :8], torch.full((5, 10, 64), 7.0, dtype=dtype, device="cuda")
    got = lm.attention(q, out=out[:, 1:9], **batch)
    ref.check_attention(got, ref.attention64(q, batch, total, new), dtype)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 9] == 7).all())


def test_table_entries_that_name_no_page():
    """Their tokens are not attended, whatever stands there."""
    batch, total = ref.make_batch([1, 2], [120, 90], 16, 2, 64)
    q = rows_of(3, 4, 64, F32)
    batch["block_table"][0, 2] = -1
    batch["block_table"][0, 5] = batch["cache"][0].shape[0]
    batch["block_table"][1, 0] = 2 ** 31 - 1
    out, lse = lm.attention(q, **batch)
    k_cache, v_cache, ks, vs = batch["cache"]
    row = 0
    for b, n in ((0, 1), (1, 2)):
        gone = torch.zeros(total[b], dtype=torch.bool)
        table = batch["block_table"][b].cpu().clone()
        for i in ((2, 5) if b == 0 else (0,)):
            gone[i * 16:(i + 1) * 16] = True
            table[i] = 0
        k, v = ref.cached(k_cache, ks, table, total[b]), ref.cached(v_cache, vs, table, total[b])
        for i in range(n):
            keep = ~gone & (torch.arange(total[b]) <= total[b] - n + i)
            for h in range(4):
                s = k[keep, h // 2] @ q[row, h].cpu().double() / 8
                want = torch.softmax(s, 0) @ v[keep, h // 2]
                assert float((out[row, h].cpu().double() - want).abs().max()) <= 2e-5 * float(v[keep].abs().max())
                assert abs(float(lse[row, h]) - float(torch.logsumexp(s, 0))) <= 2e-5 * max(1, abs(float(lse[row, h])))
            row += 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nan_reaches_only_the_rows_that_attend_it(dtype):
    """A NaN among a token's keys or values: rows that stand before it, or whose window has passed it, are as without it."""
    new, past = [6, 1, 40], [30, 100, 0]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=3)
    q = rows_of(sum(new), 4, 64, dtype)
    k_cache, v_cache = batch["cache"][:2]
    clean = lm.attention(q, window=24, **batch)

    def put(cache, b, token, head, element):
        at = int(batch["block_table"][b, token // 16])
        cache.view(torch.uint8)[at, head, token % 16, element] = 0xff

    put(v_cache, 0, 33, 0, 5)          # rows 3.. of sequence 0 attend it
    put(k_cache, 0, 34, 1, 0)
    put(v_cache, 1, 10, 0, 1)          # out of the window of the only row
    put(k_cache, 1, 40, 1, 9)
    put(v_cache, 2, 7, 1, 63)          # rows 7..30
    out, lse = lm.attention(q, window=24, **batch)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[3:6, 0:2, 5] = True
    hit[4:6, 2:4] = True
    hit[7 + 7:7 + 31, 2:4, 63] = True
    assert torch.equal(torch.isnan(out), hit)
    # other rows may move their unit of weights at another key than before: as near as rounding
    top = float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max())
    assert bool(((out[~hit] - clean[0][~hit]).abs() <= 2 * ref.LIMIT[dtype] * top + 2 * ref.half_step(clean[0][~hit].float(), dtype)).all())
    keys_hit = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    keys_hit[4:6, 2:4] = True
    assert torch.equal(torch.isnan(lse), keys_hit) and torch.allclose(lse[~keys_hit], clean[1][~keys_hit], rtol=2e-5, atol=2e-5)


def test_scores_far_apart_and_values_of_many_sizes():
    """Weights that vanish against later ones, pages whose scales differ by 2^20, queries from tiny to large."""
    new, past = [1, 1, 1], [600, 40, 1000]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=8)
    batch["cache"][3].mul_(torch.exp2(torch.randint(-10, 11, batch["cache"][3].shape, generator=torch.Generator().manual_seed(0)).float()).cuda())
    for amplitude in (1e-6, 20.0, 3000.0):
        q = rows_of(3, 8, 64, F32, amplitude=amplitude)
        out, lse = lm.attention(q, **batch)
        want, want_lse, top = ref.attention64(q, batch, total, new)
        # a score's error grows with it: a few roundings of 2^-23 of the largest, on weights and statistics
        tol = max(2e-5, 2.0 ** -20 * float(want_lse.abs().max()))
        assert float((out.cpu().double() - want).abs().max()) <= 4 * tol * top, amplitude
        assert float((lse.cpu().double() - want_lse).abs().max()) <= 2 * tol, amplitude


def test_offsets_beyond_32_bits():
    """Pages that lie more than 4 GB into the cache."""
    page, heads, dim = 256, 2, 256
    stride = heads * page * dim
    pages = (5 << 30) // stride
    k = torch.empty(pages, heads, page, dim, dtype=torch.uint8, device="cuda").view(ref.E4M3)
    v = torch.empty(pages, heads, page, dim, dtype=torch.uint8, device="cuda").view(ref.E4M3)
    ks, vs = torch.ones(pages, heads, device="cuda"), torch.ones(pages, heads, device="cuda")
    new, total = [1, 1], [300, 256]
    table = torch.tensor([[pages - 1, pages - 3], [pages - 2, -1]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(0)
    for c in (k, v):
        for p in (1, 2, 3):
            c[pages - p] = torch.randn(heads, page, dim, generator=g).to(ref.E4M3).cuda()
    batch = dict(cache=(k, v, ks, vs), block_table=table, kv_len=torch.tensor(total, dtype=torch.int32, device="cuda"), max_kv_len=300)
    q = rows_of(2, 4, dim, BF16)
    small = dict(cache=(k[pages - 3:], v[pages - 3:], ks[pages - 3:], vs[pages - 3:]), block_table=(table - (pages - 3)).clamp(min=-1))
    ref.check_attention(lm.attention(q, **batch), ref.attention64(q, small, total, new), BF16)
    kn, vn = rows_of(2, heads, dim, BF16, seed=5), rows_of(2, heads, dim, BF16, seed=6)
    lm.append(kn, vn, **batch)
    got = k[pages - 3].float()[:, (300 - 1) % page] * ks[pages - 3][:, None]
    assert float((got - kn[0].float()).abs().max()) <= float(kn[0].abs().max()) * 2.0 ** -4


def test_calls_on_another_stream_and_in_a_graph():
    new, past = [1] * 6, [50, 100, 2000, 7, 0, 900]
    batch, total = ref.make_batch(new, past, 64, 2, 128)
    q = rows_of(6, 8, 128, BF16)
    want = lm.attention(q, **batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lm.attention(q, **batch)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = lm.attention(q, **batch)
    batch["kv_len"] -= torch.tensor([0, 1, 64, 7, 0, 500], dtype=torch.int32, device="cuda")   # shorter: the device's lengths count
    graph.replay()
    shorter = lm.attention(q, **batch)
    torch.cuda.synchronize()
    assert torch.equal(captured[0], shorter[0]) and torch.equal(captured[1], shorter[1])
    assert not torch.equal(shorter[0], want[0])


PROMPTS = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, window
    ([65], [0], 64, 1, 1, 128, 0),                              # one row above what the form for few rows takes
    ([128], [128], 16, 2, 1, 128, 0),                           # two whole tiles of rows, one of keys
    ([129, 300], [0, 1000], 64, 8, 2, 128, 0),
    ([257, 1, 40], [77, 3000, 9], 32, 4, 4, 64, 0),             # items that share their sequence with none
    ([500], [100], 16, 6, 2, 80, 0),                            # three query heads to one, 80 elements
    ([700, 90], [0, 5000], 128, 2, 1, 128, 130),                # windows that are left behind within a tile
    ([100] * 30, list(range(0, 300, 10)), 64, 8, 4, 64, 0),     # more items than blocks
    ([200], [6000], 256, 16, 1, 128, 0),                        # few items: they are cut into parts
    ([70, 70], [2, 900], 16, 2, 2, 48, 1),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_attention_of_prompts(case, dtype):
    new, past, page, heads, kv_heads, dim, window = PROMPTS[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=100 + case)
    q = rows_of(sum(new), heads, dim, dtype)
    ref.check_attention(lm.attention(q, window=window, **batch), ref.attention64(q, batch, total, new, window=window), dtype)


def test_prompts_that_attend_all_tokens():
    new, past = [90, 200], [40, 0]
    batch, total = ref.make_batch(new, past, 16, 2, 64)
    q = rows_of(sum(new), 4, 64, BF16)
    for scale in (0.2, -0.1, 0.0):
        got = lm.attention(q, causal=False, window=50, scale=scale, **batch)
        ref.check_attention(got, ref.attention64(q, batch, total, new, scale=scale, causal=False, window=50), BF16)


def test_nan_in_prompts_reaches_only_the_rows_that_attend_it():
    new, past = [150, 300], [30, 100]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=3)
    q = rows_of(sum(new), 4, 64, BF16)
    clean = lm.attention(q, window=70, **batch)

    def put(cache, b, token, head, element):
        cache.view(torch.uint8)[int(batch["block_table"][b, token // 16]), head, token % 16, element] = 0x7f

    put(batch["cache"][1], 0, 60, 0, 5)        # rows 30..99 of sequence 0
    put(batch["cache"][1], 0, 60, 0, 40)
    put(batch["cache"][0], 0, 120, 1, 0)       # rows 90..
    put(batch["cache"][1], 1, 399, 1, 63)      # its last row alone
    out, lse = lm.attention(q, window=70, **batch)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[30:100, 0:2, 5] = hit[30:100, 0:2, 40] = True
    hit[90:150, 2:4] = True
    hit[449, 2:4, 63] = True
    assert torch.equal(torch.isnan(out), hit)
    top = float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max())
    assert bool(((out[~hit] - clean[0][~hit]).abs() <= 2 * ref.LIMIT[BF16] * top + 2 * ref.half_step(clean[0][~hit].float(), BF16)).all())
    keys_hit = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    keys_hit[90:150, 2:4] = True
    assert torch.equal(torch.isnan(lse), keys_hit) and torch.allclose(lse[~keys_hit], clean[1][~keys_hit], rtol=2e-5, atol=2e-5)


def test_prompts_over_missing_pages():
    """Rows whose every token has lost its page, and rows with some left."""
    new, past = [200], [0]
    batch, total = ref.make_batch(new, past, 16, 1, 64)
    q = rows_of(200, 2, 64, F16)
    batch["block_table"][0, 0] = batch["block_table"][0, 5] = -1
    out, lse = lm.attention(q, **batch)
    assert bool((out[:16] == 0).all()) and bool((lse[:16] == -math.inf).all())
    table = batch["block_table"][0].cpu().clamp(min=0)
    k, v = (ref.cached(batch["cache"][i], batch["cache"][2 + i], table, 200)[:, 0] for i in (0, 1))
    there = torch.ones(200, dtype=torch.bool)
    there[0:16] = there[80:96] = False
    for i in range(16, 200):
        keep = there & (torch.arange(200) <= i)
        for h in range(2):
            s = k[keep] @ q[i, h].cpu().double() / 8
            want = torch.softmax(s, 0) @ v[keep]
            assert bool(((out[i, h].cpu().double() - want).abs() <= ref.LIMIT[F16] * float(v[keep].abs().max()) + ref.half_step(want, F16)).all())
            assert abs(float(lse[i, h]) - float(torch.logsumexp(s, 0))) <= 2e-5 * max(1, abs(float(lse[i, h])))


@pytest.mark.parametrize("rows", [1, 200])
def test_a_wait_that_runs_out_is_reported_and_the_device_stays_usable(rows):
    """With no patience every wait for a copy gives up: the call ends, the status says so, the next one is right."""
    batch, total = ref.make_batch([rows], [300], 16, 2, 64)
    q = rows_of(rows, 4, 64, BF16)
    want = lm.attention(q, **batch)
    lib = _lib.cuda_lib()
    try:
        assert lib.ogle_cuda_set_wait_limit(0) == 0
        lm.attention(q, **batch)
        assert lib.ogle_cuda_device_status() == -6 and lib.ogle_cuda_device_status_detail() == 9
    finally:
        lib.ogle_cuda_set_wait_limit(-1)
        lib.ogle_cuda_clear_device_status()
    got = lm.attention(q, **batch)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert lib.ogle_cuda_device_status() == 0


def test_the_same_call_gives_the_same_bits():
    new, past = [1] * 3 + [5], [5000, 1, 800, 77]
    batch, total = ref.make_batch(new, past, 32, 4, 128)
    q = rows_of(8, 16, 128, F32)
    a, b = lm.attention(q, **batch), lm.attention(q, **batch)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --------------------------------------------------------------------------------------------------------- append
def check_append(new, past, page, heads, kv_heads, dim, rotary, interleaved, dtype, seed=0, spoil=None, token_major=False):
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=seed, token_major=token_major)
    rows = sum(new)
    qkv = rows_of(rows, heads + 2 * kv_heads, dim, dtype, seed=seed + 1, amplitude=2.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    if spoil:
        spoil(k, v, batch)
    table = lm.rotary_table(max(max(total), 1), rotary) if rotary else None
    before = [t.clone() for t in batch["cache"]]
    positions = torch.tensor([p + i for n, p in zip(new, past) for i in range(n)])
    kr, qr = k.cpu().float(), q.cpu().float()
    if rotary:
        kr, qr = ref.rotated32(k.cpu(), table.cpu(), positions, interleaved), ref.rotated32(q.cpu(), table.cpu(), positions, interleaved)
    want = [ref.append32(x, before[i], before[2 + i], batch["block_table"].cpu(), new, total) for i, x in ((0, kr), (1, v.cpu().float()))]
    out = lm.append(k, v, q=q, rotary=table, interleaved=interleaved, **batch)
    got = batch["cache"]
    for i in range(2):
        assert torch.equal(got[2 + i].cpu(), want[i][1]), "scales"
        assert ref.same_bytes(got[i], want[i][0]), "values"
    assert out.dtype == dtype and torch.equal(out.cpu().nan_to_num(), qr.to(dtype).nan_to_num())
    return batch, total


APPENDS = [
    # new, past, page, q heads, kv heads, dim, rotary, neighbours
    ([1], [0], 16, 4, 1, 64, 64, False),
    ([1], [700], 64, 32, 8, 128, 128, False),
    ([1] * 7, [15, 16, 17, 0, 300, 63, 1], 16, 6, 2, 64, 32, True),
    ([1, 1], [100, 31], 32, 3, 3, 80, 80, False),
    ([1, 1], [100, 31], 32, 5, 1, 80, 40, True),
    ([2, 1, 9], [14, 0, 70], 16, 4, 2, 48, 0, False),
    ([40, 1, 17], [3, 333, 0], 16, 8, 2, 128, 64, False),
    ([130, 300], [0, 60], 256, 2, 1, 256, 256, False),          # more of a page than the registers hold
    ([0, 5, 0, 33], [10, 5, 0, 1], 32, 2, 2, 16, 8, False),
    ([70] * 40, [0] * 40, 64, 2, 1, 32, 32, False),             # more sequences than a warp has lanes
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(case, dtype):
    check_append(*APPENDS[case], dtype, seed=case)


def test_append_to_a_token_major_cache():
    check_append([3, 1], [20, 40], 16, 4, 2, 64, 64, False, BF16, token_major=True)


def test_append_of_values_that_are_not_finite():
    """An infinity becomes the largest value, a NaN stays one, and the page's scale is that of the others."""
    def spoil(k, v, batch):
        v[0, 0, 3] = math.inf
        v[1, 1, 4] = -math.inf
        v[2, 0, 5] = math.nan
        v[5] = 0
        v[6, 1] = math.nan
    check_append([7], [16], 16, 2, 2, 64, 0, False, F32, spoil=spoil)


def test_append_without_a_page_stores_nothing():
    def spoil(k, v, batch):
        batch["block_table"][0, 1] = -1
    check_append([20, 3], [5, 0], 16, 2, 2, 64, 64, False, F32, spoil=spoil)


def test_tokens_one_by_one():
    """A text appended token by token: each value within half a step of e4m3 at its page's final scale, which is the one that the page's
    largest value needs. (A value that a growing scale has made subnormal is rounded once more.)"""
    page, heads, dim, n = 16, 2, 64, 50
    g = torch.Generator().manual_seed(4)
    x = torch.randn(n, heads, dim, generator=g) * torch.exp2(torch.linspace(-6, 6, n))[:, None, None]
    cache = lm.new_cache(8, heads, page, dim)
    table = torch.tensor([[5, 0, 3, 7]], dtype=torch.int32, device="cuda")
    for t in range(n):
        row = x[t:t + 1].cuda()
        assert lm.append(row, row, cache, table, torch.tensor([t + 1], dtype=torch.int32, device="cuda"), n) is None
    for c, s in ((cache[0], cache[2]), (cache[1], cache[3])):
        got = ref.cached(c, s, table[0], n)
        for first in range(0, n, page):
            part = x[first:first + page]
            scale = ref.scale_for(part.abs().amax((0, 2)))
            assert torch.equal(s[int(table[0, first // page])].cpu(), scale)
            step = torch.maximum(part.abs().double() * 2.0 ** -4, scale.double()[None, :, None] * 2.0 ** -9)
            assert bool(((got[first:first + page] - part.double()).abs() <= step).all())


def test_rotation_in_place():
    batch, total = ref.make_batch([2, 1], [3, 9], 16, 1, 64)
    table = lm.rotary_table(16, 64)
    k, q = rows_of(3, 1, 64, F16), rows_of(3, 4, 64, F16, seed=9)
    want = lm.append(k, k, q=q.clone(), rotary=table, **batch)
    got = lm.append(k, k, q=q, rotary=table, out=q, **batch)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


# --------------------------------------------------------------------------------------------------------- logits
def logits32(x, tokens, starts, prompt, rep, pres, freq, biases, allowed):
    """Row by row in fp32, each step rounded."""
    x = x.astype(np.float32).copy()
    rows, vocab = x.shape
    for r in range(rows):
        if tokens is not None:
            t = tokens[starts[r]:starts[r + 1]]
            inside = (t >= 0) & (t < vocab)
            n_prompt = prompt[r] if prompt is not None else 0
            seen = np.unique(t[inside])
            counts = np.bincount(t[n_prompt:][inside[n_prompt:]], minlength=vocab)
            if rep is not None:
                x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep[r], x[r, seen] * rep[r])
            said = np.nonzero(counts)[0]
            f = freq[r] if freq is not None else np.float32(0)
            p = pres[r] if pres is not None else np.float32(0)
            x[r, said] = (x[r, said] - f * counts[said].astype(np.float32)) - p
        if biases is not None:
            last = {int(t): v for t, v in zip(*biases[r])}
            for t, v in last.items():
                if 0 <= t < vocab:
                    x[r, t] = x[r, t] + v
        if allowed is not None:
            words = allowed[r if allowed.ndim == 2 else slice(None)]
            bits = (words[np.arange(vocab) // 32].view(np.uint32) >> (np.arange(vocab) % 32).astype(np.uint32)) & 1
            x[r, bits == 0] = -np.inf
    return x


def logits_case(rows, vocab, history, n_bias, masked, dtype, seed=0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((4 * rng.standard_normal((rows, vocab))).astype(np.float32)).to(dtype)
    counts = rng.integers(0, history + 1, rows)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tokens = (rng.random(starts[-1]) ** 3 * (vocab + 2)).astype(np.int32) - 1          # some outside
    prompt = rng.integers(0, history + 1, rows).astype(np.int32)
    rep, pres, freq = ((1 + rng.random(rows)).astype(np.float32), rng.random(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32))
    biases = [(rng.integers(-1, vocab + 1, n_bias).astype(np.int32), rng.standard_normal(n_bias).astype(np.float32)) for _ in range(rows)] if n_bias else None
    allowed = rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32) if masked else None
    return x, tokens, starts, prompt, rep, pres, freq, biases, allowed


def run_logits(x, tokens, starts, prompt, rep, pres, freq, biases, allowed, **more):
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda() if a is not None else None  # noqa: E731
    bt = bv = bs = None
    if biases is not None:
        bt, bv = np.concatenate([b[0] for b in biases]), np.concatenate([b[1] for b in biases])
        bs = np.concatenate([[0], np.cumsum([len(b[0]) for b in biases])]).astype(np.int32)
    return lm.adjust_logits(x.cuda(), d(tokens), d(starts), d(prompt), d(rep), d(pres), d(freq), d(bt), d(bv), d(bs), d(allowed), **more)


@pytest.mark.parametrize("rows,vocab,history,n_bias,masked", [
    (1, 1, 3, 1, True), (1, 31, 10, 0, True), (3, 33, 40, 5, True), (2, 4095, 300, 20, False), (5, 4096, 0, 7, True),
    (4, 4097, 5000, 0, True), (3, 32000, 800, 20, True), (2, 50001, 3000, 300, True), (33, 1003, 50, 3, False), (7, 8190, 200, 40, True)])
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
def test_logits(rows, vocab, history, n_bias, masked, dtype, out_dtype):
    """Equal to the formula in fp32, rounded once to the result's type. (Odd vocabularies: rows begin anywhere.)"""
    case = logits_case(rows, vocab, history, n_bias, masked, dtype, seed=vocab)
    got = run_logits(*case, out_dtype=out_dtype)
    want = torch.from_numpy(logits32(case[0].float().numpy(), *case[1:])).to(out_dtype)
    assert got.dtype == out_dtype and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_of_long_texts_and_bias_lists(dtype):
    """Rows around the counts that a token's word holds: 131071 tokens, 8191 biases; a token said more often than that."""
    rng = np.random.default_rng(5)
    counts, vocab = [131071, 131072, 400000, 10, 0], 20000
    x = torch.from_numpy((4 * rng.standard_normal((5, vocab))).astype(np.float32)).to(dtype)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tokens = np.concatenate([np.full(131071, 7), np.full(131072, 8), (rng.random(400000) ** 8 * vocab), np.arange(10)]).astype(np.int32)
    tokens[starts[2]:starts[2] + 200000] = 19999
    prompt = np.array([0, 1, 1000, 3, 0], dtype=np.int32)
    rep, pres, freq = np.full(5, 1.25, np.float32), np.full(5, 0.5, np.float32), np.array([1e-3, 1e-3, 1e-4, 1.0, 1.0], np.float32)
    biases = [(rng.integers(0, vocab, n).astype(np.int32), rng.standard_normal(n).astype(np.float32)) for n in (8191, 3, 8192, 9000, 30000)]
    case = (tokens, starts, prompt, rep, pres, freq, biases, None)
    got = run_logits(x, *case, out_dtype=F32)
    assert torch.equal(got.cpu(), torch.from_numpy(logits32(x.float().numpy(), *case)))


def test_logits_steps_that_are_left_out():
    x, tokens, starts, prompt, rep, pres, freq, biases, allowed = logits_case(4, 3000, 100, 6, True, F32)
    full = (tokens, starts, prompt, rep, pres, freq, biases, allowed)
    for gone in ((0, 1, 2, 3, 4, 5, 6), (2,), (3,), (4, 5), (6,), (7,), (0, 1, 2, 3, 4, 5, 7), (0, 1, 2, 3, 4, 5, 6, 7)):
        part = [None if i in gone else a for i, a in enumerate(full)]
        assert torch.equal(run_logits(x, *part).cpu(), torch.from_numpy(logits32(x.numpy(), *part)))
    one_mask = allowed[1]
    assert torch.equal(run_logits(x, *full[:-1], one_mask).cpu(), torch.from_numpy(logits32(x.numpy(), *full[:-1], one_mask)))


def test_logits_in_place_in_slices_and_not_finite():
    x, tokens, starts, prompt, rep, pres, freq, biases, allowed = logits_case(5, 777, 60, 4, True, F32)
    x[0, 5], x[1, 6], x[2, 7] = math.inf, -math.inf, math.nan
    allowed[2, 0] &= ~(1 << 7)                                  # the NaN is masked: it becomes minus infinity
    want = torch.from_numpy(logits32(x.numpy(), tokens, starts, prompt, rep, pres, freq, biases, allowed))
    for offset in (0, 1, 2, 3):
        wide = torch.full((5, 800), 9.0, device="cuda")
        wide[:, offset:offset + 777] = x.cuda()
        view = wide[:, offset:offset + 777]
        d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        bt, bv = np.concatenate([b[0] for b in biases]), np.concatenate([b[1] for b in biases])
        got = lm.adjust_logits(view, d(tokens), d(starts), d(prompt), d(rep), d(pres), d(freq), d(bt), d(bv),
                               d(np.arange(6, dtype=np.int32) * 4), d(allowed), out=view)
        assert got.data_ptr() == view.data_ptr() and torch.equal(got.cpu(), want)
        assert bool((wide[:, :offset] == 9).all()) and bool((wide[:, offset + 777:] == 9).all())
    assert float(want[2, 7]) == -math.inf


def test_logits_between_unlike_strides():
    """A result that lies differently from the logits: element by element."""
    x, *rest = logits_case(3, 500, 30, 2, True, BF16)
    out = torch.zeros(3, 511, device="cuda")[:, 3:503]
    got = run_logits(x, *rest, out=out)
    assert torch.equal(got.cpu(), torch.from_numpy(logits32(x.float().numpy(), *rest)))


def test_nothing_waited_in_vain():
    assert _lib.cuda_lib().ogle_cuda_device_status() == 0


# -------------------------------------------------------------------------------------------------------- example
def whole_text_logits(model, text, prompt_len, caches, page_tokens, pages, answers):
    """The example model's last logits from the whole text in 64 bits, over the keys and values that its cache holds."""
    w = lambda t: t.cpu().double()  # noqa: E731
    n, h, hk, d = len(text), model.q_heads, model.kv_heads, model.head_dim
    x = w(model.embedding)[text]
    table = w(model.rotary)[:n]
    for layer, cache in enumerate(caches):
        q = (x @ w(model.qkv[layer]).T).view(n, h + 2 * hk, d)[:, :h].clone()
        c, s = table[:, None, :d // 2], table[:, None, d // 2:]
        a, b = q[..., :d // 2].clone(), q[..., d // 2:].clone()
        q[..., :d // 2], q[..., d // 2:] = a * c - b * s, b * c + a * s
        k, v = (ref.cached(cache[i], cache[2 + i], torch.tensor(pages), n) for i in (0, 1))
        o = torch.zeros(n, h, d, dtype=torch.float64)
        hidden = torch.arange(n)[None] > torch.arange(n)[:, None]
        if model.window:
            hidden |= torch.arange(n)[None] <= torch.arange(n)[:, None] - model.window
        for i in range(h):
            p = torch.softmax((q[:, i] @ k[:, i // (h // hk)].T * d ** -0.5).masked_fill(hidden, -math.inf), 1)
            o[:, i] = p @ v[:, i // (h // hk)]
        x = x + o.reshape(n, -1) @ w(model.out[layer]).T
    return x[-1] @ w(model.embedding).T


@pytest.mark.parametrize("window", [0, 9])
def test_example_answers(window):
    """Prompts and single tokens through products, append, attention and logits: each step's logits are those of the whole text. (The
    cache holds what was quantised on the way, so keys and values are taken from it.) Tolerance: fp32-grade products and sums
    over two layers, 1e-4 of the largest logit."""
    from ogle_b200 import lm_example
    model = lm_example.Model(window=window)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(1, 1000, (n,), generator=g).tolist() for n in (5, 1, 40, 17)]
    answers = lm_example.Answers(model, prompts, favoured=((7, 4.0), (31, -2.0)))
    for _ in range(6):
        texts = [list(t) for t in answers.texts]
        got = answers.step().cpu().double()
        for b, text in enumerate(texts):
            want = whole_text_logits(model, text, len(prompts[b]), answers.caches, 16, answers.pages[b], answers)
            seen, said = torch.tensor(sorted(set(text))), torch.bincount(torch.tensor(text[len(prompts[b]):] or [0]), minlength=1000).double()
            if len(text) == len(prompts[b]):
                said.zero_()
            raw = float(want.abs().max())
            want[seen] = torch.where(want[seen] > 0, want[seen] / np.float64(np.float32(1.3)), want[seen] * np.float64(np.float32(1.3)))
            want -= said * np.float64(np.float32(0.2)) + (said > 0) * 0.5
            want[7] += 4.0
            want[31] -= 2.0
            assert float(got[b, 0]) == -math.inf
            assert float((got[b, 1:] - want[1:]).abs().max()) <= 1e-4 * raw
    assert all(0 not in t[len(p):] for t, p in zip(answers.texts, prompts))


def test_example_answers_do_not_depend_on_the_batch():
    from ogle_b200 import lm_example
    model = lm_example.Model()
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(1, 1000, (n,), generator=g).tolist() for n in (3, 30, 12)]
    together = lm_example.Answers(model, prompts)
    for _ in range(8):
        together.step()
    for i, p in enumerate(prompts):
        alone = lm_example.Answers(model, [p])
        for _ in range(8):
            alone.step()
        assert alone.texts[0] == together.texts[i]


def widened(batch):
    """The same batch under a bound of a million tokens: the attention cuts it into ranges, where short bounds have a cluster of blocks a
    tile of rows."""
    table, page = batch["block_table"], batch["cache"][0].shape[2]
    wide = torch.full((table.shape[0], (1 << 20) // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return {**batch, "block_table": wide, "max_kv_len": 1 << 20}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_under_a_wide_bound(case, dtype):
    new, past, page, heads, kv_heads, dim, window = CASES[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=case)
    q = rows_of(sum(new), heads, dim, dtype)
    got = lm.attention(q, window=window, **widened(batch))
    ref.check_attention(got, ref.attention64(q, batch, total, new, window=window), dtype)
    got = lm.attention(q, **widened(batch))
    ref.check_attention(got, ref.attention64(q, batch, total, new), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_many_sequences_in_windows(dtype):
    """More tiles of rows than the GPU has blocks for clusters."""
    new, past = [1 + b % 3 for b in range(210)], [(37 * b) % 300 for b in range(210)]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=4)
    q = rows_of(sum(new), 4, 64, dtype)
    for window in (0, 33):
        got = lm.attention(q, window=window, **batch)
        ref.check_attention(got, ref.attention64(q, batch, total, new, window=window), dtype)


def test_missing_pages_and_empty_sequences_under_a_wide_bound():
    new, past = [1, 0, 1, 3, 2], [10, 5, 0, 100, 300]
    batch, total = ref.make_batch(new, past, 16, 2, 128)
    batch["block_table"][4, 3] = -1
    q = rows_of(7, 8, 128, F32)
    batch["kv_len"][0] = 0
    batch["kv_len"][3] = 2                                       # of three rows the first stands before the text
    short, wide = lm.attention(q, **batch), lm.attention(q, **widened(batch))
    top = float(batch["cache"][1].float().nan_to_num().abs().amax((0, 1, 2, 3)) * batch["cache"][3].max())
    assert torch.equal(torch.isinf(short[1]), torch.isinf(wide[1])) and bool(torch.isinf(wide[1][0]).all())
    assert bool((wide[0][0] == 0).all()) and bool((wide[0][2] == 0).all())
    assert float((short[0] - wide[0]).abs().max()) <= 2 * ref.LIMIT[F32] * top


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nan_under_a_wide_bound(dtype):
    new, past = [6, 1], [30, 100]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=3)
    at = int(batch["block_table"][0, 2])
    batch["cache"][1].view(torch.uint8)[at, 0, 1, 5] = 0xff     # token 33 of sequence 0: its rows 3.. attend it
    q = rows_of(7, 4, 64, dtype)
    for b in (batch, widened(batch)):
        out, lse = lm.attention(q, **b)
        hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
        hit[3:6, 0:2, 5] = True
        assert torch.equal(torch.isnan(out), hit) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("wide", [False, True])
def test_both_forms_report_a_wait_that_runs_out(wide):
    batch, total = ref.make_batch([1, 2], [700, 90], 16, 2, 128)
    q = rows_of(3, 8, 128, BF16)
    lib = _lib.cuda_lib()
    want = lm.attention(q, **(widened(batch) if wide else batch))
    lib.ogle_cuda_set_wait_limit(0)
    try:
        lm.attention(q, **(widened(batch) if wide else batch))
        torch.cuda.synchronize()
        assert lib.ogle_cuda_device_status() != 0
    finally:
        lib.ogle_cuda_set_wait_limit(-1)
        lib.ogle_cuda_clear_device_status()
    again = lm.attention(q, **(widened(batch) if wide else batch))
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_attention_of_prompts_under_a_wide_bound(case, dtype):
    """The tensor cores' form, which short calls do without."""
    new, past, page, heads, kv_heads, dim, window = PROMPTS[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=100 + case)
    q = rows_of(sum(new), heads, dim, dtype)
    for causal in (True, False):
        got = lm.attention(q, window=window, causal=causal, **widened(batch))
        ref.check_attention(got, ref.attention64(q, batch, total, new, window=window, causal=causal), dtype)


@pytest.mark.parametrize("rows", [150, 300])
def test_nan_and_missing_pages_in_prompts_under_a_wide_bound(rows):
    new, past = [rows, 200], [30, 100]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=3)
    q = rows_of(sum(new), 4, 64, BF16)
    clean = lm.attention(q, window=70, **widened(batch))
    ref.check_attention(clean, ref.attention64(q, batch, total, new, window=70), BF16)
    at = int(batch["block_table"][0, 5])
    batch["cache"][1].view(torch.uint8)[at, 1, 4, 33] = 0x7f    # token 84 of sequence 0: rows 54..123 attend it
    out, lse = lm.attention(q, window=70, **widened(batch))
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[54:124, 2:4, 33] = True
    assert torch.equal(torch.isnan(out), hit) and bool(torch.isfinite(lse).all())
    batch["block_table"][0, 5] = -1                             # nobody attends its 16 tokens, nor the NaN
    for b in (batch, widened(batch)):
        gone = lm.attention(q, window=70, **b)
        assert bool(torch.isfinite(gone[0]).all())
    few, many = lm.attention(q, window=70, **batch), gone
    top = float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max())
    assert bool(((few[0].float() - many[0].float()).abs() <= 2 * ref.LIMIT[BF16] * top + 2 * ref.half_step(few[0].float(), BF16)).all())
    assert torch.allclose(few[1], many[1], rtol=2e-5, atol=2e-5)


def test_prompts_longer_than_their_text_under_a_wide_bound():
    """The device says that a sequence has fewer tokens than rows: the first rows stand before the text."""
    batch, total = ref.make_batch([400, 300], [0, 50], 64, 2, 128)
    q = rows_of(700, 8, 128, F16)
    batch["kv_len"][0] = 90
    for b in (batch, widened(batch)):
        out, lse = lm.attention(q, **b)
        assert bool((out[:310] == 0).all()) and bool(torch.isinf(lse[:310]).all())
        assert bool(torch.isfinite(lse[310:]).all())
        only = {**b, "row_start": torch.tensor([0, 90, 390], dtype=torch.int32, device="cuda"), "max_rows": 300}
        same = lm.attention(q[310:], **only)
        limit = 2 * ref.LIMIT[F16] * float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max()) + 2 * ref.half_step(same[0].float(), F16)
        assert bool(((out[310:].float() - same[0].float()).abs() <= limit).all())


def logits_in_place(view, tokens, starts, prompt, rep, pres, freq, biases, allowed):
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    bs = np.concatenate([[0], np.cumsum([len(b[0]) for b in biases])]).astype(np.int32)
    return lm.adjust_logits(view, d(tokens), d(starts), d(prompt), d(rep), d(pres), d(freq), d(np.concatenate([b[0] for b in biases])),
                            d(np.concatenate([b[1] for b in biases])), d(bs), d(allowed), out=view)


@pytest.mark.parametrize("vocab", [1021, 1022, 1023, 2042, 2045, 8190, 32767])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_logits_of_vocabularies_just_below_whole_pieces(vocab, rows, dtype):
    """A row that begins on a 16-byte boundary needs a block less than one that does not: penalties are applied once, in place too, tokens far
    outside the vocabulary are ignored, and nothing behind a row is touched."""
    x, tokens, starts, prompt, rep, pres, freq, biases, allowed = logits_case(rows, vocab, 600, 9, True, dtype, seed=vocab + rows)
    rng = np.random.default_rng(rows)
    out_of = rng.random(len(tokens)) < 0.3
    tokens[out_of] = vocab + (rng.random(int(out_of.sum())) * 3000).astype(np.int32)
    case = (tokens, starts, prompt, rep, pres, freq, biases, allowed)
    want = torch.from_numpy(logits32(x.float().numpy(), *case)).to(dtype)
    wide = torch.full((rows + 1, vocab // 8 * 8 + 4096), 9.0, dtype=dtype, device="cuda")      # rows on boundaries
    for offset in (0, 1):
        wide.fill_(9.0)
        view = wide[:rows, offset:offset + vocab]
        view.copy_(x)
        got = logits_in_place(view, *case)
        assert got.data_ptr() == view.data_ptr() and torch.equal(got.cpu(), want)
        assert bool((wide[:, :offset] == 9).all()) and bool((wide[:rows, offset + vocab:] == 9).all()) and bool((wide[rows] == 9).all())
    assert torch.equal(run_logits(x, *case).cpu(), want)


def attention_through_c(q, batch, out, lse, fill):
    """lm.attention by way of the C entry point, in a workspace whose every byte is `fill`. Returns the workspace's size."""
    rows, heads, dim = q.shape
    lib = _lib.cuda_lib()
    b = lm._batch(batch["cache"], batch["block_table"], batch["kv_len"], batch["max_kv_len"], batch["row_start"], batch["max_rows"], rows, heads, q.dtype)
    p = lm._ATTENTION(q.data_ptr(), out.data_ptr(), lse.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1), dim ** -0.5, 1, 0, 0)
    n = lib.ogle_cuda_paged_attention_workspace_bytes(b, p)
    workspace = torch.full((n,), fill, dtype=torch.uint8, device="cuda")
    assert lib.ogle_cuda_paged_attention(b, p, workspace.data_ptr(), n, lm._stream()) == 0
    return n


@pytest.mark.parametrize("past,kv_heads", [([30000] + [10] * 19, 8), ([100000, 9, 9], 1), ([40000] + [30] * 90, 8)])
def test_a_block_that_gives_up_leaves_segments_behind_it(past, kv_heads):
    """Ranges that have several segments, in a workspace of arbitrary bytes: the call ends, reports itself and stores nothing outside its rows."""
    n = len(past)
    batch, total = ref.make_batch([1] * n, past, 64, kv_heads, 64)
    q = rows_of(n, 2 * kv_heads, 64, BF16)
    want = lm.attention(q, **batch)
    wide, lse = torch.full((n + 2, 2 * kv_heads, 64), 5.0, dtype=BF16, device="cuda"), torch.full((n + 2, 2 * kv_heads), 5.0, device="cuda")
    out, lib = wide[1:n + 1], _lib.cuda_lib()
    assert attention_through_c(q, batch, out, lse[1:n + 1], 0x7f) > _lib.ATTENTION_NO_WORKSPACE      # ranges, no clusters
    assert torch.equal(out, want[0]) and torch.equal(lse[1:n + 1], want[1])
    lib.ogle_cuda_set_wait_limit(0)
    try:
        attention_through_c(q, batch, out, lse[1:n + 1], 0x7f)
        torch.cuda.synchronize()
        assert lib.ogle_cuda_device_status() == -6 and lib.ogle_cuda_device_status_detail() == 9
    finally:
        lib.ogle_cuda_set_wait_limit(-1)
        lib.ogle_cuda_clear_device_status()
    for t in (wide, lse):
        assert bool((t[0] == 5).all()) and bool((t[n + 1] == 5).all())
    again = lm.attention(q, **batch)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_a_bound_of_no_rows_leaves_everything_as_it_is():
    batch, total = ref.make_batch([2, 1], [30, 400], 16, 2, 64)
    batch["max_rows"] = 0
    q = rows_of(3, 4, 64, BF16)
    out, before = torch.full_like(q, 5.0), [t.clone() for t in batch["cache"]]
    assert lm.attention(q, out=out, **batch)[0] is out
    lm.append(q[:, :2], q[:, 2:], q=q, out=out, **batch)
    torch.cuda.synchronize()
    assert bool((out == 5).all()) and _lib.cuda_lib().ogle_cuda_device_status() == 0
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(batch["cache"], before))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_first_copies_of_many_short_blocks(dim):
    """Blocks that ask for copies as soon as they have begun, in both kinds of division, again and again: the same bits every time."""
    n = 60
    batch, total = ref.make_batch([1] * n, [(53 * b) % 130 for b in range(n)], 16, 4, dim, seed=dim)
    q = rows_of(n, 8, dim, BF16)
    for b in (batch, widened(batch)):
        want = lm.attention(q, **b)
        ref.check_attention(want, ref.attention64(q, b, total, [1] * n), BF16)
        for _ in range(50):
            got = lm.attention(q, **b)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert _lib.cuda_lib().ogle_cuda_device_status() == 0


def poisoned_memory(*like):
    """Memory of these sizes handed back to the allocator full of NaN: what the next call's results take is not what was right before."""
    held = [torch.full_like(t, math.nan) for t in like for _ in range(2)]
    del held


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompts_shorter_than_their_bound(dim, dtype):
    """As many rows as sequences x max_rows, but fewer of them in row_start: sequences of a few rows in a padded batch are answered, too."""
    bound, batches = 700, ([3, 700], [1, 1], [0, 60], [700, 0], [699, 5])
    for new in batches:
        batch, total = ref.make_batch(new, [400, 900], 64, 2, dim, seed=sum(new))
        batch["max_rows"], n = bound, sum(new)
        q = rows_of(2 * bound, 4, dim, dtype)
        poisoned_memory(q)
        out, lse = lm.attention(q, **batch)
        ref.check_attention((out[:n], lse[:n]), ref.attention64(q[:n], batch, total, new), dtype)


def test_a_captured_prompt_replayed_with_other_rows():
    """A step captured for a prompt of 1024 rows, replayed with rows and lengths of other steps."""
    rows, heads, page = 1024, 8, 64
    batch, total = ref.make_batch([rows], [3000], page, 2, 128, seed=9)
    q = rows_of(rows, heads, 128, BF16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = lm.attention(q, **batch)
    for n, past in ((1024, 3000), (3, 3000), (40, 17), (500, 0), (1, 4023)):
        batch["row_start"].copy_(torch.tensor([0, n], dtype=torch.int32))
        batch["kv_len"].fill_(past + n)
        out.fill_(math.nan)
        lse.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        ref.check_attention((out[:n], lse[:n]), ref.attention64(q[:n], batch, [past + n], [n]), BF16)
        assert bool(torch.isnan(lse[n:]).all())                  # rows behind row_start's last are nobody's


def rows64(q, batch, b, first, last, length, window=0, causal=True):
    """(out, lse, largest |v|) of rows q at positions first.. of sequence b, over the tokens below `last`, of `length` in the cache."""
    k, v = (ref.cached(batch["cache"][i], batch["cache"][2 + i], batch["block_table"][b], length)[:last] for i in (0, 1))
    n, heads, dim = q.shape
    pos, j = first + torch.arange(n)[:, None], torch.arange(last)[None]
    hidden = (j > pos) & causal | (j <= pos - window) & (window > 0)
    out, lse = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dtype=torch.float64)
    for h in range(heads):
        kh = h // (heads // k.shape[1])
        s = (q[:, h].cpu().double() @ k[:, kh].T * dim ** -0.5).masked_fill(hidden, -math.inf)
        lse[:, h] = torch.logsumexp(s, 1)
        out[:, h] = torch.softmax(s, 1).nan_to_num() @ v[:, kh]
    return out, lse, float(v.abs().max())


@pytest.mark.parametrize("new,past,max_rows,max_kv_len", [([5], [40], 3, 45), ([5, 1], [40, 90], 5, 60), ([4, 9], [100, 30], 2, 90),
                                                          ([900], [300], 600, 1200), ([900, 50], [300, 2000], 900, 1000)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_rows_and_tokens_beyond_the_bounds(new, past, max_rows, max_kv_len, dtype):
    """They are left out; those that are left keep their positions."""
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=max_kv_len)
    batch.update(max_rows=max_rows, max_kv_len=max_kv_len)
    q = rows_of(sum(new), 4, 64, dtype)
    for window, causal in ((0, True), (37, True), (37, False)):
        out, lse = lm.attention(q, window=window, causal=causal, **batch)
        row = 0
        for b, n in enumerate(new):
            m = min(n, max_rows)
            want = rows64(q[row:row + m], batch, b, past[b], min(total[b], max_kv_len), total[b], window, causal)
            ref.check_attention((out[row:row + m], lse[row:row + m]), want, dtype)
            row += n


@pytest.mark.parametrize("new,past,max_rows,max_kv_len", [([5], [40], 3, 45), ([5, 1], [40, 90], 5, 60), ([4, 40], [100, 30], 35, 62)])
def test_append_of_rows_beyond_the_bounds(new, past, max_rows, max_kv_len):
    """As an append of the rows within the bounds alone."""
    rows = sum(new)
    qkv = rows_of(rows, 8, 64, F32, amplitude=2.0)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    table = lm.rotary_table(max(n + p for n, p in zip(new, past)), 64)
    batch, total = ref.make_batch(new, past, 16, 2, 64)
    before = [t.clone() for t in batch["cache"]]
    out = torch.full((rows, 4, 64), 5.0, device="cuda")
    lm.append(k, v, q=q, rotary=table, out=out, **{**batch, "max_rows": max_rows, "max_kv_len": max_kv_len})
    keep = [max(0, min(n, max_rows, max_kv_len - p)) for n, p in zip(new, past)]
    at = torch.tensor([sum(new[:b]) + i for b, m in enumerate(keep) for i in range(m)])
    ends = [p + m if m else 0 for p, m in zip(past, keep)]
    positions = torch.tensor([p + i for p, m in zip(past, keep) for i in range(m)])
    for i, x in ((0, ref.rotated32(k.cpu()[at], table.cpu(), positions, False)), (1, v.cpu()[at])):
        want = ref.append32(x, before[i], before[2 + i], batch["block_table"].cpu(), keep, ends)
        assert torch.equal(batch["cache"][2 + i].cpu(), want[1]) and ref.same_bytes(batch["cache"][i], want[0])
    assert torch.equal(out.cpu()[at], ref.rotated32(q.cpu()[at], table.cpu(), positions, False))
    left = torch.ones(rows, dtype=torch.bool)
    left[at] = False
    assert bool((out.cpu()[left] == 5).all())


@pytest.mark.parametrize("rows", [20, 1100])
def test_the_longest_window(rows):
    """A window of 2^31 - 1 is none, for rows that stand before the text, too (not causal: they attend all of it)."""
    batch, total = ref.make_batch([rows], [0], 64, 2, 64)
    q = rows_of(rows, 4, 64, BF16)
    batch["kv_len"].fill_(12)
    for causal in (True, False):
        want = lm.attention(q, causal=causal, **batch)
        got = lm.attention(q, causal=causal, window=2 ** 31 - 1, **batch)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool(torch.isinf(want[1][:rows - 12]).all()) == causal


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("new", [[1, 3], [90, 200]])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_that_vanish_against_hidden_ones(dtype, new, wide):
    """Scores whose factor is below the smallest fp32 number are 0; those of hidden keys are minus infinity all the same."""
    batch, total = ref.make_batch(new, [50, 20], 16, 2, 64)
    batch["cache"][2].mul_(2.0 ** -60)
    q = rows_of(sum(new), 4, 64, dtype, amplitude=1e-18)
    for scale in (0.0, 1e-20, -1e-20):
        got = lm.attention(q, scale=scale, **(widened(batch) if wide else batch))
        ref.check_attention(got, ref.attention64(q, batch, total, new, scale=scale), dtype)


def check_each(got, q, batch, total, new, dtype, window=0, factor=1.0):
    """Against 64 bits (scores times `factor`), each element within what its own weights and values allow: LIMIT of the sum of |weight x value| - not of the largest value
    in the cache -, 2^-20 of the largest sum of |q k| for scores above 30, the result's rounding, and for each key a smallest fp16 number, 2^-25, against the row's largest weight x scale, which stands
    for at least 2^7; a value is at most 448 scales: 448 x 2^-32 < 2^-23 of it. Weights are fp32 numbers: below 2^-126 of the row's largest they are 0."""
    out, lse = (t.double() for t in got)
    heads, row, page = q.shape[1], 0, batch["cache"][0].shape[2]
    group = heads // batch["cache"][0].shape[1]
    for b, n in enumerate(new):
        at = batch["block_table"][b, :-(-total[b] // page)].long()

        def tokens(cache, scale):                               # [heads][tokens][...] of the sequence
            x = cache.view(torch.uint8)[at].view(ref.E4M3).double() * scale[at].double()[..., None, None]
            return x.transpose(0, 1).flatten(1, 2)[:, :total[b]].repeat_interleave(group, 0)

        k, v = (tokens(batch["cache"][i], batch["cache"][2 + i]) for i in (0, 1))
        scales = batch["cache"][3][at].double().T.repeat_interleave(page, 1)[:, :total[b]].repeat_interleave(group, 0)
        pos, j = torch.arange(total[b] - n, total[b], device="cuda")[:, None], torch.arange(total[b], device="cuda")[None]
        hidden = (j > pos) | (j <= pos - window) & (window > 0)
        x = q[row:row + n].double().transpose(0, 1) * (factor * q.shape[2] ** -0.5)
        s = (x @ k.transpose(1, 2)).masked_fill(hidden, -math.inf)
        size = (x.abs() @ k.abs().transpose(1, 2)).masked_fill(hidden, 0).amax(2, keepdim=True)
        p = torch.softmax(s, 2)
        want, sums = p @ v, p @ v.abs()
        step = ref.half_step(want, dtype).clamp(min={F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}[dtype]) + total[b] * 2.0 ** -117 * scales.amax(1)[:, None, None]
        limit = (ref.LIMIT[dtype] + 2.0 ** -20 * size) * sums + step + total[b] * 2.0 ** -23 * (p * scales[:, None]).amax(2, keepdim=True)
        over = (out[row:row + n].transpose(0, 1) - want).abs() / limit
        if dtype == F16:                                         # beyond the type's largest number: an infinity
            over = over.masked_fill((want.abs() + limit >= 65504) & (out[row:row + n].transpose(0, 1).abs() >= 65504), 0)
        over = over.amax()
        assert float(over) <= 1, (b, float(over))
        assert float((lse[row:row + n].T - torch.logsumexp(s, 2)).abs().max()) <= 2e-5 * max(1.0, float(s.masked_fill(hidden, 0).abs().max()))
        row += n


SPREADS = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, window: some calls of so many keys that a block goes through several pages
    ([1] * 40, [1500 + 37 * b for b in range(40)], 16, 8, 4, 64, 0),
    ([5] * 30, [900 + 50 * b for b in range(30)], 32, 16, 8, 128, 700),
    ([3, 16] * 12, [1300 + 60 * b for b in range(24)], 16, 12, 4, 256, 0),
    ([2] * 48, [1000] * 48, 16, 32, 2, 128, 0),
    ([5, 12], [43, 200], 16, 8, 4, 128, 50),                    # rows in a window that others of the tile have left
]


def outliers(batch, total, apart):
    """Every eighth page of a sequence of several, the first among them, has values 2^apart as large and keys against which queries that are
    positive score far below all others."""
    k, v, ks, vs = batch["cache"]
    page = k.shape[2]
    for b, t in enumerate(total):
        for i in range(0, -(-t // page), 8) if t > page else ():
            at = int(batch["block_table"][b, i])
            vs[at] *= 2.0 ** apart
            k.view(torch.uint8)[at] |= 0x80


@pytest.mark.parametrize("apart", [12, 24, 40])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(SPREADS)))
def test_pages_of_values_far_apart(case, dtype, apart):
    """Large values that a row does not attend, or hardly, leave the small ones that it does attend as they are."""
    new, past, page, heads, kv_heads, dim, window = SPREADS[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=200 + case)
    outliers(batch, total, apart)
    q = rows_of(sum(new), heads, dim, dtype, amplitude=8.0).abs()
    for b in (batch, widened(batch)):
        check_each(lm.attention(q, window=window, **b), q, b, total, new, dtype, window)


def append_rows(cache, table, x, start, together):
    """Rows x [n, heads, dim] as keys and values of one sequence from position `start` on, in calls of so many rows."""
    n, page = len(x), cache[0].shape[2]
    for i in range(0, n, together):
        part = x[i:i + together].cuda()
        m = len(part)
        lm.append(part, part, cache, table, torch.tensor([start + i + m], dtype=torch.int32, device="cuda"), table.shape[1] * page,
                  row_start=torch.tensor([0, m], dtype=torch.int32, device="cuda"), max_rows=m)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("together", [1, 3, 20])
def test_pages_that_begin_with_zeros(together, dtype):
    """Zeros ask for no scale: it is 0 until the head has another value, and then what that needs, also in a page used before."""
    page, heads, dim = 16, 3, 64
    x = torch.zeros(20, heads, dim)
    g = torch.Generator().manual_seed(2)
    x[5:, 0] = 1e-3 * torch.randn(15, dim, generator=g)          # zeros, then small values
    x[7, 1, 3], x[8, 1, 4] = 1e-30, -0.0                         # one value alone
    x = x.to(dtype)                                              # the last head: zeros
    cache = lm.new_cache(3, heads, page, dim)
    for s in cache[2:]:
        s.fill_(1024.0)                                          # what an earlier text has left
    table = torch.tensor([[2, 0]], dtype=torch.int32, device="cuda")
    append_rows(cache, table, x, 0, together)
    for c, s in ((cache[0], cache[2]), (cache[1], cache[3])):
        for at, first, end in ((2, 0, 16), (0, 16, 20)):
            top = x[first:end].float().abs().amax((0, 2))
            want = torch.where(top > 0, ref.scale_for(top), torch.zeros(()))
            assert torch.equal(s[at].cpu(), want)
        got, want = ref.cached(c, s, table[0], 20), x.double()
        scale = s.cpu().double()[[2] * 16 + [0] * 4][..., None]
        # half a step of e4m3 at the final scale, and as much where the scale has grown since (the value was rounded twice)
        assert bool(((got - want).abs() <= torch.maximum(want.abs() * 2.0 ** -3, scale * 2.0 ** -9)).all())
        assert bool((got[:, 2] == 0).all()) and bool((got[:5] == 0).all())


def test_infinities_and_nan_before_the_first_value():
    """They ask for no scale either: an infinity is the largest value that the scale has once there is one, a NaN stays one."""
    page, heads, dim = 16, 2, 64
    x = torch.zeros(6, heads, dim)
    x[1, 0, 0], x[1, 0, 1], x[2, 0, 2] = math.inf, -math.inf, math.nan
    x[3, 0, 5] = 0.01
    x[4, 1, 7] = math.inf
    for together in (1, 6):
        cache = lm.new_cache(1, heads, page, dim)
        append_rows(cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), x, 0, together)
        scale = float(ref.scale_for(torch.tensor(0.01)))
        assert torch.equal(cache[2].cpu(), torch.tensor([[scale, 0.0]]))
        got = cache[0].cpu().float()
        assert float(got[0, 0, 1, 0]) == 448 and float(got[0, 0, 1, 1]) == -448 and math.isnan(float(got[0, 0, 2, 2]))
        assert abs(float(got[0, 0, 3, 5]) * scale - 0.01) <= 0.01 * 2.0 ** -4
        assert float(got[0, 1, 4, 7]) == 448


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("new,heads,dtype", [([1, 4], 8, F32), ([1, 4], 8, BF16), ([300, 260], 8, F32), ([300, 260], 8, BF16), ([300, 260], 8, F16)])
def test_attention_over_pages_of_zeros(dtype, new, heads, wide):
    """Keys and values of scale 0 are zeros - scores of 0, no part in the result - and take no bits from small values beside them. What
    their bytes are does not matter (an infinity stored before any value is 448)."""
    batch, total = ref.make_batch(new, [200, 30], 16, 2, 64, seed=5)
    k, v, ks, vs = batch["cache"]
    vs.mul_(2.0 ** -30)
    for b, t in enumerate(total):
        for i in range(0, t // 16, 2):
            at = int(batch["block_table"][b, i])
            (ks if i % 4 else vs)[at] = 0.0
            k.view(torch.uint8)[at, :, 3] = v.view(torch.uint8)[at, :, 5] = 0x7e        # 448
    q = rows_of(sum(new), heads, 64, dtype)
    b = widened(batch) if wide else batch
    check_each(lm.attention(q, **b), q, b, total, new, dtype)


SPREAD_PROMPTS = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, window: all of more rows than the form for few rows takes
    ([700, 900], [300, 0], 16, 8, 2, 64, 0),
    ([520], [2000], 64, 4, 1, 128, 0),                          # few items: cut into parts
    ([1100, 600], [100, 900], 32, 6, 2, 80, 300),
    ([300] * 12, [170 * b for b in range(12)], 16, 16, 2, 128, 0),
]


@pytest.mark.parametrize("apart", [6, 12, 24, 40])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(SPREAD_PROMPTS)))
def test_prompts_over_pages_of_values_far_apart(case, dtype, apart):
    new, past, page, heads, kv_heads, dim, window = SPREAD_PROMPTS[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=300 + case)
    outliers(batch, total, apart)
    q = rows_of(sum(new), heads, dim, dtype, amplitude=8.0).abs()
    for b in (batch, widened(batch)):
        check_each(lm.attention(q, window=window, **b), q, b, total, new, dtype, window)


@pytest.mark.parametrize("which,apart", [(2, 20), (2, 30), (3, 20), (3, 30)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", range(len(SPREAD_PROMPTS)))
def test_prompts_before_keys_or_values_of_another_size(case, dtype, which, apart):
    """Keys or values of the text's last pages 2^apart as large: rows before them are as without them, small as theirs are."""
    new, past, page, heads, kv_heads, dim, window = SPREAD_PROMPTS[case]
    batch, total = ref.make_batch(new, past, page, kv_heads, dim, seed=400 + case)
    batch["cache"][which].mul_(2.0 ** -apart)
    for b, t in enumerate(total):
        for i in range(max(0, t // page - 3), -(-t // page)):
            batch["cache"][which][int(batch["block_table"][b, i])] *= 2.0 ** apart
    if which == 3 and dtype == F16:
        batch["cache"][3].mul_(2.0 ** 8)                        # fp16 results end at 2^-24 and at 65504
    q = rows_of(sum(new), heads, dim, dtype, amplitude=4.0)
    if which == 2:
        q *= 2.0 ** 4
    for b in (batch, widened(batch)):
        check_each(lm.attention(q, window=window, scale=2.0 ** (apart - 4) * dim ** -0.5 if which == 2 else None, **b), q, b, total, new, dtype, window,
                   2.0 ** (apart - 4) if which == 2 else 1.0)


@pytest.mark.parametrize("gap", [20, 55, 62, 66])
@pytest.mark.parametrize("rows,seqs,dtype", [(600, 1, BF16), (600, 1, F16), (1, 1, F32), (1, 48, F32), (1, 48, BF16), (5, 48, F16), (5, 48, BF16), (40, 12, F32)])
def test_values_beside_a_key_of_all_weight_and_no_value(rows, seqs, dtype, gap):
    """One key, of a page whose values are zeros, has nearly all of the weight; what the others add is near the smallest fp32 numbers."""
    new = [rows] * seqs
    batch, total = ref.make_batch(new, [200 + 1200 * (seqs > 1)] * seqs, 16, 2, 64, seed=6)
    k, v, ks, vs = batch["cache"]
    k.view(torch.uint8).zero_()
    ks.fill_(1.0)
    vs.mul_(2.0 ** -30)
    for b in range(seqs):
        at = int(batch["block_table"][b, 2])
        vs[at] = 0.0
        k.view(torch.uint8)[at, :, 5] = 0x38                     # 1
    q = torch.full((sum(new), 4, 64), 1.0, dtype=dtype, device="cuda")
    factor = gap / 64 * 8
    for b in (batch, widened(batch)):
        check_each(lm.attention(q, scale=factor / 8, **b), q, b, total, new, dtype, 0, factor)


@pytest.mark.parametrize("factor", [1e3, 1e6, 1e9, -1e9])
@pytest.mark.parametrize("new,past,window", [([1] * 24, [1200] * 24, 0), ([1, 3], [40, 700], 0), ([7] * 12, [900] * 12, 500), ([600, 300], [0, 900], 0), ([530], [3000], 700)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_of_any_size(new, past, window, factor, dtype):
    """Where fp32 scores lie further apart than weights reach, the largest still has a weight, and no weight is infinite."""
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=len(new))
    q = rows_of(sum(new), 4, 64, dtype, amplitude=4.0)
    for b in (batch, widened(batch)):
        check_each(lm.attention(q, scale=factor / 8, window=window, **b), q, b, total, new, dtype, window, factor)


@pytest.mark.parametrize("new,kv_len", [([4, 1, 30], [2, 0, 40]), ([1, 1, 1], [0, 5, 0]), ([40, 3], [0, 3])])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rotary", [0, 64])
def test_queries_of_rows_that_stand_before_the_text(new, kv_len, dtype, rotary):
    """The device says that a sequence has fewer tokens than rows: such rows' queries are 0, as the attention's results for them are."""
    batch, total = ref.make_batch(new, [100] * len(new), 16, 2, 64)
    batch["kv_len"].copy_(torch.tensor(kv_len, dtype=torch.int32))
    rows = sum(new)
    qkv = rows_of(rows, 10, 64, dtype)
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    table = lm.rotary_table(200, rotary) if rotary else None
    positions = torch.tensor([t - n + i for n, t in zip(new, kv_len) for i in range(n)])
    want = ref.rotated32(q.cpu(), table.cpu(), positions.clamp(min=0), False) if rotary else q.cpu().float()
    want[positions < 0] = 0
    poisoned_memory(torch.empty(rows, 6, 64, dtype=dtype, device="cuda"))
    assert torch.equal(lm.append(k, v, q=q, rotary=table, **batch).cpu(), want.to(dtype))
    in_place = q.clone()
    assert torch.equal(lm.append(k, v, q=in_place, out=in_place, rotary=table, **batch).cpu(), want.to(dtype))


def takes_the_prompt_form(q, batch):
    """The tensor cores' form asks for two parts of 256 rows for each of 148 blocks, more than the other form ever does."""
    rows, heads, dim = q.shape
    b = lm._batch(batch["cache"], batch["block_table"], batch["kv_len"], batch["max_kv_len"], batch["row_start"], batch["max_rows"], rows, heads, q.dtype)
    p = lm._ATTENTION(q.data_ptr(), q.data_ptr(), 0, q.stride(0), q.stride(1), q.stride(0), q.stride(1), 1.0, 1, 0, 0)
    return _lib.cuda_lib().ogle_cuda_paged_attention_workspace_bytes(b, p) >= 148 * 2 * 256 * ((64 if dim <= 64 else 128) + 2) * 4


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_the_limit_between_the_forms(dtype, dim):
    """The most rows that the form for few rows takes, and one more."""
    for wide in (False, True):
        forms, limit = [], 0
        for rows in (60, 4000):
            batch, _ = ref.make_batch([rows], [0], 64, 1, dim)
            forms.append(takes_the_prompt_form(rows_of(rows, 1, dim, dtype), widened(batch) if wide else batch))
        assert forms == [False, True]
        low, high = 60, 4000
        while high - low > 1:
            rows = (low + high) // 2
            batch, _ = ref.make_batch([rows], [0], 64, 1, dim)
            if takes_the_prompt_form(rows_of(rows, 1, dim, dtype), widened(batch) if wide else batch):
                high = rows
            else:
                low = rows
        for rows in (low, high):
            batch, total = ref.make_batch([rows], [0], 64, 1, dim)
            q = rows_of(rows, 1, dim, dtype)
            b = widened(batch) if wide else batch
            assert takes_the_prompt_form(q, b) == (rows == high)
            ref.check_attention(lm.attention(q, **b), ref.attention64(q, batch, total, [rows]), dtype)


@pytest.mark.parametrize("scale", [0.2, -0.1, 0.0])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 50), (True, 70)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_form_with_negative_and_vanishing_scales(dtype, causal, window, scale):
    new, past = [300, 90], [40, 700]
    batch, total = ref.make_batch(new, past, 16, 2, 80)
    q, b = rows_of(sum(new), 4, 80, dtype), widened(batch)
    assert takes_the_prompt_form(q, b)
    got = lm.attention(q, causal=causal, window=window, scale=scale, **b)
    ref.check_attention(got, ref.attention64(q, batch, total, new, scale=scale, causal=causal, window=window), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_form_with_nan_among_keys_and_values(dtype):
    new, past = [150, 300], [30, 100]
    batch, total = ref.make_batch(new, past, 16, 2, 64, seed=3)
    q, b = rows_of(sum(new), 4, 64, dtype), widened(batch)
    assert takes_the_prompt_form(q, b)
    clean = lm.attention(q, window=70, **b)

    def put(cache, b, token, head, element):
        cache.view(torch.uint8)[int(batch["block_table"][b, token // 16]), head, token % 16, element] = 0x7f

    put(batch["cache"][1], 0, 60, 0, 5)        # rows 30..99 of sequence 0
    put(batch["cache"][1], 0, 60, 0, 40)
    put(batch["cache"][0], 0, 120, 1, 0)       # rows 90..
    put(batch["cache"][1], 1, 399, 1, 63)      # its last row alone
    out, lse = lm.attention(q, window=70, **b)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[30:100, 0:2, 5] = hit[30:100, 0:2, 40] = True
    hit[90:150, 2:4] = True
    hit[449, 2:4, 63] = True
    assert torch.equal(torch.isnan(out), hit)
    top = float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max())
    assert bool(((out[~hit] - clean[0][~hit]).abs() <= 2 * ref.LIMIT[dtype] * top + 2 * ref.half_step(clean[0][~hit].float(), dtype)).all())
    keys_hit = torch.zeros(lse.shape, dtype=torch.bool, device="cuda")
    keys_hit[90:150, 2:4] = True
    assert torch.equal(torch.isnan(lse), keys_hit) and torch.allclose(lse[~keys_hit], clean[1][~keys_hit], rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_form_over_missing_pages(dtype):
    """Rows whose every token has lost its page, and rows with some left: as the form for few rows has them."""
    batch, total = ref.make_batch([200], [0], 16, 1, 64)
    q = rows_of(200, 2, 64, dtype)
    batch["block_table"][0, 0] = batch["block_table"][0, 5] = -1
    b = widened(batch)
    assert takes_the_prompt_form(q, b) and not takes_the_prompt_form(q, batch)
    out, lse = lm.attention(q, **b)
    assert bool((out[:16] == 0).all()) and bool((lse[:16] == -math.inf).all())
    few = lm.attention(q, **batch)
    top = float(batch["cache"][1].float().nan_to_num().abs().max() * batch["cache"][3].max())
    assert bool(((out.float() - few[0].float()).abs() <= 2 * ref.LIMIT[dtype] * top + 2 * ref.half_step(few[0].float(), dtype)).all())
    assert torch.allclose(lse[16:], few[1][16:], rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("limit", [0, 1, 40])
@pytest.mark.parametrize("new,past,apart", [([300], [200], 0), ([700, 130], [0, 900], 0), ([150] * 9, [2000] * 9, 0), ([700, 130], [200, 900], 30)])
def test_prompt_form_reports_a_wait_that_runs_out(new, past, apart, limit):
    """Whichever role's wait it is: the call ends, stores nothing outside its rows, and the next one is right."""
    batch, total = ref.make_batch(new, past, 16, 2, 64)
    if apart:
        outliers(batch, total, apart)
    n = sum(new)
    q, b = rows_of(n, 4, 64, BF16), widened(batch)
    assert takes_the_prompt_form(q, b)
    want, lib = lm.attention(q, **b), _lib.cuda_lib()
    wide, lse = torch.full((n + 2, 4, 64), 5.0, dtype=BF16, device="cuda"), torch.full((n + 2, 4), 5.0, device="cuda")
    lib.ogle_cuda_set_wait_limit(limit)
    try:
        attention_through_c(q, b, wide[1:n + 1], lse[1:n + 1], 0x7f)
        torch.cuda.synchronize()
        status, detail = lib.ogle_cuda_device_status(), lib.ogle_cuda_device_status_detail()
    finally:
        lib.ogle_cuda_set_wait_limit(-1)
        lib.ogle_cuda_clear_device_status()
    if limit == 0 or status:                                     # (a few polls may be enough: each waits a while)
        assert status == -6 and detail == 9
    else:
        assert torch.equal(wide[1:n + 1], want[0]) and torch.equal(lse[1:n + 1], want[1])
    for t in (wide, lse):
        assert bool((t[0] == 5).all()) and bool((t[n + 1] == 5).all())
    again = lm.attention(q, **b)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]) and lib.ogle_cuda_device_status() == 0
