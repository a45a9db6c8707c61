"""The operators that search and choose over the paged cache (ogle_b200/lm.py) against plain implementations."""
import ctypes as C
import math
import random

import pytest
import torch

import lm_checks
import search_checks as ref
from ogle_b200 import _lib, lm, lm_example

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


# ------------------------------------------------------------------------------------------------------ beam_step
def beam_case(groups, beams, vocab, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(groups * beams, vocab, generator=g)).to(dtype)
    scores = -6 * torch.rand(groups * beams, generator=g) - 20 * torch.rand(groups, generator=g).repeat_interleave(beams)
    return x.cuda(), scores.cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 4, 7, 8), (3, 2, 255, 4), (2, 3, 4095, 6), (1, 4, 4097, 8), (5, 1, 8192, 2), (2, 5, 8193, 10), (1, 4, 32000, 8),
    (40, 4, 2001, 8), (2, 1024, 301, 128), (3, 8, 50001, 16), (1, 16, 150000, 32), (1, 100, 997, 128), (2, 2, 20, 128), (70, 8, 9001, 16), (1, 2, 129, 64)])
def test_beam_step(groups, beams, vocab, count, dtype):
    x, scores = beam_case(groups, beams, vocab, dtype)
    ends = [int(x[0].float().argmax()), vocab // 2]
    ref.check_beam_step(lm.beam_step(x, scores, beams, count, ends=ints(ends)), ref.beam_step(x, scores, beams, count, ends))
    ref.check_beam_step(lm.beam_step(x, None, beams, count), ref.beam_step(x, None, beams, count))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [500, 1030, 1500, 2047, 8192 + 1100, 4096 + 1300])
@pytest.mark.parametrize("beams,count", [(1, 1), (4, 40), (2, 128)])
def test_beam_step_of_batches_that_few_threads_have(beams, count, vocab, dtype):
    x, scores = beam_case(2, beams, vocab, dtype, seed=6)
    ref.check_beam_step(lm.beam_step(x, scores, beams, count), ref.beam_step(x, scores, beams, count))
    x[:, vocab // 9:] = -math.inf
    ref.check_beam_step(lm.beam_step(x, scores, beams, count), ref.beam_step(x, scores, beams, count))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [261, 515, 769, 1289, 2040])
@pytest.mark.parametrize("end", [-20.0, 0.0, 20.0])
def test_beam_step_of_rows_that_end_in_a_warp_with_few_logits(end, vocab, dtype):
    """The row's last few logits the least, ordinary or the largest; counts that the other warps' threads reach, and that they do not."""
    x, scores = beam_case(3, 3, vocab, dtype, seed=8)
    x[:, vocab - 5:] += end
    for count in (1, 6, 16, 33, 65, 128):
        ref.check_beam_step(lm.beam_step(x, scores, 3, count), ref.beam_step(x, scores, 3, count))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [300, 8192, 70001])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "lowest", "few", "two values"])
def test_beam_step_of_logits_in_order_and_alike(kind, vocab, dtype):
    """Rows whose every logit passes the border so far, or equals it."""
    beams, count = 3, 16
    x = torch.zeros(beams, vocab)
    i = torch.arange(vocab)
    if kind == "rising":
        x += i * (20.0 / vocab)
    elif kind == "falling":
        x -= i * (20.0 / vocab)
    elif kind == "lowest":                                   # a mask of the type's lowest value, and a handful that it lets through
        x += torch.finfo(dtype).min
        x[:, 5::vocab // 5] = torch.randn(beams, len(range(5, vocab, vocab // 5)), generator=torch.Generator().manual_seed(1))
    elif kind == "few":
        x += -math.inf
        x[0, vocab - 1] = 2.0
        x[2, 7] = -3.0
    elif kind == "two values":
        x[:, i % 3 == 1] = 1.0
    x, scores = x.to(dtype).cuda(), torch.tensor([-1.0, -1.3, -1.9]).cuda()
    ref.check_beam_step(lm.beam_step(x, scores, beams, count), ref.beam_step(x, scores, beams, count))


def test_beam_step_of_beams_that_are_alike():
    """Equal totals of different beams: by beam, then by token."""
    x, _ = beam_case(2, 4, 3001, F32)
    for b in (1, 3):
        x[b] = x[0]
    x[6] = x[5]
    scores = torch.tensor([-2.0, -2.0, -5.0, -2.0, -1.0, -3.0, -3.0, -9.0]).cuda()
    ref.check_beam_step(lm.beam_step(x, scores, 4, 16), ref.beam_step(x, scores, 4, 16))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_beam_step_of_values_that_are_not_finite(dtype):
    x, scores = beam_case(3, 4, 9001, dtype, seed=4)
    x[0, 5:9000:7] = math.nan
    x[1, [3, 8000]] = math.inf
    x[2] = -math.inf
    x[3, 8500:] = math.inf
    x[4, :8600] = -math.inf                                  # nothing in a block's first batches
    x[6] = math.nan
    scores[5], scores[7], scores[8:] = -math.inf, math.nan, -math.inf
    scores[9] = math.inf
    got = lm.beam_step(x, scores, 4, 8)
    ref.check_beam_step(got, ref.beam_step(x, scores, 4, 8))
    assert bool((got[1][2] == -1).all()) and bool((got[3][8:] == -1).all())      # a group without a text


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [8000, 30001])
def test_beam_step_of_logits_behind_a_mask_and_far_apart(vocab, dtype):
    """Masked for thousands of tokens, then logits of any size; steps upwards by more than an exponential holds; nothing but the lowest."""
    lowest = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(9)
    x = torch.randn(12, vocab, generator=g)
    x[0, :vocab - 100] = lowest
    x[1, :vocab - 100] = -math.inf
    x[2, :vocab - 100] = lowest
    x[2, vocab - 100:] -= 100
    x[3, :vocab // 2] = lowest
    x[3, vocab // 2:] -= 1000
    x[4] += 50 * (torch.arange(vocab) // (vocab // 7)).float()
    x[5] -= 50 * (torch.arange(vocab) // (vocab // 7)).float()
    x[6] = lowest
    x[7] = lowest
    x[7, 3] = -20000
    x[8] *= 10000
    x[9] = -30000 if dtype == F16 else -2e6
    x[10] = -30000 if dtype == F16 else -2e6
    x[10, vocab - 5:] = -0.9e6 if dtype != F16 else -29000
    x[11] = 65000 if dtype == F16 else 3e7
    x = x.to(dtype).cuda()
    scores = -torch.rand(12, generator=g).cuda()
    ref.check_beam_step(lm.beam_step(x, scores, 1, 6), ref.beam_step(x, scores, 1, 6))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift,stride", [(0, 5003), (1, 5004), (3, 5001), (5, 5008), (7, 6000)])
def test_beam_step_of_rows_at_any_address(shift, stride, dtype):
    x, scores = beam_case(2, 3, 5000, dtype)
    room = torch.full((6 * stride + 16,), math.nan, dtype=dtype, device="cuda")
    view = room[shift:shift + 6 * stride].view(6, stride)[:, :5000]
    view.copy_(x)
    ref.check_beam_step(lm.beam_step(view, scores, 3, 6), ref.beam_step(x, scores, 3, 6))


@pytest.mark.parametrize("spread", [0.01, 1.0, 12.0])
def test_beam_step_sums_are_near_64_bits(spread):
    """The scores of single rows, whose largest logit's total is minus the logarithm of the sum: flat, ordinary and peaked rows."""
    x, _ = beam_case(64, 1, 128001, F32, spread=spread)
    got = lm.beam_step(x, None, 1, 4)[0]
    want = torch.log_softmax(x.double(), 1).topk(4).values
    assert float((got.double() - want).abs().max()) <= 2.0 ** -22 + float(want.abs().max()) * 2.0 ** -24


def test_beam_step_results_do_not_depend_on_the_run():
    x, scores = beam_case(9, 4, 60001, BF16)
    first = lm.beam_step(x, scores, 4, 8)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, lm.beam_step(x, scores, 4, 8)))


# ------------------------------------------------------------------------------------------------------ pages
def check_advance(table, kv_len, parent, new, refs, page, blocks=None):
    wide = len(table[0]) if table else 1
    t = ints(table).view(len(table), wide)
    got = lm.advance_pages(t, ints(kv_len), ints(parent), ints(new) if isinstance(new, list) else new, ints(refs), page, blocks=blocks)
    want = ref.advance(table, kv_len, parent, new, refs, page, blocks if blocks is not None else wide)
    for g, w in zip(got, want):
        assert g.cpu().tolist() == [list(x) if isinstance(x, tuple) else x for x in w]
    return [list(map(list, want[0]))] + [list(w) for w in want[1:]]


def counts(tables, pages, held=()):
    refs = [0] * pages
    for t in tables:
        for row in t:
            for p in row:
                if 0 <= p < pages:
                    refs[p] += 1
    for p in held:
        refs[p] += 1
    return refs


@pytest.mark.parametrize("page,pages,seqs,blocks", [(16, 40, 5, 6), (64, 3000, 60, 20), (32, 1025, 33, 7), (16, 70, 1, 30), (16, 8192, 24, 40), (16, 8193, 24, 40),
                                                    (32, 6000, 25, 9)])
def test_pages_of_texts_that_grow_fork_end_and_are_cut(page, pages, seqs, blocks):
    r = random.Random(pages)
    refs = [0] * pages
    held = [pages - 1, 3]                                    # pages that another table names
    for p in held:
        refs[p] = 1
    # prompts
    table, kv_len, refs, copies, state = check_advance([[-1] * blocks], [0], [-1] * seqs, [r.randint(0, blocks * page // 2) for _ in range(seqs)], refs, page)
    for step in range(12):
        short = state[1] > 0
        kv_len = [n if r.random() < 0.8 else max(0, n - r.randint(0, 2 * page)) for n in kv_len]       # some give tokens back
        parent = [r.choice([i, r.randrange(len(table)), -1 if r.random() < 0.3 else i]) for i in range(len(table))]
        new = [r.choice([1, 1, 1, 0, r.randint(2, 3 * page), -5]) for _ in parent] if step % 2 else 1
        old = table
        table, kv_len, refs, copies, state = check_advance(table, kv_len, parent, new, refs, page, blocks if step != 7 else blocks + 3)
        assert refs == counts([table], pages, held)
        if short:
            break
    check_advance(table, kv_len, [], 1, refs, page)


def test_pages_that_run_out():
    page, table = 16, [[0, 1, -1], [0, 2, -1]]
    refs = counts([table], 5)
    got = check_advance(table, [20, 32], [0, 0, 1, 1, 0], 1, refs, page)
    assert got[4] == [1, 3] and got[3][0] == (-1, -1, 0) or got[4][1] > 0
    # and with none free from the start
    check_advance(table, [20, 32], [0, 0, 1], [40, 1, 16], counts([table], 3), page)


def test_pages_of_tables_with_gaps_and_strange_numbers():
    page = 16
    table = [[4, -1, 5, -1], [9, 6, 1000, -7], [8, 8, 2, 1]]
    refs = counts([table], 12)
    check_advance(table, [40, 33, 50], [0, 0, 1, 2, 2, 99, -3], [1, 20, 1, 14, 15, 3, 0], refs, page)
    check_advance(table, [-5, 100, 64], [2, 1, 0, 0], [1, 1, 1, 1], refs, page)
    check_advance(table, [40, 33, 50], [0, 1, 2], 1, refs, page, blocks=2)


def test_a_last_page_that_somebody_else_has_is_copied_for_all():
    page, table = 16, [[0, 1, -1]]
    refs = counts([table], 8, held=[1])
    got = check_advance(table, [20], [0, 0], 1, refs, page)
    assert got[3] == [(1, 2, 4), (1, 3, 4)] and got[2][1] == 1


@pytest.mark.parametrize("pages", [1, 1023, 1024, 1025, 3 << 20])
def test_pools_of_any_size(pages):
    """More than 2^20 pages: a count stands for more than 1024 of them."""
    g = torch.Generator().manual_seed(pages)
    refs = (torch.rand(pages, generator=g) < (0.999 if pages > 5000 else 0.6)).int()
    free = torch.nonzero(refs == 0)[:, 0]
    new = torch.tensor([100, 0, 37, 500] * 20, dtype=torch.int32)
    table, kv_len, now, copies, state = lm.advance_pages(ints([[-1] * 40]), ints([0]), torch.full((80,), -1, dtype=torch.int32).cuda(), new.cuda(), refs.cuda(), 16)
    wanted = (-(-new // 16)).tolist()
    at, asked = table.cpu(), 0
    for i, n in enumerate(wanted):
        mine = free[asked:asked + n].tolist()
        assert at[i].tolist() == mine + [-1] * (40 - len(mine)), i
        asked += n
    assert state.tolist() == [max(0, len(free) - asked), max(0, asked - len(free))]
    assert torch.equal((now.cpu() == 0).sum(), torch.tensor(max(0, len(free) - asked)))


def test_advance_of_nothing():
    table, kv_len, refs, copies, state = lm.advance_pages(ints([[2, -1]]), ints([5]), torch.empty(0, dtype=torch.int32).cuda(), 1, ints([0, 0, 1, 1]), 16)
    assert table.shape == (0, 2) and refs.tolist() == [0, 0, 0, 1] and state.tolist() == [3, 0]
    got = lm.advance_pages(torch.empty(0, 3, dtype=torch.int32).cuda(), torch.empty(0, dtype=torch.int32).cuda(), ints([-1, 0]), 20, ints([0] * 5), 16)
    assert got[0].tolist() == [[0, 1, -1], [2, 3, -1]] and got[4].tolist() == [1, 0]


@pytest.mark.parametrize("pages,seqs,blocks,most", [(50, 4, 5, 100), (50, 4, 5, 3), (2100, 30, 40, 500), (2100, 30, 40, 0), (1024, 1, 1, 5), (3, 1, 3, 3),
                                                    (8192, 20, 300, 2000), (8193, 20, 300, 2000), (5000, 110, 300, 900)])
@pytest.mark.parametrize("used", [0.0, 0.3, 0.9, 1.0])
def test_compact(pages, seqs, blocks, most, used):
    r = random.Random(pages + most)
    mine = r.sample(range(pages), int(used * pages))
    table = [[r.choice(mine + [-1]) if mine else -1 for _ in range(blocks)] for _ in range(seqs)]
    table[0][0] = pages + 5
    refs = counts([table], pages, held=mine[:3])
    got = lm.compact_pages(ints(table), ints(refs), most, 32)
    want = ref.compact(table, refs, most, 32)
    for g, w in zip(got, want):
        assert g.cpu().tolist() == [list(x) if isinstance(x, tuple) else x for x in w]


def test_compact_a_large_pool_in_calls_of_a_few():
    g = torch.Generator().manual_seed(5)
    refs = (torch.rand(1500000, generator=g) < 0.01).int().cuda()
    table = torch.nonzero(refs)[:, 0].int().view(1, -1)
    for _ in range(100):
        table, refs, copies, state = lm.compact_pages(table, refs, 1000, 16)
        if int(state[1]) == 0:
            break
    used = int(state[0])
    assert bool((refs[:used] == 1).all()) and bool((refs[used:] == 0).all()) and torch.equal(table.sort().values[0].long(), torch.arange(used, device="cuda"))


def random_bytes(shape, seed):
    return torch.randint(0, 255, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8)


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("heads,page,dim,layers", [(1, 16, 16, 1), (8, 64, 128, 3), (5, 32, 80, 2), (2, 1024, 256, 1), (3, 128, 48, 70)])
def test_copy_pages(heads, page, dim, layers, token_major):
    pages = 12
    copies = [(0, 5, page), (1, 6, 1), (2, 7, page - 1), (-1, -1, 0), (3, 8, 0), (3, 9, 7), (11, 10, page + 9), (4, pages, page), (4, -1, 5)]
    caches, bounds, want = [], [], []
    for layer in range(layers):
        cache = []
        for i in range(2):
            c = random_bytes((pages, page, heads, dim) if token_major else (pages, heads, page, dim), 10 * layer + i).cuda().view(torch.float8_e4m3fn)
            cache.append(c.transpose(1, 2) if token_major else c)
        scales = [torch.rand(pages, heads).cuda() for _ in range(2)]
        caches.append((*cache, *scales))
        bounds.append((random_bytes((pages, heads, 2, dim), layer).view(torch.int8).cuda(), torch.rand(pages, heads).cuda()))
        before = [t.cpu().clone() for t in (*caches[-1], *bounds[-1])]
        k, v = (t.view(torch.uint8) for t in before[:2])
        for src, dst, tokens in copies:
            if src < 0 or not 0 <= dst < pages:
                continue
            for t in (k, v):
                t[dst, :, :min(tokens, page)] = t[src, :, :min(tokens, page)]
            for t in before[2:]:
                t[dst] = t[src]
        want.append(before)
    lm.copy_pages(caches, ints(copies), bounds=bounds)
    for cache, b, before in zip(caches, bounds, want):
        for g, w in zip((*cache, *b), before):
            assert torch.equal(g.cpu().view(torch.uint8) if g.dtype == torch.float8_e4m3fn else g.cpu(), w.view(torch.uint8) if w.dtype == torch.float8_e4m3fn else w)
    lm.copy_pages([], ints(copies))
    lm.copy_pages(caches, torch.empty(0, 3, dtype=torch.int32).cuda())


# ------------------------------------------------------------------------------------------------------ bounds and choices
def with_bounds(batch, total):
    """Bounds of all pages of a batch, as appending its tokens step by step leaves them."""
    cache = batch["cache"]
    bounds = lm.new_bounds(cache)
    start = [0]
    for t in total:
        start.append(start[-1] + t)
    lm.page_bounds(cache, bounds, batch["block_table"], batch["kv_len"], batch["max_kv_len"], row_start=ints(start), max_rows=max(max(total), 1))
    return bounds


BOUNDS = [([1, 1], [0, 15], 16, 1, 16), ([1, 3, 40], [700, 62, 5], 64, 8, 128), ([5, 1], [60, 333], 32, 5, 80), ([1, 2], [500, 1000], 256, 2, 256),
          ([1], [1023], 1024, 3, 48), ([130], [70], 128, 1, 64)]


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("case", range(len(BOUNDS)))
def test_page_bounds(case, token_major):
    new, past, page, heads, dim = BOUNDS[case]
    batch, total = lm_checks.make_batch(new, past, page, heads, dim, seed=case, token_major=token_major)
    k, _, ks, _ = batch["cache"]
    bounds = lm.new_bounds(batch["cache"])
    bounds[0].fill_(77)
    lm.page_bounds(batch["cache"], bounds, **batch_only(batch))
    host, touched = k.cpu(), set()
    for b, n in enumerate(new):
        for c in range((total[b] - n) // page, (total[b] - 1) // page + 1):
            at = int(batch["block_table"][b, c])
            touched.add(at)
            lo_hi, unit = ref.page_bounds(host, ks.cpu(), at, min(page, total[b] - c * page))
            assert torch.equal(bounds[0][at].cpu().double(), lo_hi) and torch.equal(bounds[1][at].cpu().double(), unit)
    rest = [p for p in range(k.shape[0]) if p not in touched]
    assert bool((bounds[0][rest] == 77).all()) and bool((bounds[1][rest] == 0).all())


def batch_only(batch):
    return {k: v for k, v in batch.items() if k != "cache"}


def test_bounds_of_nan_and_of_pages_of_zeros():
    batch, total = lm_checks.make_batch([40], [0], 16, 2, 32)
    k, _, ks, _ = batch["cache"]
    at = batch["block_table"][0]
    raw = k.view(torch.uint8)
    raw[at[0], 0, 3] = 0x7f                                  # one key
    raw[at[0], 1, :, 5] = 0xff                               # one element of all keys
    raw[at[1]] = 0x7f
    raw[at[2], 1] = 0x80
    ks[at[2], 1] = 0
    bounds = lm.new_bounds(batch["cache"])
    lm.page_bounds(batch["cache"], bounds, **batch_only(batch))
    for c, tokens in ((0, 16), (1, 16), (2, 8)):
        lo_hi, unit = ref.page_bounds(k.cpu(), ks.cpu(), int(at[c]), tokens)
        assert torch.equal(bounds[0][at[c]].cpu().double(), lo_hi) and torch.equal(bounds[1][at[c]].cpu().double(), unit)


def check_choice(q, batch, total, new, bounds, count, first=1, last=1):
    chosen = lm.choose_pages(q, batch["cache"], bounds, count=count, first=first, last=last, **batch_only(batch)).cpu()
    lo_hi, unit, table = bounds[0].cpu(), bounds[1].cpu(), batch["block_table"].cpu()
    page, kv_heads = batch["cache"][0].shape[2], batch["cache"][0].shape[1]
    pages, group, row = batch["cache"][0].shape[0], q.shape[1] // kv_heads, 0
    for b, n in enumerate(new):
        here = torch.where((table[b] >= 0) & (table[b] < pages), table[b], -1)
        for r in range(n):
            own = (total[b] - n + r) // page if total[b] - n + r >= 0 else -1
            for h in range(kv_heads):
                want = ref.choose_row(q[row, h * group:(h + 1) * group].cpu(), lo_hi[:, h], unit[:, h], here, own, count, first, last)
                assert chosen[row, h].tolist() == want, (b, r, h)
            row += 1


CHOICES = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, count, first, last
    ([1], [0], 16, 1, 1, 16, 1, 0, 1),
    ([1], [700], 64, 32, 8, 128, 4, 1, 1),
    ([1, 1, 1, 1], [0, 15, 16, 1000], 16, 8, 2, 64, 8, 1, 2),
    ([1, 1], [4000, 130], 16, 16, 1, 128, 16, 2, 3),
    ([3, 1, 20], [300, 900, 61], 16, 6, 2, 80, 5, 1, 1),      # three heads to one: five rows to a tile
    ([40], [500], 32, 2, 2, 256, 7, 0, 2),                    # one head to one: sixteen rows
    ([2, 1], [400, 30], 16, 40, 2, 48, 3, 1, 1),              # twenty heads to one
    ([1, 5], [6000, 5000], 16, 4, 4, 64, 64, 1, 1),           # more than 256 pages
    ([2], [2000], 16, 120, 1, 96, 12, 1, 1),
    ([1, 1, 1], [4080, 4064, 4095], 16, 8, 2, 64, 100, 1, 1),        # 256 pages, one less, one more
    ([2, 4, 1], [300, 1000, 7], 16, 20, 1, 80, 9, 1, 1),      # a row to a tile, few pages
    ([4, 4], [500, 200], 64, 4, 1, 128, 3, 1, 1),             # four rows to a tile
    ([1, 2], [700, 90], 16, 256, 1, 256, 5, 1, 1),
    ([1], [140000], 16, 2, 1, 16, 96, 1, 1),                  # more than 8192 pages
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(CHOICES)))
def test_choose_pages(case, dtype):
    new, past, page, heads, kv_heads, dim, count, first, last = CHOICES[case]
    batch, total = lm_checks.make_batch(new, past, page, kv_heads, dim, seed=case)
    bounds = with_bounds(batch, total)
    q = torch.randn(sum(new), heads, dim, generator=torch.Generator().manual_seed(case)).to(dtype).cuda()
    check_choice(q, batch, total, new, bounds, count, first, last)


def test_choices_among_equal_scores_missing_pages_and_strange_queries():
    new, past = [2, 3, 1], [3000, 6000, 90]
    batch, total = lm_checks.make_batch(new, past, 16, 2, 64)
    bounds = with_bounds(batch, total)
    table = batch["block_table"]
    table[0, 5:40] = -1
    table[0, 187] = -1                                        # the rows' own
    table[1, ::3] = 10 ** 6
    bounds[0][table[1, 1:300:3].long()] = bounds[0][table[1, 1].long()].clone()
    bounds[1][table[1, 1:300:3].long()] = bounds[1][table[1, 1].long()].clone()
    q = torch.randn(6, 6, 64, generator=torch.Generator().manual_seed(1)).cuda()
    q[0, 0, 3], q[0, 4, :5], q[1], q[4, 2:] = math.inf, math.nan, 0, 1e-42
    check_choice(q, batch, total, new, bounds, 9)
    check_choice(q, batch, total, new, bounds, 150, first=3, last=20)


def test_choices_of_rows_before_the_text_and_of_none():
    batch, total = lm_checks.make_batch([4, 1, 0, 2], [60, 0, 9, 200], 16, 2, 64)
    bounds = with_bounds(batch, total)
    batch["kv_len"][0] = 2                                    # of four rows two stand before the text
    batch["kv_len"][1] = 0
    q = torch.randn(7 + 3, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()      # and three rows that no sequence has
    room = torch.full((10, 2, 6), 99, dtype=torch.int32, device="cuda")
    got = lm.choose_pages(q, batch["cache"], bounds, count=6, **batch_only(batch))
    assert bool((got[:2] == -1).all()) and got[2:4, :, 0].eq(0).all() and bool((got[2:4, :, 1:] == -1).all()) and bool((got[4] == -1).all())
    table = batch["block_table"].cpu()
    for r in (5, 6):
        want = ref.choose_row(q[r, :2].cpu(), bounds[0][:, 0].cpu(), bounds[1][:, 0].cpu(), table[3].tolist(), (200 + r - 5) // 16, 6, 1, 1)
        assert got[r, 0].tolist() == want
    del room


def test_choices_in_more_than_one_launch():
    """More scores than are kept at a time: tables whose pages are few, but for some at their ends."""
    blocks, rows, kv_heads = 1 << 17, 300, 2
    batch, total = lm_checks.make_batch([1] * 3, [300, 200, 100], 16, kv_heads, 16)
    bounds = with_bounds(batch, total)
    table = torch.full((1, blocks), -1, dtype=torch.int32)
    table[0, 5:20] = batch["block_table"][0, :15].cpu()
    table[0, blocks - 40:blocks - 30] = batch["block_table"][1, :10].cpu()
    big = dict(cache=batch["cache"], block_table=table.cuda(), kv_len=ints([blocks * 16 - 100]), max_kv_len=blocks * 16, row_start=ints([0, rows]), max_rows=rows)
    q = torch.randn(rows, 4, 16, generator=torch.Generator().manual_seed(1)).cuda()
    check_choice(q, big, [blocks * 16 - 100], [rows], bounds, 4)


# ------------------------------------------------------------------------------------------------------ attention over chosen pages
def random_choice(new, total, page, kv_heads, count, seed=0, own=True):
    r = random.Random(seed)
    rows = []
    for b, n in enumerate(new):
        for i in range(n):
            mine = (total[b] - n + i) // page
            row = []
            for _ in range(kv_heads):
                some = set(r.sample(range(mine + 1), min(mine + 1, r.choice([count, count, max(1, count // 2)]))))
                if own:
                    some = set(sorted(some)[:count - 1]) | {mine}
                row.append(sorted(some) + [-1] * (count - len(some)))
            rows.append(row)
    return ints(rows)


SPARSE = [
    # new rows, earlier tokens, page, q heads, kv heads, dim, count
    ([1], [0], 16, 1, 1, 16, 1),
    ([1], [7000], 64, 32, 8, 128, 16),
    ([1, 1, 1, 1], [0, 15, 16, 1000], 16, 8, 2, 64, 5),
    ([1] * 9, [3, 63, 64, 65, 127, 511, 2047, 0, 300], 64, 8, 8, 128, 3),
    ([1, 1], [130, 4000], 128, 16, 1, 128, 4),
    ([1, 1, 1], [77, 300, 5], 32, 15, 5, 80, 6),
    ([1, 1], [260, 1029], 256, 6, 2, 256, 2),
    ([5, 3, 5], [0, 62, 1500], 32, 8, 4, 256, 9),             # drafts: some rows to a tile
    ([3, 1, 7, 2], [10, 900, 61, 0], 16, 8, 2, 64, 7),
    ([40, 1, 17], [300, 333, 100], 16, 8, 8, 128, 12),        # a head to a head: sixteen rows to a tile
    ([35], [600], 16, 4, 4, 96, 33),
    ([12], [400], 16, 40, 2, 64, 6),                          # twenty heads to one: tiles that begin inside a row
    ([1, 1], [2000, 50], 16, 80, 1, 128, 30),
    ([70, 64], [500, 900], 32, 8, 2, 128, 10),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(SPARSE)))
def test_sparse_attention(case, dtype):
    new, past, page, heads, kv_heads, dim, count = SPARSE[case]
    batch, total = lm_checks.make_batch(new, past, page, kv_heads, dim, seed=case)
    q = (1.5 * torch.randn(sum(new), heads, dim, generator=torch.Generator().manual_seed(case))).to(dtype).cuda()
    chosen = random_choice(new, total, page, kv_heads, count, seed=case)
    got = lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch))
    lm_checks.check_attention(got, ref.sparse64(q, batch, total, new, chosen), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new,past,page,heads,kv_heads,dim,count", [
    ([1], [12000], 128, 16, 4, 96, 79), ([1, 1, 1], [9000, 77, 0], 64, 16, 1, 128, 90), ([1], [5000], 64, 4, 2, 256, 60),
    ([1, 1], [7000, 6500], 128, 16, 4, 64, 47), ([3, 1], [8000, 8000], 64, 20, 2, 64, 64), ([4, 2], [6000, 30], 32, 8, 1, 128, 100)])
def test_sparse_attention_of_few_rows_over_many_pages(new, past, page, heads, kv_heads, dim, count, dtype):
    batch, total = lm_checks.make_batch(new, past, page, kv_heads, dim, seed=21)
    q = torch.randn(sum(new), heads, dim, generator=torch.Generator().manual_seed(22)).to(dtype).cuda()
    chosen = random_choice(new, total, page, kv_heads, count, seed=23)
    got = lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch))
    lm_checks.check_attention(got, ref.sparse64(q, batch, total, new, chosen), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sparse_attention_over_all_pages_is_attention(dtype):
    new, past, page = [1, 4, 30], [900, 333, 20], 16
    batch, total = lm_checks.make_batch(new, past, page, 2, 64)
    q = torch.randn(sum(new), 8, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    chosen = torch.arange(60, dtype=torch.int32).repeat(sum(new), 2, 1).cuda()
    got = lm.sparse_attention(q, batch["cache"], chosen, scale=0.2, **batch_only(batch))
    lm_checks.check_attention(got, lm_checks.attention64(q, batch, total, new, scale=0.2), dtype)


@pytest.mark.parametrize("new", [[1, 1], [6, 5], [40, 33]])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_what_is_not_chosen_does_not_reach_a_row(dtype, new):
    """NaN, huge scales and missing pages among what a row has not chosen; rows that have chosen nothing."""
    past, page = [700, 300], 16
    batch, total = lm_checks.make_batch(new, past, page, 2, 64)
    rows = sum(new)
    chosen = random_choice(new, total, page, 2, 6, seed=3)
    k, v, ks, vs = batch["cache"]
    table = batch["block_table"]
    # two pages that the even rows may have and the odd ones have not
    odd = torch.arange(rows, device="cuda") % 2 == 1
    for b, c in ((0, 10), (1, 4)):
        at = int(table[b, c])
        v.view(torch.uint8)[at, :, 3] = 0x7f
        k.view(torch.uint8)[at, :, 5] = 0xff
        ks[at] = 2.0 ** 60
    kept = [[[c for c in row if c not in (10, 4)] if odd[i] else row for row in rows_] for i, rows_ in enumerate(chosen.tolist())]
    chosen = ints([[row + [-1] * (6 - len(row)) for row in rows_] for rows_ in kept])
    chosen[rows - 1] = -1
    table[1, 2] = -1
    q = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    got = lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch))
    want = ref.sparse64(q, batch, total, new, chosen)
    clean = odd.cpu()
    clean[rows - 1] = True
    lm_checks.check_attention([t[clean.cuda()] for t in got], (want[0][clean], want[1][clean], want[2]), dtype)
    assert bool((got[0][rows - 1] == 0).all()) and bool((got[1][rows - 1] == -math.inf).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [[1] * 80, [6] * 30])
def test_nan_among_many_pages(new, dtype):
    """More steps of a warp than it looks up at once; a few texts have NaN among the values of pages that they, or some of their rows, chose."""
    page, kv_heads = 64, 8
    batch, total = lm_checks.make_batch(new, [4000] * len(new), page, kv_heads, 16)
    q = torch.randn(sum(new), 16, 16, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    chosen = random_choice(new, total, page, kv_heads, 50, seed=4)
    v, table = batch["cache"][1].view(torch.uint8), batch["block_table"].tolist()
    for b, c, token, element in ((0, 3, 5, 2), (2, 40, 63, 0), (2, 41, 0, 15), (7, 62, 1, 9)):
        v[table[b][c], :, token, element] = 0x7f
    lm_checks.check_attention(lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch)), ref.sparse64(q, batch, total, new, chosen), dtype)


def test_rows_that_stand_before_the_text_or_are_nobodys():
    batch, total = lm_checks.make_batch([4, 1, 2], [60, 0, 200], 16, 2, 64)
    batch["kv_len"][0] = 2
    batch["kv_len"][1] = 0
    q = torch.randn(7 + 3, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    chosen = torch.arange(13, dtype=torch.int32).repeat(10, 2, 1).cuda()
    out = torch.full((10, 4, 64), 5.0, device="cuda")
    got, lse = lm.sparse_attention(q, batch["cache"], chosen, out=out, **batch_only(batch))
    assert bool((got[[0, 1, 4]] == 0).all()) and bool((lse[[0, 1, 4]] == -math.inf).all()) and bool((got[7:] == 5).all())
    want, lse_want = lm.attention(q, batch["cache"], **batch_only(batch))
    assert torch.allclose(got[[2, 3, 5, 6]], want[[2, 3, 5, 6]], atol=1e-4) and torch.allclose(lse[[2, 3, 5, 6]], lse_want[[2, 3, 5, 6]], atol=1e-4)


def test_strides_of_queries_choices_and_results():
    new, past = [3, 2], [200, 50]
    batch, total = lm_checks.make_batch(new, past, 16, 2, 64, token_major=True)
    wide = torch.randn(5, 9, 96, generator=torch.Generator().manual_seed(1)).cuda()
    q, chosen = wide[:, 2:6, 16:80], random_choice(new, total, 16, 2, 4)
    room = torch.full((5, 3, 9), 10 ** 6, dtype=torch.int32, device="cuda")
    room[:, 1:, 2:6] = chosen
    out = torch.zeros(5, 8, 128, device="cuda")[:, 1:5, 32:96]
    got = lm.sparse_attention(q, batch["cache"], room[:, 1:, 2:6], out=out, **batch_only(batch))
    assert got[0].data_ptr() == out.data_ptr()
    lm_checks.check_attention(got, ref.sparse64(q, batch, total, new, chosen), F32)
    bounds = with_bounds(batch, total)
    check_choice(q, batch, total, new, bounds, 4)


@pytest.mark.parametrize("rows", [1, 30])
def test_a_wait_that_runs_out_is_reported(rows):
    lib = _lib.cuda_lib()
    batch, total = lm_checks.make_batch([rows], [500], 16, 2, 64)
    q = torch.randn(rows, 4, 64).cuda()
    chosen = random_choice([rows], total, 16, 2, 8)
    lib.ogle_cuda_set_wait_limit(0)
    try:
        lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch))
        assert lib.ogle_cuda_device_status() == -6
    finally:
        lib.ogle_cuda_set_wait_limit(-1)
        lib.ogle_cuda_clear_device_status()
    got = lm.sparse_attention(q, batch["cache"], chosen, **batch_only(batch))
    lm_checks.check_attention(got, ref.sparse64(q, batch, total, [rows], chosen), F32)
    assert lib.ogle_cuda_device_status() == 0


# ------------------------------------------------------------------------------------------------------ together
def search_step(s):
    """A step of a search over chosen pages, all of it on the device."""
    table, kv_len, refs, copies, state = lm.advance_pages(s["table"], s["kv_len"], s["parent"], 1, s["refs"], 16)
    lm.copy_pages([s["cache"]], copies, bounds=[s["bounds"]])
    batch = dict(block_table=table, kv_len=kv_len, max_kv_len=s["most"])
    q = lm.append(s["k"], s["v"], s["cache"], q=s["q"], **batch)
    lm.page_bounds(s["cache"], s["bounds"], **batch)
    chosen = lm.choose_pages(q, s["cache"], s["bounds"], count=3, **batch)
    out, lse = lm.sparse_attention(q, s["cache"], chosen, **batch)
    logits = out.flatten(1) @ s["words"]
    found = lm.beam_step(logits, s["scores"], 4, 8)
    packed = lm.compact_pages(table, refs, 10, 16)
    return (table, kv_len, refs, copies, state, chosen, out, lse, *found, *packed)


def search_state(seed):
    g = torch.Generator().manual_seed(seed)
    cache = lm.new_cache(60, 2, 16, 64)
    table, kv_len = torch.full((8, 6), -1, dtype=torch.int32), torch.tensor([70, 70, 70, 70, 33, 33, 33, 33], dtype=torch.int32)
    table[:4, :4], table[4:, :2] = torch.arange(4, dtype=torch.int32), torch.arange(4, 6, dtype=torch.int32)
    for i in range(4):
        table[i, 4], table[4 + i, 2] = 20 + i, 30 + i
    refs = torch.bincount(table[table >= 0].long(), minlength=60).int()
    rows = [torch.randn(8, n, 64, generator=g).cuda() for n in (2, 2, 4)]
    return dict(cache=cache, bounds=lm.new_bounds(cache), table=table.cuda(), kv_len=kv_len.cuda(), refs=refs.cuda(), most=96, k=rows[0], v=rows[1], q=rows[2],
                parent=ints([0, 0, 2, 1, 4, -1, 7, 7]), scores=-torch.rand(8, generator=g).cuda(), words=torch.randn(256, 500, generator=g).cuda())


def test_a_captured_search_is_replayed_with_other_inputs():
    s, other = search_state(1), search_state(2)
    other["parent"], other["kv_len"] = ints([3, 3, 3, 0, 5, 4, 5, -1]), ints([70, 65, 80, 66, 32, 47, 33, 40])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        search_step(search_state(1))
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured = search_step(s)
    for inputs in (other, search_state(3), other):
        plain = {k: tuple(x.clone() for x in v) if isinstance(v, tuple) else v.clone() if isinstance(v, torch.Tensor) else v for k, v in inputs.items()}
        for k in s:
            if isinstance(s[k], tuple):
                for a, b in zip(s[k], inputs[k]):
                    a.view(torch.uint8).copy_(b.view(torch.uint8)) if a.dtype == torch.float8_e4m3fn else a.copy_(b)
            elif isinstance(s[k], torch.Tensor):
                s[k].copy_(inputs[k])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, search_step(plain)):
            assert torch.equal(a, b)


def test_two_searches_at_once_on_two_streams():
    alone = [search_step(search_state(i)) for i in (5, 6)]
    streams, states = [torch.cuda.Stream() for _ in range(2)], [search_state(i) for i in (5, 6)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for stream, state in zip(streams, states):
            with torch.cuda.stream(stream):
                fresh = {k: tuple(x.clone() for x in v) if isinstance(v, tuple) else v for k, v in state.items()}
                got.append(search_step(fresh))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def prompts_of(lengths, vocab, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, vocab, (n,), generator=g).tolist() for n in lengths]


def check_pages(search):
    """The counts are what the table says, and no page that a text writes to is another's."""
    table, refs, page = search.table.tolist(), search.refs.tolist(), search.page_tokens
    assert refs == counts([table], len(refs))
    for row, n in zip(table, search.kv_len.tolist()):
        assert all(p >= 0 for p in row[:-(-n // page)]) and all(p == -1 for p in row[-(-n // page):])
        if n % page:
            assert refs[row[n // page]] == 1


@pytest.mark.parametrize("chosen", [0, 3])
def test_search_scores_are_those_of_the_whole_texts(chosen):
    """The score of every text that a search has found is the sum of its tokens' log probabilities when it is read as one prompt; and no text of
    the same length that its step could have had instead scores higher than what was kept."""
    model = lm_example.Model(layers=2, chosen=chosen)
    search = lm_example.Search(model, prompts_of([37, 5, 64], model.vocab), 4, pages=120, ends=(7, 11), steps=25)
    for step in range(20):
        search.step()
        check_pages(search)
        if step % 6 == 5:
            while int(search.compact(5)[1]):
                pass
            check_pages(search)
    left, ended = search.texts()
    assert all(len(t) == 4 for t in left)
    texts = [(g, score, text) for kind in (left, ended) for g, found in enumerate(kind) for score, text in found]
    for g, score, text in texts:
        prompt = search.prompts[g]
        whole = lm_example.Search(model, [prompt + text], 1, pages=40, steps=1)      # fills a cache of its own
        rows = len(prompt) + len(text)
        batch = dict(block_table=whole.table, kv_len=whole.kv_len, max_kv_len=whole.most, row_start=ints([0, rows]), max_rows=rows)
        x = model.rows(torch.tensor(prompt + text).cuda(), whole.caches, batch, whole.bounds)
        logits = torch.log_softmax(model.logits(x).double(), 1)
        at = torch.arange(len(prompt) - 1, rows - 1, device="cuda")
        want = float(logits[at, torch.tensor(text).cuda()].sum())
        # A value that was stored under a smaller scale first may be another one of the 8-bit numbers, rounded twice, and pages are chosen by them.
        # What this looks for - a page that is another text's, a copy that was not made - moves a score by units.
        assert abs(score - want) <= 0.05 * len(text), (score, want)


def test_search_with_one_beam_takes_the_likeliest_tokens():
    model = lm_example.Model(layers=1)
    prompts = prompts_of([20, 3, 33], model.vocab)
    search = lm_example.Search(model, prompts, 1, steps=30)
    answers = lm_example.Answers(model, prompts, repetition=1.0, presence=0.0, frequency=0.0, forbidden=())
    for _ in range(15):
        search.step()
    for _ in range(16):
        answers.step()
    assert [found[0][1] for found in search.texts()[0]] == [t[n:] for t, n in zip(answers.texts, answers.prompt_len)]


def test_search_without_enough_pages_says_so():
    model = lm_example.Model(layers=1)
    search = lm_example.Search(model, prompts_of([30, 30], model.vocab), 4, pages=9, steps=30)
    for _ in range(20):
        search.step()
    with pytest.raises(RuntimeError):
        search.texts()


def test_offsets_beyond_32_bits():
    """Pages more than 2 GB apart: bounds, choice, attention and copies as over a packed cache."""
    new, past = [1, 5], [70, 40]
    batch, total = lm_checks.make_batch(new, past, 16, 2, 64)
    k, v, ks, vs = batch["cache"]
    apart, pages = (1 << 31) + 4096, k.shape[0]
    assert pages <= 12
    room = torch.empty(apart * (pages - 1) + 4096, dtype=torch.uint8, device="cuda")
    far = [room[i * 2048:].as_strided(k.shape, (apart, 1024, 64, 1)).view(torch.float8_e4m3fn) for i in range(2)]
    for a, b in zip(far, (k, v)):
        a.view(torch.uint8).copy_(b.view(torch.uint8))
    cache, rest = (*far, ks, vs), batch_only(batch)
    bounds = with_bounds(batch, total)
    got = lm.new_bounds(cache)
    start = ints([0, total[0], sum(total)])
    lm.page_bounds(cache, got, rest["block_table"], rest["kv_len"], rest["max_kv_len"], row_start=start, max_rows=max(total))
    assert torch.equal(got[0], bounds[0]) and torch.equal(got[1], bounds[1])
    q = torch.randn(6, 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    chosen = lm.choose_pages(q, cache, bounds, count=3, **rest)
    lm_checks.check_attention(lm.sparse_attention(q, cache, chosen, **rest), ref.sparse64(q, batch, total, new, chosen), F32)
    copies = ints([(0, pages - 1, 16), (1, pages - 2, 5)])
    lm.copy_pages([cache], copies, bounds=[bounds])
    lm.copy_pages([(k, v, ks.clone(), vs.clone())], copies)
    for a, b in zip(far, (k, v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_step_of_nothing(dtype):
    got = lm.beam_step(torch.empty(4, 0, dtype=dtype, device="cuda"), None, 2, 3)
    assert got[0].shape == (2, 3) and bool((got[1] == -1).all()) and got[3].tolist() == [-1] * 4 and bool((got[5] == -math.inf).all())
    got = lm.beam_step(torch.empty(0, 10, dtype=dtype, device="cuda"), None, 2, 3)
    assert got[0].shape == (0, 3) and got[3].shape == (0,)


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    batch, total = lm_checks.make_batch([1, 1], [50, 20], 16, 2, 64)
    cache, rest = batch["cache"], batch_only(batch)
    bounds, q, one = lm.new_bounds(cache), torch.randn(2, 4, 64).cuda(), ints([1, 1])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: lm.beam_step(torch.zeros(2, 9, device="cuda:0"), None, 2, 4), lambda: lm.advance_pages(rest["block_table"], rest["kv_len"], one, 1, one, 16),
                 lambda: lm.compact_pages(rest["block_table"], one, 4, 16), lambda: lm.copy_pages([cache], torch.zeros(1, 3, dtype=torch.int32, device="cuda:0")),
                 lambda: lm.page_bounds(cache, bounds, **rest), lambda: lm.choose_pages(q, cache, bounds, **rest),
                 lambda: lm.sparse_attention(q, cache, torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda:0"), **rest)):
        with pytest.raises(ValueError):
            call()


def test_bounds_under_bounds_that_are_far_too_wide():
    """max_rows and max_kv_len say more than 2^30 rows x heads; a batch of few rows of many possible ones."""
    new, past = [5, 1, 0], [40, 700, 3]
    batch, total = lm_checks.make_batch(new, past, 16, 2, 64)
    want, got = lm.new_bounds(batch["cache"]), lm.new_bounds(batch["cache"])
    lm.page_bounds(batch["cache"], want, **batch_only(batch))
    wide = batch_only(batch)
    wide["block_table"] = torch.cat([wide["block_table"], torch.full((3, 5000), -1, dtype=torch.int32, device="cuda")], 1)
    wide["max_rows"], wide["max_kv_len"] = 400000, 80000
    lm.page_bounds(batch["cache"], got, **wide)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(1)).cuda()
    bounds = with_bounds(batch, total)
    narrow = lm.choose_pages(q, batch["cache"], bounds, count=5, **batch_only(batch))
    wide["max_rows"] = 40
    assert torch.equal(narrow, lm.choose_pages(q, batch["cache"], bounds, count=5, **wide))
    a, b = lm.sparse_attention(q, batch["cache"], narrow, **batch_only(batch)), lm.sparse_attention(q, batch["cache"], narrow, **wide)
    lm_checks.check_attention(a, ref.sparse64(q, batch, total, new, narrow), F32)
    lm_checks.check_attention(b, ref.sparse64(q, batch, total, new, narrow), F32)


def test_nothing_waited_in_vain():
    assert _lib.cuda_lib().ogle_cuda_device_status() == 0


# ------------------------------------------------------------------------------------------------------ batches of other shapes
def check_bounds(batch, total, new, most, bounds, row_start):
    """The bounds of the pages that the first `most` rows of each sequence were appended to, and of no other."""
    k, _, ks, _ = batch["cache"]
    page = k.shape[2]
    lm.page_bounds(batch["cache"], bounds, batch["block_table"], batch["kv_len"], batch["max_kv_len"], row_start=row_start, max_rows=most)
    touched = set()
    for b, n in enumerate(new):
        begin = total[b] - n
        for c in range(begin // page, (begin + min(n, most) - 1) // page + 1) if n else ():
            at = int(batch["block_table"][b, c])
            touched.add(at)
            lo_hi, unit = ref.page_bounds(k.cpu(), ks.cpu(), at, min(page, total[b] - c * page))
            assert torch.equal(bounds[0][at].cpu().double(), lo_hi) and torch.equal(bounds[1][at].cpu().double(), unit), (b, c)
    rest = [p for p in range(k.shape[0]) if p not in touched]
    assert bool((bounds[0][rest] == 77).all())


@pytest.mark.parametrize("new,past,most,before", [
    ([1, 1, 1, 1], [40, 15, 16, 0], 1, 8),                   # rows that no sequence has, before the first
    ([5, 1, 20], [30, 100, 0], 20, 1000),
    ([100, 1], [3, 50], 10, 0),                              # more rows than max_rows
    ([33, 40, 2, 0, 17], [0, 16, 31, 9, 200], 16, 0),
    ([70, 70], [10, 300], 33, 5)])
def test_bounds_of_batches_whose_rows_lie_anywhere(new, past, most, before):
    batch, total = lm_checks.make_batch(new, past, 16, 2, 64)
    bounds = lm.new_bounds(batch["cache"])
    bounds[0].fill_(77)
    check_bounds(batch, total, new, most, bounds, batch["row_start"] + before)


def test_choices_behind_append_of_more_rows_than_count():
    """append and page_bounds with one batch that begins behind rows which nobody has, and whose sequences have more rows than max_rows; the pages that got
    large keys are then the next token's choice."""
    new, past, page, most, before = [90, 1, 70], [100, 200, 500], 16, 12, 6
    batch, total = lm_checks.make_batch(new, past, page, 2, 64)
    bounds = with_bounds(batch, total)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(before + sum(new), 2, 64, generator=g).cuda() for _ in range(2))
    call = dict(batch_only(batch), row_start=batch["row_start"] + before, max_rows=most)
    lm.append(30 * k, v, batch["cache"], **call)
    lm.page_bounds(batch["cache"], bounds, **call)
    q = torch.randn(3, 4, 64, generator=g).cuda()
    chosen = lm.choose_pages(q, batch["cache"], bounds, batch["block_table"], batch["kv_len"], batch["max_kv_len"], count=4).cpu()
    keys, scales, table = batch["cache"][0].cpu(), batch["cache"][2].cpu(), batch["block_table"].cpu()
    for b in range(3):
        own, pages = (total[b] - 1) // page, table[b].tolist()
        for h in range(2):
            lo_hi, unit = torch.zeros(keys.shape[0], 2, 64), torch.zeros(keys.shape[0], dtype=torch.float64)
            for c in range(own + 1):
                found, size = ref.page_bounds(keys, scales, pages[c], min(page, total[b] - c * page))
                lo_hi[pages[c]], unit[pages[c]] = found[h].float(), size[h]
            want = ref.choose_row(q[b, 2 * h:2 * h + 2].cpu(), lo_hi, unit, table[b], own, 4, 1, 1)
            assert chosen[b, h].tolist() == want, (b, h)
            if new[b] > most:
                assert past[b] // page + 1 in want or past[b] // page in want


# ------------------------------------------------------------------------------------------------------ the example's ends
def test_search_ends_texts_at_their_first_token():
    model = lm_example.Model(layers=1)
    prompts, beams = prompts_of([20, 3], model.vocab), 3
    plain = lm_example.Search(model, prompts, beams, steps=4)
    first, score = (t.view(2, beams)[:, 0].tolist() for t in plain.next[1:])
    search = lm_example.Search(model, prompts, beams, ends=sorted(set(first)), steps=4)
    for _ in range(4):
        search.step()
    left, ended = search.texts()
    for g in range(2):
        assert any(text == [first[g]] and abs(s - score[g]) < 1e-5 for s, text in ended[g])
        assert len(left[g]) == beams and all(not set(text) & set(first) for _, text in left[g])
        assert all(text[-1] in first and not set(text[:-1]) & set(first) for _, text in ended[g])


def test_search_with_many_end_tokens_keeps_its_beams():
    model = lm_example.Model(layers=1)
    search = lm_example.Search(model, prompts_of([20, 3, 9], model.vocab), 2, ends=range(0, model.vocab, 2), steps=12)
    for _ in range(12):
        search.step()
    left, ended = search.texts()
    assert all(len(found) == 2 for found in left) and all(t % 2 for found in left for _, text in found for t in text)
    assert all(text[-1] % 2 == 0 and all(t % 2 for t in text[:-1]) for found in ended for _, text in found)


def test_search_refuses_a_step_too_many():
    model = lm_example.Model(layers=1)
    search = lm_example.Search(model, prompts_of([20, 3], model.vocab), 2, steps=5)
    for _ in range(5):
        search.step()
    before = search.texts()
    with pytest.raises(ValueError):
        search.step()
    assert search.texts() == before


# ------------------------------------------------------------------------------------------------------ several callers
def test_choices_of_two_threads_with_queries_of_different_sizes():
    """Two host threads, each on a stream of its own, whose queries take 64 and 128 KB of shared memory."""
    import threading
    calls, failed = [], []
    for group, seed in ((128, 1), (256, 2)):
        batch, total = lm_checks.make_batch([1, 1], [5000, 300], 16, 1, 256, seed=seed)
        bounds = with_bounds(batch, total)
        q = torch.randn(2, group, 256, generator=torch.Generator().manual_seed(seed)).cuda()
        calls.append(lambda q=q, batch=batch, bounds=bounds: lm.choose_pages(q, batch["cache"], bounds, count=5, **batch_only(batch)))
    alone = [c() for c in calls]
    torch.cuda.synchronize()

    def many(call, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got = [call() for _ in range(400)]
            stream.synchronize()
            assert all(torch.equal(g, want) for g in got)
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=many, args=a) for a in zip(calls, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


class OfAnotherDevice(torch.Tensor):
    """Says that it lies on device 1; its memory is the current one's."""
    def get_device(self):
        return 1


def elsewhere(t):
    return t.as_subclass(OfAnotherDevice)


def test_every_tensor_of_another_device_is_refused():
    batch, total = lm_checks.make_batch([1, 1], [50, 20], 16, 2, 64)
    cache, bounds = batch["cache"], with_bounds(batch, total)
    q, one = torch.randn(2, 4, 64).cuda(), ints([1, 1])
    chosen, copies = ints([[[0, -1]] * 2] * 2), ints([[-1, -1, 0]])
    named = dict(block_table=batch["block_table"], kv_len=batch["kv_len"], row_start=batch["row_start"])
    most = dict(max_kv_len=batch["max_kv_len"], max_rows=1)
    calls = [
        (lambda logits, scores, ends: lm.beam_step(logits, scores, 2, 4, ends=ends), dict(logits=torch.zeros(2, 9, device="cuda"), scores=torch.zeros(2, device="cuda"), ends=one)),
        (lambda **t: lm.advance_pages(page_tokens=16, **t), dict(block_table=batch["block_table"], kv_len=one, parent=one, new=one, refs=ints([1] * 8))),
        (lambda **t: lm.compact_pages(most=1, page_tokens=16, **t), dict(block_table=batch["block_table"], refs=ints([1] * 8))),
        (lambda copies, k, v, ks, vs, lo_hi, unit: lm.copy_pages([cache, (k, v, ks, vs)], copies, bounds=[bounds, (lo_hi, unit)]),
         dict(copies=copies, k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], lo_hi=bounds[0], unit=bounds[1])),
        (lambda k, v, ks, vs, lo_hi, unit, **t: lm.page_bounds((k, v, ks, vs), (lo_hi, unit), **t, **most),
         dict(k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], lo_hi=bounds[0], unit=bounds[1], **named)),
        (lambda q, k, v, ks, vs, lo_hi, unit, **t: lm.choose_pages(q, (k, v, ks, vs), (lo_hi, unit), count=2, **t, **most),
         dict(q=q, k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], lo_hi=bounds[0], unit=bounds[1], **named)),
        (lambda q, k, v, ks, vs, chosen, out, **t: lm.sparse_attention(q, (k, v, ks, vs), chosen, out=out, **t, **most),
         dict(q=q, k=cache[0], v=cache[1], ks=cache[2], vs=cache[3], chosen=chosen, out=torch.zeros_like(q), **named))]
    for call, tensors in calls:
        call(**tensors)
        for name in tensors:
            with pytest.raises(ValueError):
                call(**{**tensors, name: elsewhere(tensors[name])})
                pytest.fail(f"{name} of {call}")
