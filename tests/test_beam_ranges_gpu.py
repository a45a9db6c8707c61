"""lm.beam_step where a block goes over several batches of a row (many rows): masks, steps and logits of any size in the later ones."""
import math

import pytest
import torch

import search_checks as ref
from ogle_b200 import lm

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SMS = 148


def batches_of_a_range(rows, vocab, dtype):
    """As csrc/kernels/beam.cu shares a row out: batches of 4 x 16 bytes for each of 256 threads, three blocks to an SM."""
    batch = 4096 if dtype == F32 else 8192
    batches = -(-(vocab + (3 if dtype == F32 else 7)) // batch)
    return -(-batches // max(3 * SMS // rows, 1)), batch


def check(got, want):
    assert not any(bool(torch.isnan(got[i]).any()) for i in (0, 5))
    ref.check_beam_step(got, want)


def masked_until(n, value, size, every=1):
    """A mask of `value` up to token n, and of all but every so-many-th behind it; the others ordinary logits about `size`."""
    def fill(x, lowest):
        masked = torch.arange(len(x)) % every != 0
        masked[:n] = True
        x += size
        x[masked] = lowest if value == "lowest" else value
    return fill


def stepped(height, wide):
    def fill(x, lowest):
        x += height * (torch.arange(len(x)) // wide).float()
    return fill


def few(tokens):
    def fill(x, lowest):
        x[:] = -math.inf
        for t, value in tokens.items():
            x[t] = value
    return fill


def at(tokens, value):
    def fill(x, lowest):
        x[tokens] = value
    return fill


def all_alike(x, lowest):
    x[:] = 3.0


def two_sizes(x, lowest):
    x[:] = torch.where(torch.arange(len(x)) % 3 == 1, 1.0, 0.0)


def many_larger_ones(x, lowest):
    x[20000:23000] = 9.0                                     # more than are kept, in a later batch
    x[50000:] = 9.5


# 24576 tokens are a range of 120 rows: the first batches of the second range are masked in all of these. Masks that end 600 tokens before a batch's end,
# or leave few tokens, let fewer logits pass at once than are kept.
MASKS = [masked_until(*where, size, every) for where in ((33768, -math.inf), (40360, -math.inf), (40360, "lowest"), (40360, -2e6))
         for size, every in ((0, 1), (-100, 1), (-700, 1), (-720, 1), (-800, 1), (-1000, 1), (-20000, 1), (-1000, 31), (-740, 50))]
MASKS += [few({10000: -10000.0, 12000: 5.0, 30000: 1.0}), few({40000: -900.0, 40001: -901.0, 69999: -2000.0})]
ORDERS = [stepped(50.0, 5000), stepped(-50.0, 5000), stepped(-700.0, 9000), at([9000, 33333], math.nan), at(slice(60000, 60009), math.nan),
          all_alike, two_sizes, many_larger_ones, at([69000], 38.0), at([9000, 69000], 80.0), at(slice(30000, 31000), 20.0)]


def logits_of(kinds, rows, vocab, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g)
    for r in range(rows):
        kinds[r % len(kinds)](x[r], torch.finfo(dtype).min)
    if dtype == F16:
        x = torch.where(torch.isfinite(x), x.clamp(min=torch.finfo(F16).min), x)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kinds", [MASKS, ORDERS], ids=["masks", "orders"])
@pytest.mark.parametrize("rows", [120, 230])
def test_logits_behind_the_first_batch(rows, kinds, dtype):
    vocab = 70001
    assert batches_of_a_range(rows, vocab, dtype)[0] >= (3 if rows == 120 else 9)
    x = logits_of(kinds, rows, vocab, dtype)
    check(lm.beam_step(x, None, 1, 8), ref.beam_step(x, None, 1, 8))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_groups_of_masked_rows(dtype):
    """Three tokens of a grammar's, one of them at a bias far below the others, in beams whose order hangs on the sums."""
    groups, beams, vocab = 24, 5, 49999
    assert batches_of_a_range(groups * beams, vocab, dtype)[0] >= 3
    x = logits_of([few({10000: -10000.0, 12000: 5.0, 30000: 1.0}), few({33000: -1000.0, 33001: -1000.5}), masked_until(30000, -math.inf, -5000),
                   masked_until(45000, "lowest", 4), stepped(-1000.0, 20000)], groups * beams, vocab, dtype)
    scores = (-3 * torch.rand(groups * beams, generator=torch.Generator().manual_seed(2))).cuda()
    check(lm.beam_step(x, scores, beams, 10), ref.beam_step(x, scores, beams, 10))


@pytest.mark.parametrize("rows", [1, 120])
def test_logits_about_a_million_below_zero(rows):
    """An additive mask of -10^6 over whole rows: fp32 logits on both sides of what single exponents are for, in batches, ranges and rows."""
    vocab = 70001
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(3)) - 1e6
    x[::3, :24576] = -1000000.5
    x[::3, 24576:] = -999999.5
    x[1::6, :40000] = -1000003.0
    x[1::6, 40000:] = -999995.0
    x[4::6] = -1000040.0
    x[4::6, 33333] = -999990.0
    x = x.cuda()
    check(lm.beam_step(x, None, 1, 4), ref.beam_step(x, None, 1, 4))


# ------------------------------------------------------------------------------------------------------ sums
def climbing(x, batch, height, step=0.0):
    """`height` above the first batch from the third on; in the second in every tenth token, so that not too many pass at once."""
    t = torch.arange(x.shape[-1])
    x[..., batch:2 * batch][..., ::10] = height
    x[..., 2 * batch:] = (height - step * (t % 16).float())[2 * batch:]


def checked_sums(x, limit):
    """The best total of each row, its score chosen so that the total is near 0 and its rounding below 2^-36."""
    exact = torch.logsumexp(x.double(), 1)
    scores = (exact - x.double().amax(1)).float()
    want = scores.double() - exact + x.double().amax(1)
    assert float(want.abs().max()) < 2.0 ** -12
    got = lm.beam_step(x, scores, 1, 4)[0][:, 0].double()
    assert float((got - want).abs().max()) <= limit, float((got - want).abs().max())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("step", [0.0, 2.0 ** -6, 2.0 ** -4])
def test_sums_of_rows_that_rise_above_their_first_batch(step, dtype):
    """A first batch at 0 and the rest up to 39 above it. 2^-22 for what a weight near the reference is off by, 2 ulp; the rounding of its exponent below 2
    is 2^-24 ln 2, and so is half a step of each of its six sums: 2^-21 is their total."""
    rows, vocab = 120, 70001
    each, batch = batches_of_a_range(rows, vocab, dtype)
    assert each >= 3
    x = 0.3 * torch.randn(rows, vocab, generator=torch.Generator().manual_seed(5))
    for r in range(rows):
        climbing(x[r], batch, 39.0 - 0.25 * r, step)
    checked_sums(x.to(dtype).cuda(), 2.0 ** -21)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [3, 120])
def test_sums_of_thousands_of_alike_far_below_the_largest(rows, dtype):
    """The exponent of each of them is rounded alike: by 2^-20 of 16 to 32, by 2^-21 below."""
    vocab = 70001
    x = torch.zeros(rows, vocab)
    x[:, 2345] = torch.linspace(4.0, 14.0, rows)
    x[:, 60000] = x[:, 2345] - 0.5
    checked_sums(x.to(dtype).cuda(), 2.0 ** -19)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("edge,rest", [(30.0, 39.5), (1.25, 1.0), (12.0, 0.0), (11.25, 0.0), (13.5, 0.0), (12.75, 0.25), (0.0, 38.0), (10.5, 0.0), (20.0, 33.25),
                                       (25.5, 30.75), (3.25, 39.0), (8.5, 36.25)])
def test_beams_alike_whose_batches_are_not(edge, rest, dtype):
    """The same logits in rows that lie differently to 16 bytes: what is the last of one row's first batch is in the other's second."""
    beams, vocab, groups = 4, 70001, 30
    each, batch = batches_of_a_range(groups * beams, vocab, dtype)
    assert each >= 3
    x = torch.zeros(groups * beams, vocab)
    climbing(x, batch, rest)
    x[:, batch - 2] = edge
    x[:, 50000] = max(edge, rest) + 0.5
    x, stride = x.to(dtype).cuda(), vocab + vocab % 2 + 1                  # an odd number
    room = torch.zeros(len(x) * stride + 16, dtype=dtype, device="cuda")
    view = room[:len(x) * stride].view(len(x), stride)[:, :vocab]
    view.copy_(x)
    scores = torch.full((len(x),), -2.0).cuda()
    got, (want, gap) = lm.beam_step(view, scores, beams, 8), ref.beam_step(x, scores, beams, 8)
    assert gap > 2.0 ** -18
    for i in (1, 2, 3, 4):
        assert torch.equal(got[i].cpu().long(), want[i].long()), i
    for i in (0, 5):
        assert bool(((got[i].cpu().double() - want[i]).abs() <= 2.0 ** -19 + want[i].abs() * 2.0 ** -24).all())


# ------------------------------------------------------------------------------------------------------ totals that 64 bits cannot tell apart
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 300), (3, 70001), (120, 70001)])
def test_a_beams_order_is_its_logits(rows, vocab, dtype):
    """Beside an infinite logit (the largest number), or a score as large, all other totals of a beam are the same number."""
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(4))
    x[:, vocab // 3] = math.inf
    x = x.to(dtype).cuda()
    check(lm.beam_step(x, None, 1, 8), ref.beam_step(x, None, 1, 8))
    x[:, vocab // 3] = 0
    scores = torch.full((rows,), -1e30).cuda()
    check(lm.beam_step(x, scores, 1, 128), ref.beam_step(x, scores, 1, 128))
    if rows % 3 == 0:
        check(lm.beam_step(x, scores, 3, 128), ref.beam_step(x, scores, 3, 128))
