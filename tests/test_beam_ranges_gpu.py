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


# 24576 tokens are a range of 120 rows: the first batches of the second range are masked in all of these. Masks that end 600 tokens before a batch's end,
# or leave few tokens, let fewer logits pass at once than are kept.
MASKS = [masked_until(*where, size, every) for where in ((33768, -math.inf), (40360, -math.inf), (40360, "lowest"), (40360, -2e6))
         for size, every in ((0, 1), (-100, 1), (-700, 1), (-720, 1), (-800, 1), (-1000, 1), (-20000, 1), (-1000, 31), (-740, 50))]
MASKS += [few({10000: -10000.0, 12000: 5.0, 30000: 1.0}), few({40000: -900.0, 40001: -901.0, 69999: -2000.0})]


def logits_of(kinds, rows, vocab, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g)
    for r in range(rows):
        kinds[r % len(kinds)](x[r], torch.finfo(dtype).min)
    if dtype == F16:
        x = torch.where(torch.isfinite(x), x.clamp(min=torch.finfo(F16).min), x)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [120, 230])
def test_logits_behind_the_first_batch(rows, dtype):
    vocab = 70001
    assert batches_of_a_range(rows, vocab, dtype)[0] >= (3 if rows == 120 else 9)
    x = logits_of(MASKS, rows, vocab, dtype)
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
