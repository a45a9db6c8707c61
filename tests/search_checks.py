"""Plain implementations of the operators that search and choose over the paged cache, for their tests: whole numbers as they are, all
others in 64 bits."""
import math

import torch


def beam_step(logits, scores, beams, count, ends=()):
    """What lm.beam_step returns, its scores in 64 bits, and the smallest distance between neighbouring totals of different beams."""
    rows, vocab = logits.shape
    x = logits.cpu().double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(logits.dtype).max)
    s = torch.zeros(rows, dtype=torch.float64) if scores is None else scores.cpu().double()
    out, gap = [[] for _ in range(6)], math.inf
    for g in range(rows // beams):
        totals, at = [], []
        for b in range(beams):
            r = g * beams + b
            keep = torch.nonzero(x[r] > -math.inf)[:, 0]
            if not torch.isfinite(s[r]) or len(keep) == 0:
                continue
            top = x[r].max()
            total = s[r] - torch.log(torch.exp(x[r] - top).sum()) + (x[r][keep] - top)
            order = torch.sort(-x[r][keep], stable=True).indices[:count]
            totals.append(total[order])
            at.append(b * vocab + keep[order])
        totals, at = (torch.cat(totals), torch.cat(at)) if totals else (torch.zeros(0, dtype=torch.float64), torch.zeros(0, dtype=torch.long))
        order = torch.sort(-totals, stable=True).indices[:count + 1]
        totals, at = totals[order], at[order]
        for i in range(len(at) - 1):
            if at[i] // vocab != at[i + 1] // vocab and totals[i] != totals[i + 1]:
                gap = min(gap, float((totals[i] - totals[i + 1]) / max(1.0, abs(float(totals[i])) * 2.0 ** -20)))
        totals, at = totals[:count], at[:count]
        missing = count - len(at)
        out[0].append(torch.cat([totals, torch.full((missing,), -math.inf, dtype=torch.float64)]))
        out[1].append(torch.cat([at // vocab, torch.full((missing,), -1)]))
        out[2].append(torch.cat([at % vocab, torch.full((missing,), -1)]))
        on = [i for i in range(len(at)) if int(at[i] % vocab) not in ends][:beams]
        missing = beams - len(on)
        out[3].append(torch.cat([g * beams + at[on] // vocab, torch.full((missing,), -1)]))
        out[4].append(torch.cat([at[on] % vocab, torch.full((missing,), -1)]))
        out[5].append(torch.cat([totals[on], torch.full((missing,), -math.inf, dtype=torch.float64)]))
    groups = rows // beams
    shaped = [torch.stack(o) if o else torch.zeros(0, count if i < 3 else beams) for i, o in enumerate(out)]
    return [o.view(groups, count) if i < 3 else o.reshape(-1) for i, o in enumerate(shaped)], gap


def check_beam_step(got, want):
    want, gap = want
    # neighbours so near that 22 bits of a logarithm may swap them would prove nothing
    assert gap > 2.0 ** -20, gap
    for i in (1, 2, 3, 4):
        assert got[i].dtype == torch.int32 and torch.equal(got[i].cpu().long(), want[i].long()), i
    for i in (0, 5):
        a, b = got[i].cpu().double(), want[i]
        assert got[i].dtype == torch.float32 and torch.equal(torch.isinf(a), torch.isinf(b) | (b.abs() > 3.4028235677973366e38))
        fine = torch.isfinite(a)
        # the total's rounding to fp32, and the logarithm's 2^-22
        limit = b[fine].abs() * 2.0 ** -24 + 2.0 ** -22
        assert bool(((a - b)[fine].abs() <= limit).all()), float(((a - b)[fine].abs() - limit).max())


def advance(table, kv_len, parent, new, refs, page, blocks=None):
    """What lm.advance_pages returns, as lists."""
    blocks = len(table[0]) if blocks is None and table else blocks or 0
    pages, now = len(refs), list(refs)

    def is_page(p):
        return 0 <= p < pages

    for row in table:
        for p in row:
            if is_page(p):
                now[p] -= 1
    free = [p for p in range(pages) if refs[p] == 0]
    tables, lengths, copies, missing, kept = [], [], [], 0, set()
    for i, p in enumerate(parent):
        there = 0 <= p < len(table)
        old = max(kv_len[p], 0) if there else 0
        more = max(new[i] if isinstance(new, list) else new, 0)
        row, copy = [-1] * blocks, (-1, -1, 0)
        for c in range(min(blocks, -(-(old + more) // page))):
            if c < old // page:
                row[c] = table[p][c] if c < len(table[p]) else -1
                continue
            half = c * page < old
            if half:
                has = table[p][c] if c < len(table[p]) else -1
                if not is_page(has):
                    continue
                if refs[has] == 1 and p not in kept:
                    kept.add(p)
                    row[c] = has
                    continue
            row[c] = free.pop(0) if free else -1
            missing += row[c] < 0
            if half and row[c] >= 0:
                copy = (has, row[c], old % page)
        for q in row:
            if is_page(q):
                now[q] += 1
        tables.append(row)
        lengths.append(old + more)
        copies.append(copy)
    return tables, lengths, now, copies, [now.count(0), missing]


def compact(table, refs, most, page):
    refs, used = list(refs), sum(r != 0 for r in refs)
    pairs = list(zip([p for p in range(used, len(refs)) if refs[p] != 0], [p for p in range(used) if refs[p] == 0]))
    left = max(0, len(pairs) - most)
    pairs = pairs[:most]
    to = dict(pairs)
    for a, b in pairs:
        refs[b], refs[a] = refs[a], 0
    copies = [(a, b, page) for a, b in pairs] + [(-1, -1, 0)] * (most - len(pairs))
    return [[to.get(p, p) for p in row] for row in table], refs, copies, [used, left]


def power_of_two(amax):
    """The smallest power of two t with amax <= 127 t; 1 for 0."""
    return 1.0 if amax == 0 else 2.0 ** math.ceil(math.log2(amax / 127))


def page_bounds(k, k_scale, page, tokens):
    """(bounds [heads, 2, dim], unit [heads]) of the first tokens of a page."""
    lo_hi, unit = [], []
    for h in range(k.shape[1]):
        x = k[page, h, :tokens].double()
        lo = torch.where(torch.isnan(x), math.inf, x).amin(0)
        hi = torch.where(torch.isnan(x), -math.inf, x).amax(0)
        lo, hi = torch.where(torch.isinf(lo), 0.0, lo), torch.where(torch.isinf(hi), 0.0, hi)
        t = power_of_two(float(torch.maximum(lo.abs(), hi.abs()).max()))
        lo_hi.append(torch.stack([torch.floor(lo / t), torch.ceil(hi / t)]))
        unit.append(t * float(k_scale[page, h]))
    return torch.stack(lo_hi), torch.tensor(unit, dtype=torch.float64)


def choose_row(q, bounds, unit, pages, own, count, first, last):
    """A row's choice for one kv head. q [heads of the group, dim]; bounds and unit of the head's pages; pages of the row's blocks up to its own."""
    q = torch.where(torch.isfinite(q.double()), q.double(), 0.0)
    q = torch.round(q / power_of_two(float(q.abs().max()))).clamp(-127, 127)
    there = torch.nonzero(torch.as_tensor(pages)[:own + 1] >= 0)[:, 0].tolist()
    always = [c for c in there if c < first or c > own - last]
    rest = [c for c in there if c not in set(always)]
    if len(rest) > count - len(always):
        at = torch.tensor([int(pages[c]) for c in rest])
        lo, hi = bounds[at, 0].double(), bounds[at, 1].double()
        score = (q.clamp(min=0) @ hi.T + q.clamp(max=0) @ lo.T).amax(0) * unit[at].double()
        order = torch.sort(-score, stable=True).indices[:count - len(always)]
        rest = [rest[i] for i in order.tolist()]
    have = sorted(always + rest)
    return have + [-1] * (count - len(have))


def sparse64(q, batch, total, new, chosen, scale=None):
    """(out, lse, largest |v|) of every row over its chosen pages, in 64 bits."""
    k_cache, v_cache, ks, vs = (t.cpu() for t in batch["cache"])
    rows, heads, dim = q.shape
    kv_heads, page = k_cache.shape[1], k_cache.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    table, chosen, q = batch["block_table"].cpu(), chosen.cpu(), q.cpu().double()
    out, lse = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.full((rows, heads), -math.inf, dtype=torch.float64)
    row, top, group = 0, 0.0, heads // kv_heads
    for b, n in enumerate(new):
        for r in range(n):
            place = total[b] - n + r
            for h in range(kv_heads):
                blocks = [c for c in chosen[row, h].tolist() if c >= 0 and c * page <= place and 0 <= int(table[b, c]) < k_cache.shape[0]]
                if not blocks:
                    continue
                at = table[b, blocks].long()
                j = (torch.tensor(blocks)[:, None] * page + torch.arange(page)).reshape(-1)
                seen = j <= place
                k = (k_cache[at, h].double() * ks[at, h].double()[:, None, None]).reshape(-1, dim)[seen]
                v = (v_cache[at, h].double() * vs[at, h].double()[:, None, None]).reshape(-1, dim)[seen]
                s = q[row, h * group:(h + 1) * group] @ k.T * scale
                lse[row, h * group:(h + 1) * group] = torch.logsumexp(s, 1)
                out[row, h * group:(h + 1) * group] = torch.softmax(s, 1) @ v
                top = max(top, float(torch.nan_to_num(v).abs().max()))
            row += 1
    return out, lse, top
