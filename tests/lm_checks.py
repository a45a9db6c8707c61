"""Plain implementations in 64 bits of the language-model operators, for their tests."""
import math

import torch

E4M3 = torch.float8_e4m3fn


def make_batch(new, past, page, kv_heads, dim, seed=0, spare=2, device="cuda", token_major=False):
    """A cache with random contents for sequences of new[b] rows behind past[b] tokens, its pages in random order.
    Unused bytes - spare pages, slots behind a sequence's end - are NaN."""
    g = torch.Generator().manual_seed(seed)
    total = [n + p for n, p in zip(new, past)]
    blocks = [-(-t // page) for t in total]
    pages, wide = sum(blocks) + spare, max(max(blocks), 1)
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(new), wide), -1, dtype=torch.int32)
    first = 0
    cache = []
    for _ in range(2):
        x = torch.randn(pages, kv_heads, page, dim, generator=g) * torch.exp2(torch.randn(pages, kv_heads, 1, 1, generator=g))
        scale = scale_for(x.abs().amax((2, 3)))
        c = (x / scale[..., None, None]).to(E4M3)
        cache.append((c, scale))
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(blocks):
        table[b, :n] = order[first:first + n]
        first += n
        for i in range(n):
            used[table[b, i], :max(0, min(page, total[b] - i * page))] = True
    for c, _ in cache:
        c.view(torch.uint8)[(~used)[:, None, :].expand(pages, kv_heads, page)] = 0x7f
    (k, ks), (v, vs) = cache
    if token_major:        # [pages][tokens][heads][dim] in memory
        k, v = (c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3) for c in (k, v))
        k, v = (c.view(torch.uint8).transpose(1, 2).to(device).transpose(1, 2).view(E4M3) for c in (k, v))
    else:
        k, v = k.to(device), v.to(device)
    row_start = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
    return dict(cache=(k, v, ks.to(device), vs.to(device)), block_table=table.to(device),
                kv_len=torch.tensor(total, dtype=torch.int32, device=device), max_kv_len=max(total), row_start=row_start.to(device),
                max_rows=max(new)), total


def scale_for(amax):
    """The smallest power of two s with amax <= 448 s; 1 for 0."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875)), torch.ones_like(amax))


def cached(c, scale, table, n):
    """The first n tokens [n, heads, dim] of a sequence in 64 bits."""
    page = c.shape[2]
    at = table[:-(-n // page)].long().cpu()
    x = c.cpu()[at].double() * scale.cpu()[at].double()[..., None, None]
    return x.transpose(1, 2).reshape(-1, c.shape[1], c.shape[3])[:n]


def attention64(q, batch, total, new, scale=None, causal=True, window=0):
    """(out, lse, largest |v|) of every row, in 64 bits."""
    k_cache, v_cache, ks, vs = batch["cache"]
    rows, heads, dim = q.shape
    q = q.cpu().double()
    scale = dim ** -0.5 if scale is None else scale
    out, lse = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.full((rows, heads), -math.inf, dtype=torch.float64)
    row, top = 0, 0.0
    for b, n in enumerate(new):
        k = cached(k_cache, ks, batch["block_table"][b], total[b])
        v = cached(v_cache, vs, batch["block_table"][b], total[b])
        if total[b]:
            top = max(top, float(torch.nan_to_num(v).abs().max()))
        if total[b] and n:
            pos, j = torch.arange(total[b] - n, total[b])[:, None], torch.arange(total[b])[None]
            hidden = torch.zeros(n, total[b], dtype=torch.bool)
            if causal:
                hidden |= j > pos
            if window:
                hidden |= j <= pos - window
            hidden_all = hidden.all(1)
            for h in range(heads):
                kh = h // (heads // k.shape[1])
                # a hidden token is left out, not multiplied by 0
                s = (q[row:row + n, h] @ k[:, kh].T * scale).masked_fill(hidden, -math.inf)
                p = torch.softmax(s, 1).masked_fill(hidden, 0.0)
                lse[row:row + n, h] = torch.logsumexp(s, 1)
                out[row:row + n, h] = (p @ v[:, kh]).masked_fill(hidden_all[:, None], 0.0)
        row += n
    return out, lse, top


#: In units of the largest |v|: for 16-bit activations the rounding of each weight to 11 bits, and 2e-5 for sums, scores and
#: exponentials in fp32 (scores up to about 30: 30 x 2^-22 of each weight, on both sides of the division). The result's own rounding
#: comes on top, element by element.
LIMIT = {torch.float32: 2e-5, torch.float16: 2.0 ** -11 + 2e-5, torch.bfloat16: 2.0 ** -11 + 2e-5}
BITS = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}


def half_step(x, dtype):
    """Half the distance between neighbours of x in the type: what rounding x to it may change."""
    return torch.exp2(torch.frexp(x.abs())[1].double() - 1 - BITS[dtype])


def check_attention(got, want, dtype):
    out, lse, top = want
    got_out, got_lse = got[0].cpu().double(), got[1].cpu().double()
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    assert torch.equal(torch.isnan(got_out), torch.isnan(out))
    limit = LIMIT[dtype] * max(top, 1e-30) + half_step(out.nan_to_num(), dtype)
    over = ((got_out - out).nan_to_num().abs() - limit).max() if out.numel() else 0.0
    assert float(over) <= 0, (float(over), top)
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), empty) and bool((got_out[empty] == 0).all())
    if (~empty).any():
        e = (got_lse - lse)[~empty].nan_to_num().abs() / lse[~empty].nan_to_num().abs().clamp(min=1)
        assert float(e.max()) <= 2e-5, float(e.max())


def rotated32(x, table, positions, interleaved):
    """Rotation in fp32, each operation rounded."""
    x = x.float().clone()
    R = table.shape[1]
    c, s = table[positions][:, None, :R // 2], table[positions][:, None, R // 2:]
    a, b = (x[..., 0:R:2].clone(), x[..., 1:R:2].clone()) if interleaved else (x[..., :R // 2].clone(), x[..., R // 2:R].clone())
    u, v = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:R:2], x[..., 1:R:2] = u, v
    else:
        x[..., :R // 2], x[..., R // 2:R] = u, v
    return x


def append32(x, cache, scale, table, new, total):
    """What appending x [rows, heads, dim] (fp32) makes of one of the caches: (cache, scale), from copies on the host."""
    cache, scale = cache.cpu().contiguous().clone(), scale.cpu().clone()
    page, row = cache.shape[2], 0
    for b, n in enumerate(new):
        t = total[b] - n
        while t < total[b]:
            end = min(total[b], (t // page + 1) * page)
            at, slot = int(table[b, t // page]), t % page
            part = x[row:row + end - t]
            row += end - t
            if at >= 0:
                finite = torch.where(torch.isfinite(part), part.abs(), torch.zeros(()))
                top = finite.amax((0, 2))
                need = torch.where(top > 0, scale_for(top), torch.zeros(()))
                old = scale[at].clone() if slot else torch.zeros_like(need)
                now = torch.maximum(old, need)
                now = torch.where(now > 0, now, torch.ones(()))
                if slot:
                    # what the page has is moved even where nobody will read it: the bytes behind the new rows
                    keep = torch.ones(page, dtype=torch.bool)
                    keep[slot:slot + end - t] = False
                    moved = (cache[at].float() * (old / now)[:, None, None]).to(E4M3)
                    grown = (now > old)[:, None] & keep[None]
                    cache[at] = torch.where(grown[..., None], moved.float(), cache[at].float()).to(E4M3)
                y = (part / now[:, None]).clamp(-448, 448)      # a NaN stays one
                cache.view(torch.uint8)[at, :, slot:slot + end - t] = y.transpose(0, 1).contiguous().to(E4M3).view(torch.uint8)
                scale[at] = now
            t = end
    return cache, scale


def same_bytes(a, b):
    """Equal e4m3 values, any NaN like any other."""
    a, b = a.cpu().float(), b.cpu().float()
    return bool(torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num()))
