"""Performance cases of the operators that search and choose over the paged cache: a step of a beam search, the pages that
follow it (shared, copied, freed, compacted), and attention over the pages that a cheap score chooses for each query.

A case is a dict of plain values. `listed()` gives the named ones, `draw(rng)` one more of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass - the framework's calls where `own` is set,
else elementary torch operations -, `work(case)` the bytes and operations a pass cannot do without, and `exact(case, seed)` the
same results from the definitions in 64 bits.

Kinds:
  beam     lm.beam_step: the best continuations over all beams and tokens of a group
  fork     lm.advance_pages, lm.copy_pages: tables of the texts that go on, new pages, copies of the pages that two texts would write to
  compact  lm.compact_pages, lm.copy_pages: used pages move to the front of the pool
  choose   lm.page_bounds, lm.choose_pages: bounds of the pages that were appended to, then the pages that each query attends
  sparse   lm.sparse_attention: attention over the chosen pages

The cache is e4m3 [pages][kv heads][page tokens][head dim] with one power-of-two scale for each page and head. Sequence b has
rows row_start[b]..row_start[b + 1] of the call and kv_len[b] tokens in the cache, the rows' own among them.
"""
import math
import random

import torch

own = False

DTYPE = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
E4M3_MAX = 448.0


def listed():
    return [
        # one request, four beams, the framework's own activations: latency
        dict(name="beam_one", kind="beam", groups=1, beams=4, vocab=32000, count=8, masked=False, dtype="fp32"),
        # a batch under grammars that leave a quarter of the tokens, an odd vocabulary
        dict(name="beam_masked_24", kind="beam", groups=24, beams=5, vocab=49999, count=10, masked=True, dtype="fp16"),
        # a large batch of wide searches
        dict(name="beam_batch_48", kind="beam", groups=48, beams=8, vocab=128001, count=16, masked=False, dtype="bf16"),
        # the pages behind one request's step, small pages
        dict(name="fork_one", kind="fork", groups=1, beams=4, past=700, new=1, kv_heads=8, dim=128, page=16, layers=2),
        # the pages behind a batch's step: four layers of caches copied together
        dict(name="fork_batch_64", kind="fork", groups=64, beams=8, past=1500, new=1, kv_heads=8, dim=128, page=64, layers=4),
        # a small pool after a few answers have ended
        dict(name="compact_small", kind="compact", pages=700, used=0.5, seqs=12, kv_heads=4, dim=64, page=32, layers=1, most=64),
        # a pool of many small pages, thousands of them to move
        dict(name="compact_pool", kind="compact", pages=50001, used=0.6, seqs=300, kv_heads=2, dim=96, page=16, layers=4, most=8192),
        # a serving batch's next tokens, lengths of all kinds
        dict(name="choose_step_64", kind="choose", seqs=64, new=1, past=8000, q_heads=32, kv_heads=8, dim=128, page=64, count=16, dtype="bf16"),
        # drafts over a few documents of great length, small pages
        dict(name="choose_long_drafts", kind="choose", seqs=3, new=4, past=150000, q_heads=16, kv_heads=2, dim=128, page=32, count=64,
             dtype="fp16"),
        # one user's next token in a long document: latency
        dict(name="sparse_one", kind="sparse", seqs=1, new=1, past=30000, q_heads=32, kv_heads=8, dim=128, page=64, count=16, dtype="bf16"),
        # the ordinary serving batch
        dict(name="sparse_step_64", kind="sparse", seqs=64, new=1, past=8000, q_heads=32, kv_heads=8, dim=128, page=64, count=24, dtype="bf16"),
        # a chunk of a prompt deep in two long documents, neighbours choosing alike
        dict(name="sparse_chunk", kind="sparse", seqs=2, new=500, past=40000, q_heads=32, kv_heads=8, dim=128, page=64, count=24, dtype="bf16"),
    ]


def _near(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "fork", "compact", "choose", "sparse", "sparse"])
    while True:
        if kind == "beam":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
            case = dict(kind=kind, groups=_near(rng, 1, 200), beams=beams, vocab=_near(rng, 500, 150000), count=rng.choice([beams, 2 * beams]),
                        masked=rng.random() < 0.3, dtype=rng.choice(["fp32", "fp16", "bf16"]))
            if case["groups"] * beams * case["vocab"] <= 48 * 8 * 128001 and case["vocab"] >= 20 * case["count"]:
                return case
        elif kind == "fork":
            case = dict(kind=kind, groups=_near(rng, 1, 100), beams=rng.choice([1, 2, 3, 4, 5, 8]), past=_near(rng, 1, 4000),
                        new=rng.choice([1, 1, rng.randint(2, 100)]), kv_heads=rng.choice([1, 2, 4, 5, 8]), dim=rng.choice([64, 80, 128, 256]),
                        page=rng.choice([16, 32, 64, 128]), layers=rng.choice([1, 2, 3, 4]))
            if _pool(case) * _page_bytes(case) * case["layers"] <= 4 << 30:
                return case
        elif kind == "compact":
            case = dict(kind=kind, pages=_near(rng, 20, 60000), used=rng.choice([0.1, 0.5, 0.8, 0.97]), seqs=_near(rng, 1, 400),
                        kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 96, 128]), page=rng.choice([16, 32, 64]), layers=rng.choice([1, 2, 4]),
                        most=_near(rng, 16, 8192))
            if case["pages"] * _page_bytes(case) * case["layers"] <= 50001 * 6144 * 4 and case["seqs"] * 4 <= case["pages"]:
                return case
        else:
            kv_heads = rng.choice([1, 2, 4, 5, 8])
            case = dict(kind=kind, seqs=_near(rng, 1, 128), new=rng.choice([1, 1, 1, rng.randint(2, 8), _near(rng, 9, 600)]),
                        past=_near(rng, 200, 200000), q_heads=kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 16]), kv_heads=kv_heads,
                        dim=rng.choice([64, 80, 96, 128, 128, 256]), page=rng.choice([16, 32, 64, 64, 128]), count=_near(rng, 4, 96),
                        dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]))
            rows, keys = case["seqs"] * case["new"], min(case["count"] * case["page"], case["past"] + case["new"])
            cached = case["seqs"] * (case["past"] + case["new"]) * kv_heads * case["dim"]
            if cached > 64 * 8001 * 8 * 128:
                continue
            if kind == "choose" and rows * case["q_heads"] * case["dim"] * ((case["past"] + case["new"]) // case["page"] + 1) <= 2e10:
                return case
            # no dearer than the chunk: the plain form gathers every row's keys in 32 bits
            if kind == "sparse" and rows * case["q_heads"] * keys * case["dim"] <= 1000 * 32 * 24 * 64 * 128 and rows * kv_heads * keys >= 2000:
                return case


def _page_bytes(case):
    return 2 * case["kv_heads"] * case["page"] * case["dim"]


def _lengths(case):
    """(new rows, earlier tokens) of each sequence: known to the host, as a scheduler knows them. The first has the most; the others
    go by their number."""
    r = random.Random(case["seqs"] * 1000003 + case["new"] * 1009 + case["past"])
    new = [case["new"]] + [r.randint(max(1, case["new"] // 8), case["new"]) for _ in range(case["seqs"] - 1)]
    past = [case["past"]] + [r.randint(min(1, case["past"]), case["past"]) for _ in range(case["seqs"] - 1)]
    return new, past


def _prompt_and_answer(case):
    """Tokens of each group's prompt, whose full pages its beams share, and of the answers so far (the same for a group's beams)."""
    r = random.Random(case["groups"] * 1000003 + case["beams"] * 1009 + case["past"])
    total = [case["past"]] + [r.randint(max(1, case["past"] // 8), case["past"]) for _ in range(case["groups"] - 1)]
    return [(t - t // 4, t // 4) for t in total]


def _pool(case):
    """Pages of the pool of a fork: what the tables name, what the step may ask for, and some to spare."""
    n = 5
    for prompt, answer in _prompt_and_answer(case):
        shared = prompt // case["page"]
        n += shared + case["beams"] * (-(-(prompt + answer) // case["page"]) - shared)
    return n + case["groups"] * case["beams"] * (1 + -(-case["new"] // case["page"]))


def work(case):
    kind = case["kind"]
    if kind == "beam":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * SIZE[case["dtype"]] + 16) + 12 * case["groups"] * case["count"], "flops": 0}
    if kind == "fork":
        # of a group's beams about a third find their parent taken: half a page each, read and written
        seqs, blocks = case["groups"] * case["beams"], max(-(-(p + a + case["new"]) // case["page"]) for p, a in _prompt_and_answer(case))
        copies = 0 if case["beams"] == 1 else seqs // 3
        return {"bytes": 8 * seqs * blocks + 8 * _pool(case) + copies * _page_bytes(case) * case["layers"], "flops": 0}
    if kind == "compact":
        moves = min(case["most"], int(case["pages"] * case["used"] * (1 - case["used"])))
        return {"bytes": 8 * case["pages"] + 8 * int(case["pages"] * case["used"]) + 2 * moves * _page_bytes(case) * case["layers"], "flops": 0}
    new, past = _lengths(case)
    rows, size, kv = sum(new), SIZE[case["dtype"]], case["kv_heads"] * case["dim"]
    blocks = [-(-(n + p) // case["page"]) for n, p in zip(new, past)]
    pairs = sum(n * b for n, b in zip(new, blocks))
    if kind == "choose":
        fresh = sum((p + n - 1) // case["page"] - p // case["page"] + 1 for n, p in zip(new, past))
        return {"bytes": fresh * (case["page"] * kv + 2 * kv + 8 * case["kv_heads"]) + sum(blocks) * (2 * kv + 4 * case["kv_heads"] + 4)
                + rows * (case["q_heads"] * case["dim"] * size + 4 * case["kv_heads"] * case["count"]),
                "flops": 2 * pairs * case["q_heads"] * case["dim"]}
    keys = sum(n * min(case["count"] * case["page"], p + n) for n, p in zip(new, past))
    read = sum(min(case["count"] * case["page"], p + n) for n, p in zip(new, past))
    return {"bytes": rows * (case["q_heads"] * (2 * case["dim"] * size + 4) + 4 * case["kv_heads"] * case["count"]) + 2 * read * kv,
            "flops": 4 * keys * case["q_heads"] * case["dim"]}


def _power_of_two_scale(amax, most=E4M3_MAX):
    """The smallest power of two s with amax <= most s (1 where there is nothing); most is below 2^9 and not below 2^8, or 127."""
    m, e = torch.frexp(amax)
    bits, border = (9, 0.875) if most == E4M3_MAX else (7, 127 / 128)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - bits + (m > border)), torch.ones_like(amax))


def _filled_cache(shape, g):
    """Random keys or values as a running service has them: a page's head has its own amplitude, a few channels are larger. Made a
    few pages at a time."""
    pages, heads, page, dim = shape
    cache = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(pages, heads, device="cuda")
    wide = 1 + 2 * (torch.rand(1, heads, 1, dim, generator=g, device="cuda") < 0.03)
    step = max(1, (1 << 28) // (heads * page * dim))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        x = torch.randn(n, heads, page, dim, generator=g, device="cuda")
        x += torch.randn(n, heads, 1, dim, generator=g, device="cuda")       # neighbours are alike
        x *= torch.exp2(0.7 * torch.randn(n, heads, 1, 1, generator=g, device="cuda"))
        x *= wide
        scale[p:p + n] = _power_of_two_scale(x.abs().amax((2, 3)))
        cache[p:p + n] = (x / scale[p:p + n, :, None, None]).to(cache.dtype)
    return cache, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"beam": _prepare_beam, "fork": _prepare_fork, "compact": _prepare_compact, "choose": _prepare_attention,
            "sparse": _prepare_attention}[case["kind"]](case, g)


def _prepare_beam(case, g):
    rows, V = case["groups"] * case["beams"], case["vocab"]
    x = 2.5 * torch.randn(rows, V, generator=g, device="cuda")
    likely = torch.randint(0, V, (rows, 6), generator=g, device="cuda")
    x.scatter_add_(1, likely, 3 + 8 * torch.rand(rows, 6, generator=g, device="cuda"))
    if case["masked"]:
        x[torch.rand(rows, V, generator=g, device="cuda") < 0.75] = -math.inf
    scores = -40 * torch.rand(rows, generator=g, device="cuda").view(case["groups"], case["beams"])
    # beams of a group are not far apart; a few have ended, but never a group's first
    scores = scores[:, :1] - 6 * torch.rand(scores.shape, generator=g, device="cuda")
    gone = torch.rand(scores.shape, generator=g, device="cuda") < 0.05
    gone[:, 0] = False
    scores[gone] = -math.inf
    ends = torch.cat([likely[0, :1], torch.randint(0, V, (1,), generator=g, device="cuda")]).int()
    return dict(case=case, logits=x.to(DTYPE[case["dtype"]]), scores=scores.reshape(-1).contiguous(), ends=ends)


def _prepare_fork(case, g):
    page, beams, pool = case["page"], case["beams"], _pool(case)
    texts = _prompt_and_answer(case)
    wide = max(-(-(p + a + case["new"]) // page) for p, a in texts)
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((len(texts) * beams, wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, (prompt, answer) in enumerate(texts):
        shared, all_blocks = prompt // page, -(-(prompt + answer) // page)
        rows = table[i * beams:(i + 1) * beams]
        rows[:, :shared] = order[at:at + shared]
        at += shared
        mine = beams * (all_blocks - shared)
        rows[:, shared:all_blocks] = order[at:at + mine].view(beams, -1)
        at += mine
    kv_len = torch.tensor([p + a for p, a in texts], dtype=torch.int32).repeat_interleave(beams).cuda()
    refs = torch.bincount(table[table >= 0].long(), minlength=pool).int()
    refs[order[at]] = 1                                     # a page that another table holds
    # of a group's beams the better ones are chosen more often; one in twenty ends
    pick = (torch.rand(len(texts), beams, generator=g, device="cuda") ** 1.5 * beams).int().clamp_(max=beams - 1)
    parent = pick + (torch.arange(len(texts), device="cuda") * beams)[:, None]
    parent[torch.rand(parent.shape, generator=g, device="cuda") < 0.05] = -1
    parent = parent.reshape(-1).int()
    new = torch.where(parent >= 0, case["new"], 0).int()
    caches = [_filled_cache((pool, case["kv_heads"], page, case["dim"]), g) + _filled_cache((pool, case["kv_heads"], page, case["dim"]), g)
              for _ in range(case["layers"])]
    caches = [(k, v, ks, vs) for k, ks, v, vs in caches]
    return dict(case=case, table=table, kv_len=kv_len, refs=refs, parent=parent, new=new, caches=caches)


def _prepare_compact(case, g):
    pages, seqs = case["pages"], case["seqs"]
    used = torch.randperm(pages, generator=g, device="cuda")[:max(1, int(pages * case["used"]))].int()
    # the sequences have all used pages between them, the first a quarter of them twice over
    each = -(-len(used) // seqs)
    table = torch.full((seqs, each + 3), -1, dtype=torch.int32, device="cuda")
    flat = torch.full((seqs * each,), -1, dtype=torch.int32, device="cuda")
    flat[:len(used)] = used
    table[:, :each] = flat.view(seqs, each)
    if seqs > 1:
        shared = each // 4
        table[1:, :shared] = torch.where(table[1:, :shared] >= 0, table[:1, :shared], -1)
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    caches = []
    for _ in range(case["layers"]):
        (k, ks), (v, vs) = (_filled_cache((pages, case["kv_heads"], case["page"], case["dim"]), g) for _ in range(2))
        caches.append((k, v, ks, vs))
    return dict(case=case, table=table, refs=refs, caches=caches)


def _prepare_attention(case, g):
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    page, Hq, Hkv, D = case["page"], case["q_heads"], case["kv_heads"], case["dim"]
    pages = [-(-t // page) for t in total]
    wide, pool = max(pages), sum(pages) + 3
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((case["seqs"], wide), -1, dtype=torch.int32, device="cuda")
    first = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[first:first + n]
        first += n
    s = dict(case=case, table=table, max_rows=max(new), max_kv_len=max(total))
    s["kv_len"] = torch.tensor(total, dtype=torch.int32).cuda()
    s["row_start"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32).cuda()
    k, ks = _filled_cache((pool, Hkv, page, D), g)
    rows = sum(new)
    # the rows of a sequence are neighbours in a text: their queries are alike
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"), output_size=rows)
    q = torch.randn(len(new), Hq, D, generator=g, device="cuda")[seq] + 0.7 * torch.randn(rows, Hq, D, generator=g, device="cuda")
    s["q"] = q.to(DTYPE[case["dtype"]])
    if case["kind"] == "choose":
        s["cache"] = (k, k, ks, ks)                         # the values are not looked at
        lo_hi, scale = torch.empty(pool, Hkv, 2, D, dtype=torch.int8, device="cuda"), torch.empty(pool, Hkv, device="cuda")
        step = max(1, (1 << 27) // (Hkv * page * D))
        filled = torch.full((pool,), page, device="cuda")
        for p in range(0, pool, step):
            lo_hi[p:p + step], scale[p:p + step] = _bounds(k[p:p + step], ks[p:p + step], filled[p:p + step])
        s["bounds"] = (lo_hi, scale)
        return s
    v, vs = _filled_cache((pool, Hkv, page, D), g)
    s["cache"] = (k, v, ks, vs)
    # neighbours choose much the same pages: the text's first, their own, and those that score best
    place = s["kv_len"].long()[seq] - s["row_start"].long().diff()[seq] + torch.arange(rows, device="cuda") - s["row_start"].long()[seq]
    mine = place // page
    base = torch.randn(len(new), Hkv, wide, generator=g, device="cuda")
    chosen = torch.full((rows, Hkv, case["count"]), -1, dtype=torch.int32, device="cuda")
    n = min(case["count"], wide)
    step = max(1, (1 << 27) // (Hkv * wide))
    for r in range(0, rows, step):
        score = base[seq[r:r + step]] + 0.4 * torch.randn(len(mine[r:r + step]), Hkv, wide, generator=g, device="cuda")
        block = torch.arange(wide, device="cuda")
        score[:, :, 0] = 100.0
        score.masked_fill_((block == mine[r:r + step, None])[:, None], 200.0)
        score.masked_fill_((block > mine[r:r + step, None])[:, None], -math.inf)
        value, at = score.topk(n, -1)
        at = torch.where(value > -math.inf, at, wide).sort(-1).values
        chosen[r:r + step, :, :n] = torch.where(at < wide, at, -1).int()
    s["chosen"] = chosen
    return s


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if not own:
        return {"beam": _plain_beam, "fork": _plain_fork, "compact": _plain_compact, "choose": _plain_choose, "sparse": _plain_sparse}[kind](s)
    from ogle_b200 import lm
    if kind == "beam":
        return lm.beam_step(s["logits"], s["scores"], case["beams"], case["count"], ends=s["ends"])
    if kind == "fork":
        table, kv_len, refs, copies, state = lm.advance_pages(s["table"], s["kv_len"], s["parent"], s["new"], s["refs"], case["page"])
        lm.copy_pages(s["caches"], copies)
        return table, kv_len, refs, copies, state, *(t for c in s["caches"] for t in c)
    if kind == "compact":
        table, refs, copies, state = lm.compact_pages(s["table"], s["refs"], case["most"], case["page"])
        lm.copy_pages(s["caches"], copies)
        return table, refs, copies, state, *(t for c in s["caches"] for t in c)
    batch = (s["table"], s["kv_len"], s["max_kv_len"], s["row_start"], s["max_rows"])
    if kind == "choose":
        lm.page_bounds(s["cache"], s["bounds"], *batch)
        return (lm.choose_pages(s["q"], s["cache"], s["bounds"], *batch, count=case["count"]), *s["bounds"])
    return lm.sparse_attention(s["q"], s["cache"], s["chosen"], *batch)


# ---- plain forms

def _plain_beam(s):
    case = s["case"]
    G, B, V, n = case["groups"], case["beams"], case["vocab"], case["count"]
    # in 64 bits: which of two beams' tokens comes first may hang on the last bits of their sums
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    x -= torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    log_sum = x.exp().sum(1, keepdim=True).log()
    x = (s["scores"].double()[:, None] - log_sum).add(x)
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x).view(G, B * V)
    value, at = torch.sort(x, dim=1, descending=True, stable=True)      # of equal ones the first stays first
    value, at = value[:, :n], at[:, :n]
    there = value > -math.inf
    beam = torch.where(there, at // V, -1).int()
    token = torch.where(there, at % V, -1).int()
    goes_on = there & ~(token[..., None] == s["ends"]).any(-1)
    rank = goes_on.long().cumsum(1) - 1
    slot = torch.where(goes_on & (rank < B), rank, B)       # behind the last: dropped
    base = torch.arange(G, device=x.device)[:, None] * B
    parent = torch.full((G, B + 1), -1, dtype=torch.int32, device=x.device).scatter_(1, slot, (base + beam).int())[:, :B]
    last = torch.full((G, B + 1), -1, dtype=torch.int32, device=x.device).scatter_(1, slot, token)[:, :B]
    score = torch.full((G, B + 1), -math.inf, device=x.device).scatter_(1, slot, value.float())[:, :B]
    return value.float(), beam, token, parent.reshape(-1), last.reshape(-1), score.reshape(-1)


def _plain_fork(s):
    case, table, refs = s["case"], s["table"].long(), s["refs"].long()
    page, wide, pool = case["page"], s["table"].shape[1], len(s["refs"])
    parent, new = s["parent"].long(), s["new"].long()
    alive = parent >= 0
    length = torch.where(alive, s["kv_len"].long()[parent.clamp(min=0)], 0)
    col = torch.arange(wide, device=table.device)
    old = torch.where(alive[:, None], table[parent.clamp(min=0)], -1)
    full = (length // page)[:, None]
    out = torch.where(col < full, old, -1)
    # the page that is half full: the first text that goes on from it keeps it, if nobody else has it
    half = (col == full) & (length % page > 0)[:, None] & (old >= 0)
    number = torch.arange(len(parent), device=table.device)
    first = torch.full((len(s["kv_len"]),), len(parent), device=table.device).scatter_reduce_(0, parent.clamp(min=0), torch.where(alive, number, len(parent)), "amin")
    keeps = half & (first[parent.clamp(min=0)] == number)[:, None] & (refs[old.clamp(min=0)] == 1)
    out = torch.where(keeps, old, out)
    copied = half & ~keeps
    wants = copied | (col >= -(-length // page)[:, None]) & (col < -(-(length + new) // page)[:, None])
    free = torch.nonzero(refs == 0)[:, 0]
    rank = wants.reshape(-1).long().cumsum(0).view(wants.shape) - 1
    granted = wants & (rank < len(free))
    if len(free):
        out = torch.where(granted, free[rank.clamp(0, len(free) - 1)], out)
    now = refs - torch.bincount(table[table >= 0], minlength=pool) + torch.bincount(out[out >= 0], minlength=pool)
    done = copied & granted
    src, dst = torch.where(done, old, -1).amax(1), torch.where(done, out, -1).amax(1)
    tokens = torch.where(src >= 0, length % page, 0)
    copies = torch.stack([src, dst, tokens], 1).int()
    state = torch.stack([(now == 0).sum(), (wants & ~granted).sum()]).int()
    _plain_copies(s, copies)
    return out.int(), (length + new).int(), now.int(), copies, state, *(t for c in s["caches"] for t in c)


def _plain_compact(s):
    case, table, refs = s["case"], s["table"].long(), s["refs"]
    used = refs != 0
    n = used.sum()
    at = torch.arange(len(refs), device=refs.device)
    src = at[used & (at >= n)][:case["most"]]
    dst = at[~used & (at < n)][:case["most"]]
    move = at.clone()
    move[src] = dst
    out = torch.where(table >= 0, move[table.clamp(min=0)], table)
    now = refs.clone()
    now[dst] = refs[src]
    now[src] = 0
    copies = torch.tensor([-1, -1, 0], dtype=torch.int32, device=refs.device).repeat(case["most"], 1)
    copies[:len(src)] = torch.stack([src, dst, torch.full_like(src, case["page"])], 1).int()
    state = torch.stack([n, (used & (at >= n)).sum() - len(src)]).int()
    _plain_copies(s, copies)
    return out.int(), now, copies, state, *(t for c in s["caches"] for t in c)


def _plain_copies(s, copies):
    there = copies[:, 0] >= 0
    src, dst, tokens = (copies[there, i].long() for i in range(3))
    slot = torch.arange(s["case"]["page"], device=src.device)
    moved = (slot < tokens[:, None])[:, None, :, None]
    for k, v, ks, vs in s["caches"]:
        for t in (k, v):
            b = t.view(torch.uint8)
            b[dst] = torch.where(moved, b[src], b[dst])
        ks[dst] = ks[src]
        vs[dst] = vs[src]


def _bounds(k, k_scale, filled):
    """Whole-number bounds of the first filled[p] keys of pages k [pages][heads][page][dim] in every element, and their unit."""
    x = k.float()
    there = (torch.arange(k.shape[2], device=k.device) < filled[:, None])[:, None, :, None] & ~torch.isnan(x)
    top = torch.where(there, x.abs(), 0.0).amax((2, 3))
    unit = _power_of_two_scale(top, 127)
    any_there = there.any(2)
    lo = torch.where(any_there, torch.where(there, x, math.inf).amin(2), 0.0)
    hi = torch.where(any_there, torch.where(there, x, -math.inf).amax(2), 0.0)
    lo, hi = torch.floor(lo / unit[..., None]), torch.ceil(hi / unit[..., None])
    return torch.stack([lo, hi], 2).to(torch.int8), unit * k_scale


def _rows(s):
    """Sequence and position in it of each row of the call."""
    start, length = s["row_start"].long(), s["kv_len"].long()
    n = start.diff()
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n, output_size=s["q"].shape[0])
    return seq, length[seq] - n[seq] + torch.arange(s["q"].shape[0], device=n.device) - start[seq]


def _plain_choose(s):
    case, table = s["case"], s["table"].long()
    lo_hi, unit = s["bounds"]
    page, count, wide, Hkv = case["page"], case["count"], table.shape[1], case["kv_heads"]
    k, _, ks, _ = s["cache"]
    # the pages that the rows were appended to
    length, n = s["kv_len"].long(), s["row_start"].long().diff()
    block = torch.arange(wide, device=table.device)
    fresh = (block >= ((length - n) // page)[:, None]) & (block <= ((length - 1) // page)[:, None])
    at = table[fresh]
    filled = (length[:, None] - block * page).clamp(max=page)[fresh]
    for i in range(0, len(at), 4096):
        lo_hi[at[i:i + 4096]], unit[at[i:i + 4096]] = _bounds(k[at[i:i + 4096]], ks[at[i:i + 4096]], filled[i:i + 4096])
    seq, place = _rows(s)
    q = s["q"].float().view(len(seq), Hkv, -1, case["dim"])
    q = torch.where(torch.isfinite(q), q, 0.0)
    step = _power_of_two_scale(q.abs().amax((2, 3)), 127)
    q = torch.round(q / step[..., None, None]).clamp(-127, 127)
    # sequences side by side, each with as many rows as the one that has most
    B, most, G = len(table), s["max_rows"], q.shape[2]
    row = torch.arange(len(seq), device=table.device) - s["row_start"].long()[seq]
    x = q.new_zeros(B, most, Hkv, G, case["dim"])
    x[seq, row] = q
    x = x.permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * most, case["dim"])
    t = table.clamp(min=0)
    both = lo_hi[t].float().permute(0, 2, 3, 4, 1).reshape(B * Hkv, 2, case["dim"], wide)
    # products of whole numbers below 128, sums below 2^24: nothing is rounded
    dot = torch.bmm(x.clamp(min=0), both[:, 1])
    dot += torch.bmm(x.clamp(max=0), both[:, 0])
    dot = dot.view(B, Hkv, G, most, wide).amax(2)
    dot *= unit[t].transpose(1, 2)[:, :, None]
    score = dot.transpose(1, 2)[seq, row]                   # [rows][heads][blocks]
    mine = (place // page)[:, None, None]
    score.masked_fill_((block == 0) | (block == mine), math.inf)
    score.masked_fill_((block > mine) | (table < 0)[seq][:, None], -math.inf)
    value, order = torch.sort(score, dim=-1, descending=True, stable=True)
    value, order = value[..., :count], order[..., :count]
    order = torch.where(value > -math.inf, order, wide).sort(-1).values
    chosen = torch.full((len(seq), Hkv, count), -1, dtype=torch.int32, device=table.device)
    chosen[..., :order.shape[-1]] = torch.where(order < wide, order, -1).int()
    return chosen, lo_hi, unit


def _plain_sparse(s):
    case, table, chosen = s["case"], s["table"].long(), s["chosen"].long()
    page, D, Hkv, count = case["page"], case["dim"], case["kv_heads"], case["count"]
    k_cache, v_cache, ks, vs = s["cache"]
    seq, place = _rows(s)
    q = s["q"].float().view(len(seq), Hkv, -1, D)
    out, lse = torch.empty_like(s["q"]), torch.empty(s["q"].shape[:2], device=q.device)
    heads = torch.arange(Hkv, device=q.device)[:, None]
    step = max(1, (1 << 28) // (Hkv * count * page * D))
    for r in range(0, len(seq), step):
        c = chosen[r:r + step]
        at = torch.gather(table[seq[r:r + step]][:, None].expand(-1, Hkv, -1), 2, c.clamp(min=0))
        there = (c >= 0) & (at >= 0)
        at = at.clamp(min=0)

        def keys(cache, scale):
            return (cache.view(torch.uint8)[at, heads].view(cache.dtype).float() * scale[at, heads][..., None, None]).flatten(2, 3)

        j = (c[..., None] * page + torch.arange(page, device=q.device))
        hidden = (~there[..., None] | (j > place[r:r + step, None, None, None])).flatten(2)
        score = torch.matmul(q[r:r + step], keys(k_cache, ks).transpose(2, 3)) * D ** -0.5
        score.masked_fill_(hidden[:, :, None], -math.inf)
        top = score.amax(-1, keepdim=True)
        top = torch.where(top > -math.inf, top, 0.0)
        score = (score - top).exp()
        total = score.sum(-1, keepdim=True)
        o = torch.matmul(score, keys(v_cache, vs)) / torch.where(total > 0, total, 1.0)
        out[r:r + step] = o.flatten(1, 2).to(out.dtype)
        lse[r:r + step] = (top + total.log())[..., 0].flatten(1)
    return out, lse


# ---- definitions in 64 bits, written apart from the plain forms

def exact(case, seed):
    s = prepare(case, seed)
    return {"beam": _exact_beam, "fork": _exact_fork, "compact": _exact_compact, "choose": _exact_choose, "sparse": _exact_sparse}[case["kind"]](case, s)


def _exact_beam(case, s):
    G, B, V, n = case["groups"], case["beams"], case["vocab"], case["count"]
    ends = set(s["ends"].tolist())
    out = [[] for _ in range(6)]
    for g in range(G):
        found = []
        for b in range(B):
            score = float(s["scores"][g * B + b])
            if score == -math.inf:
                continue
            x = s["logits"][g * B + b].double()
            norm = float(torch.logsumexp(x, 0))
            # whatever equals the n-th largest logit is looked at: ties go to the lowest token
            cut = x.topk(min(n, V)).values[-1]
            for t in torch.nonzero((x >= cut) & (x > -math.inf))[:, 0].tolist()[:4096]:
                found.append((-(score - norm + float(x[t])), b, t))
        found.sort()
        found = found[:n]
        missing = n - len(found)
        out[0] += [-f[0] for f in found] + [-math.inf] * missing
        out[1] += [f[1] for f in found] + [-1] * missing
        out[2] += [f[2] for f in found] + [-1] * missing
        going = [f for f in found if f[2] not in ends][:B]
        missing = B - len(going)
        out[3] += [g * B + f[1] for f in going] + [-1] * missing
        out[4] += [f[2] for f in going] + [-1] * missing
        out[5] += [-f[0] for f in going] + [-math.inf] * missing
    dtypes = (torch.float64, torch.int32, torch.int32, torch.int32, torch.int32, torch.float64)
    shapes = ((G, n), (G, n), (G, n), (-1,), (-1,), (-1,))
    return tuple(torch.tensor(o, dtype=d).view(shape).cuda() for o, d, shape in zip(out, dtypes, shapes))


def _exact_copies(case, s, copies):
    for src, dst, tokens in copies:
        if src < 0:
            continue
        for k, v, ks, vs in s["caches"]:
            for t in (k, v):
                t.view(torch.uint8)[dst, :, :tokens] = t.view(torch.uint8)[src, :, :tokens]
            ks[dst], vs[dst] = ks[src], vs[src]


def _exact_fork(case, s):
    page, table = case["page"], s["table"].tolist()
    wide, refs, length = len(table[0]), s["refs"].tolist(), s["kv_len"].tolist()
    now = list(refs)
    for row in table:
        for p in row:
            if p >= 0:
                now[p] -= 1
    free = iter([p for p, r in enumerate(refs) if r == 0])
    tables, lengths, copies, missing, kept = [], [], [], 0, set()
    for parent, new in zip(s["parent"].tolist(), s["new"].tolist()):
        old = length[parent] if parent >= 0 else 0
        row, copy = [-1] * wide, (-1, -1, 0)
        for c in range(min(wide, -(-(old + new) // page))):
            here = table[parent][c] if c * page < old else None
            if here is not None and (here < 0 or (c + 1) * page <= old or refs[here] == 1 and parent not in kept):
                row[c] = here
                if (c + 1) * page > old and here >= 0:
                    kept.add(parent)
                continue
            row[c] = next(free, -1)
            missing += row[c] < 0
            if here is not None and row[c] >= 0:
                copy = (here, row[c], old - c * page)
        for p in row:
            if p >= 0:
                now[p] += 1
        tables.append(row)
        lengths.append(old + new)
        copies.append(copy)
    _exact_copies(case, s, copies)
    whole = [torch.tensor(v, dtype=torch.int32).cuda() for v in (tables, lengths, now, copies, [now.count(0), missing])]
    return (*whole, *(t.double() for c in s["caches"] for t in c))


def _exact_compact(case, s):
    refs, table = s["refs"].tolist(), s["table"].tolist()
    used = sum(r != 0 for r in refs)
    pairs = list(zip([p for p in range(used, len(refs)) if refs[p] != 0], [p for p in range(used) if refs[p] == 0]))
    left = len(pairs) - min(len(pairs), case["most"])
    pairs = pairs[:case["most"]]
    to = dict(pairs)
    for a, b in pairs:
        refs[b], refs[a] = refs[a], 0
    copies = [(a, b, case["page"]) for a, b in pairs] + [(-1, -1, 0)] * (case["most"] - len(pairs))
    _exact_copies(case, s, copies)
    whole = [torch.tensor(v, dtype=torch.int32).cuda() for v in ([[to.get(p, p) for p in row] for row in table], refs, copies, [used, left])]
    return (*whole, *(t.double() for c in s["caches"] for t in c))


def _exact_choose(case, s):
    new, past = _lengths(case)
    page, count, Hkv, D = case["page"], case["count"], case["kv_heads"], case["dim"]
    lo_hi, unit = (t.clone() for t in s["bounds"])
    k, _, ks, _ = s["cache"]
    chosen = torch.full((sum(new), Hkv, count), -1, dtype=torch.int32)
    first = 0
    if sum(n * (n + p) // page for n, p in zip(new, past)) * case["q_heads"] * D > 4e9 or sum(n * ((n + p) // page + 1) for n, p in zip(new, past)) * Hkv > 5e6:
        return None
    for b, (n, p) in enumerate(zip(new, past)):
        blocks = -(-(n + p) // page)
        at = s["table"][b, :blocks].long()
        for c in range(p // page, blocks):
            x = k[at[c], :, :min(page, n + p - c * page)].double()
            need = x.abs().amax((1, 2)) / 127
            t = torch.where(need > 0, torch.exp2(torch.ceil(torch.log2(need.clamp(min=1e-30)))), torch.ones_like(need))
            lo_hi[at[c], :, 0] = torch.floor(x.amin(1) / t[:, None]).to(torch.int8)
            lo_hi[at[c], :, 1] = torch.ceil(x.amax(1) / t[:, None]).to(torch.int8)
            unit[at[c]] = (t * ks[at[c]].double()).float()
        bound, scale = lo_hi[at].double(), unit[at].double()
        for r in range(n):
            q = s["q"][first + r].double().view(Hkv, -1, D)
            t = torch.exp2(torch.ceil(torch.log2(q.abs().amax((1, 2)) / 127)))
            q = torch.round(q / t[:, None, None])
            mine = (p + r) // page
            # the larger of both products is the one with the bound on the query's side
            dot = torch.stack([torch.maximum(q[:, h, None] * bound[:mine + 1, :, 0].transpose(0, 1), q[:, h, None] * bound[:mine + 1, :, 1].transpose(0, 1)).sum(-1)
                               for h in range(q.shape[1])]).amax(0)
            score = (dot * scale[:mine + 1].T).cpu().numpy()
            for h in range(Hkv):
                always = {0, mine}
                order = sorted((c for c in range(mine + 1) if c not in always), key=lambda c: (-score[h, c], c))
                have = sorted(list(always) + order[:max(0, count - len(always))])
                chosen[first + r, h, :len(have)] = torch.tensor(have, dtype=torch.int32)
        first += n
    return chosen.cuda(), lo_hi, unit.double()


def _exact_sparse(case, s):
    new, past = _lengths(case)
    page, Hkv, D, G = case["page"], case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    if 4 * sum(new) * case["q_heads"] * case["count"] * page * D > 4e12 or sum(new) * Hkv > 20000:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    k_cache, v_cache, ks, vs = s["cache"]
    chosen = s["chosen"].cpu()
    row = 0
    for b, (n, p) in enumerate(zip(new, past)):
        for r in range(n):
            for h in range(Hkv):
                blocks = chosen[row, h]
                blocks = blocks[blocks >= 0].long().cuda()
                at = s["table"][b].long()[blocks]
                j = (blocks[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
                seen = j <= p + r
                k = (k_cache.view(torch.uint8)[at, h].view(k_cache.dtype).double() * ks[at, h].double()[:, None, None]).reshape(-1, D)[seen]
                v = (v_cache.view(torch.uint8)[at, h].view(v_cache.dtype).double() * vs[at, h].double()[:, None, None]).reshape(-1, D)[seen]
                score = s["q"][row, h * G:(h + 1) * G].double() @ k.T / math.sqrt(D)
                lse[row, h * G:(h + 1) * G] = torch.logsumexp(score, -1)
                out[row, h * G:(h + 1) * G] = torch.softmax(score, -1) @ v
            row += 1
    return out, lse
