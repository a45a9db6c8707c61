"""Performance cases of the operators of a decoding step: keys and values appended to a paged 8-bit cache, attention over
that cache, and the adjustment of logits before a token is chosen.

A case is a dict of plain values. `listed()` gives the named ones, `draw(rng)` one more of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass through one operator - the framework's
call where `own` is set, else elementary torch operations in 32 bits - `work(case)` the bytes and operations a pass cannot do
without, and `exact(case, seed)` the same results from the definition in 64 bits.

Kinds:
  append   lm.append: rotation of new queries and keys, keys and values quantised into their pages
  attend   lm.attention: softmax attention of the new rows over the cache
  logits   lm.adjust_logits: repeated-token penalties, sparse biases and grammar masks

The cache is e4m3 [pages][kv heads][page tokens][head dim] with one power-of-two scale for each page and head. Sequence b
has rows row_start[b]..row_start[b + 1] of the call and kv_len[b] tokens in the cache once they are in it.
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
        # one user's chat, the next token: the smallest call there is
        dict(name="append_one", kind="append", seqs=1, new=1, past=700, q_heads=32, kv_heads=8, dim=128, rotary=128, paired=False,
             page=64, dtype="bf16"),
        # a serving batch's next tokens, pages of 16, interleaved pairs over half of a head
        dict(name="append_step_96", kind="append", seqs=96, new=1, past=2000, q_heads=16, kv_heads=4, dim=64, rotary=32, paired=True,
             page=16, dtype="fp32"),
        # prompts of many users admitted together, of all lengths
        dict(name="append_prompts", kind="append", seqs=13, new=4000, past=500, q_heads=32, kv_heads=8, dim=128, rotary=128,
             paired=False, page=64, dtype="bf16"),
        # one short chat, the next token: latency
        dict(name="attend_one", kind="attend", seqs=1, new=1, past=700, q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # the ordinary serving batch, lengths of all kinds
        dict(name="attend_step_64", kind="attend", seqs=64, new=1, past=8000, q_heads=32, kv_heads=8, dim=128, page=64, window=0,
             dtype="bf16"),
        # the framework's own activations are fp32: small heads, small pages
        dict(name="attend_fp32_40", kind="attend", seqs=40, new=1, past=2500, q_heads=16, kv_heads=4, dim=64, page=16, window=0,
             dtype="fp32"),
        # a few documents of great length, many query heads to a key head
        dict(name="attend_long_3", kind="attend", seqs=3, new=1, past=200000, q_heads=32, kv_heads=2, dim=128, page=128, window=0,
             dtype="fp16"),
        # drafted tokens checked together, sliding window, wide heads
        dict(name="attend_draft_window", kind="attend", seqs=24, new=5, past=20000, q_heads=8, kv_heads=4, dim=256, page=32, window=4096,
             dtype="bf16"),
        # prompts in chunks over what is in the cache already
        dict(name="attend_prompts", kind="attend", seqs=6, new=2000, past=2500, q_heads=32, kv_heads=8, dim=128, page=64, window=0,
             dtype="bf16"),
        # one user's next token under a grammar
        dict(name="logits_one", kind="logits", rows=1, vocab=32000, history=800, biases=20, masked=True, dtype="fp32", out="fp32"),
        # a serving batch without grammar: penalties and biases
        dict(name="logits_step_64", kind="logits", rows=64, vocab=128001, history=4000, biases=100, masked=False, dtype="bf16", out="fp32"),
        # a large batch of constrained answers
        dict(name="logits_grammar_400", kind="logits", rows=400, vocab=150000, history=1000, biases=10, masked=True, dtype="fp16", out="fp16"),
    ]


def _near(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "logits"])
    if kind == "logits":
        while True:
            case = dict(kind=kind, rows=_near(rng, 1, 400), vocab=_near(rng, 2000, 150000), history=_near(rng, 1, 8000),
                        biases=_near(rng, 1, 300) - 1, masked=rng.random() < 0.5, dtype=rng.choice(["fp32", "fp16", "bf16"]))
            case["out"] = rng.choice([case["dtype"], "fp32"])
            if case["rows"] * case["vocab"] * (SIZE[case["dtype"]] + SIZE[case["out"]]) <= 400 * 150000 * 4:
                return case
    while True:
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        case = dict(kind=kind, seqs=_near(rng, 1, 128), new=rng.choice([1, 1, 1, rng.randint(2, 8), _near(rng, 9, 4000)]),
                    past=_near(rng, 1, 200000), q_heads=kv_heads * rng.choice([1, 2, 3, 4, 6, 8, 16]), kv_heads=kv_heads,
                    dim=rng.choice([64, 80, 96, 128, 128, 256]), page=rng.choice([16, 32, 64, 128, 256]),
                    dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]))
        if kind == "append":
            case["rotary"] = rng.choice([case["dim"], case["dim"], case["dim"] // 2, 0])
            case["paired"] = rng.random() < 0.3
            if case["past"] > 4000:
                continue
            if work(case)["bytes"] <= work(listed()[2])["bytes"]:
                return case
        else:
            case["window"] = rng.choice([0, 0, 0, _near(rng, 100, 8000)])
            span = case["new"] + case["past"]
            score = case["seqs"] * case["q_heads"] * case["new"] * span
            cache = case["seqs"] * case["kv_heads"] * case["dim"] * span
            # no dearer than the listed ones: the plain form holds every score, and every key in 32 bits
            if score <= 6 * 32 * 2000 * 4500 and cache <= 64 * 8 * 128 * 8001 and (case["new"] > 8 or cache >= 10000):
                if work(case)["flops"] <= work(listed()[8])["flops"]:
                    return case


def _lengths(case):
    """(new rows, earlier tokens) of each sequence: known to the host, as a scheduler knows them. The first has the most; the others
    go by their number."""
    r = random.Random(case["seqs"] * 1000003 + case["new"] * 1009 + case["past"])
    new = [case["new"]] + [r.randint(max(1, case["new"] // 8), case["new"]) for _ in range(case["seqs"] - 1)]
    past = [case["past"]] + [r.randint(min(1, case["past"]), case["past"]) for _ in range(case["seqs"] - 1)]
    return new, past


def _keys_read(case):
    """Cached tokens that some row of each sequence attends, and pairs of row and key, both summed over the sequences."""
    new, past = _lengths(case)
    keys = pairs = 0
    for n, p in zip(new, past):
        w = case["window"]
        keys += n + p - (max(0, p - w + 1) if w else 0)
        pairs += sum(min(p + i + 1, w) if w else p + i + 1 for i in range(n)) if n <= 64 or w else n * p + n * (n + 1) // 2
    return keys, pairs


def work(case):
    if case["kind"] == "logits":
        n = case["rows"] * case["vocab"]
        data = n * (SIZE[case["dtype"]] + SIZE[case["out"]]) + case["rows"] * (4 * case["history"] + 8 * case["biases"] + 12)
        return {"bytes": data + (case["rows"] * -(-case["vocab"] // 32) * 4 if case["masked"] else 0), "flops": 0}
    new, past = _lengths(case)
    rows, size, kv = sum(new), SIZE[case["dtype"]], case["kv_heads"] * case["dim"]
    if case["kind"] == "append":
        pages = sum((p + n - 1) // case["page"] - p // case["page"] + 1 for n, p in zip(new, past))
        return {"bytes": rows * (2 * case["q_heads"] * case["dim"] * size + 2 * kv * (size + 1) + 4 * case["rotary"])
                + pages * 2 * case["kv_heads"] * 4, "flops": 3 * rows * case["rotary"] * (case["q_heads"] + case["kv_heads"])}
    keys, pairs = _keys_read(case)
    pages = keys / case["page"]
    return {"bytes": rows * case["q_heads"] * (2 * case["dim"] * size + 4) + keys * 2 * kv + pages * (8 * case["kv_heads"] + 4),
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


def _power_of_two_scale(amax):
    """The smallest power of two s with amax <= 448 s (1 where there is nothing)."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875)), torch.ones_like(amax))


def _filled_cache(shape, g):
    """Random keys or values as a running service has them: a page's head has its own amplitude, a few channels are larger."""
    pages, heads, page, dim = shape
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp2(0.7 * torch.randn(pages, heads, 1, 1, generator=g, device="cuda"))
    x *= 1 + 2 * (torch.rand(1, heads, 1, dim, generator=g, device="cuda") < 0.03)
    scale = _power_of_two_scale(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPE[case["dtype"]]
    if kind == "logits":
        R, V, H = case["rows"], case["vocab"], case["history"]
        s = dict(case=case)
        s["logits"] = (4 * torch.randn(R, V, generator=g, device="cuda")).to(dtype)
        count = torch.randint(H // 2, H + 1, (R,), generator=g, device="cuda")
        count[0] = H
        s["token_start"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
        n = int(count.sum())
        # a text repeats its frequent words: squared uniform numbers crowd at the low tokens
        s["tokens"] = (torch.rand(n, generator=g, device="cuda") ** 3 * V).int().clamp_(max=V - 1)
        s["prompt_len"] = (count // 2).int()
        s["repetition"] = 1 + 0.3 * torch.rand(R, generator=g, device="cuda")
        s["presence"] = 0.5 * torch.rand(R, generator=g, device="cuda")
        s["frequency"] = 0.2 * torch.rand(R, generator=g, device="cuda")
        B = case["biases"]
        s["bias_start"] = (torch.arange(R + 1, device="cuda") * B).int() if B else None
        s["bias_token"] = torch.rand(R, V, generator=g, device="cuda").topk(B, dim=1).indices.reshape(-1).int() if B else None
        s["bias_value"] = 5 * torch.randn(R * B, generator=g, device="cuda") if B else None
        if case["masked"]:
            bits = torch.randint(-2 ** 31, 2 ** 31, (2, R, -(-V // 32)), generator=g, device="cuda")
            s["allowed"] = (bits[0] & bits[1]).int()      # a quarter of the tokens may follow
        else:
            s["allowed"] = None
        return s
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    page, Hq, Hkv, D = case["page"], case["q_heads"], case["kv_heads"], case["dim"]
    pages = [-(-t // page) for t in total]
    wide = max(pages)
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((case["seqs"], wide), -1, dtype=torch.int32, device="cuda")
    first = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[first:first + n]
        first += n
    s = dict(case=case, table=table, max_rows=max(new), max_kv_len=max(total))
    s["kv_len"] = torch.tensor(total, dtype=torch.int32).cuda()
    s["row_start"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32).cuda()
    s["k_cache"], s["k_scale"] = _filled_cache((pool, Hkv, page, D), g)
    s["v_cache"], s["v_scale"] = _filled_cache((pool, Hkv, page, D), g)
    rows = sum(new)
    if kind == "append":
        # as one projection leaves them: queries, keys and values of a row side by side
        qkv = torch.randn(rows, Hq + 2 * Hkv, D, generator=g, device="cuda").to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        if case["rotary"]:
            half = case["rotary"] // 2
            angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            s["rotary"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        else:
            s["rotary"] = None
    else:
        s["q"] = (1.5 * torch.randn(rows, Hq, D, generator=g, device="cuda")).to(dtype)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        from ogle_b200 import lm
        if kind == "logits":
            return lm.adjust_logits(s["logits"], s["tokens"], s["token_start"], s["prompt_len"], s["repetition"], s["presence"],
                                    s["frequency"], s["bias_token"], s["bias_value"], s["bias_start"], s["allowed"],
                                    out_dtype=DTYPE[s["case"]["out"]])
        cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        if kind == "append":
            q = lm.append(s["k"], s["v"], cache, s["table"], s["kv_len"], s["max_kv_len"], s["row_start"], s["max_rows"], q=s["q"],
                          rotary=s["rotary"], interleaved=s["case"]["paired"])
            return q, *cache
        return lm.attention(s["q"], cache, s["table"], s["kv_len"], s["max_kv_len"], s["row_start"], s["max_rows"],
                            window=s["case"]["window"])
    if kind == "logits":
        return _plain_logits(s)
    return _plain_append(s) if kind == "append" else _plain_attention(s)


def _rows(s):
    """Sequence and position in it of each row of the call."""
    start, length = s["row_start"].long(), s["kv_len"].long()
    n = start.diff()
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n, output_size=s["q"].shape[0])
    return seq, length[seq] - n[seq] + torch.arange(s["q"].shape[0], device=n.device) - start[seq]


def _rotated(x, cs, paired):
    """x [rows][heads][dim] in 32 bits, its first dimensions rotated by cs [rows][rotary] = (cosines, sines)."""
    x = x.float()
    R = cs.shape[1]
    c, s = cs[:, None, :R // 2], cs[:, None, R // 2:]
    if paired:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _quantised_into(x, cache, scale, s, seq, pos):
    """x [rows][heads][dim] into its places of the cache; scales of the pages grow to what the new rows need."""
    page = cache.shape[2]
    at = s["table"].long()[seq, pos // page]
    amax = torch.zeros_like(scale).index_reduce_(0, at, x.abs().amax(-1), "amax")
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=scale.device).index_fill_(0, at, True)
    # of a sequence's pages one at most holds earlier tokens: the one its first new row goes to
    first = s["row_start"].long()[:-1]
    kept = (pos % page)[first] > 0
    old_page = at[first]
    old = torch.zeros_like(scale).index_copy_(0, old_page, scale[old_page] * kept[:, None])
    wanted = torch.where(amax > 0, _power_of_two_scale(amax), torch.zeros_like(amax))
    now = torch.maximum(old, wanted)
    now = torch.where(now > 0, now, torch.ones_like(now))
    ratio = torch.where(kept[:, None], scale[old_page] / now[old_page], torch.ones_like(now[old_page]))
    before = cache[old_page].float()
    cache[old_page] = (before * ratio[:, :, None, None]).to(cache.dtype)
    cache[at, :, pos % page] = (x / now[at][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
    scale.copy_(torch.where(touched[:, None], now, scale))


def _plain_append(s):
    seq, pos = _rows(s)
    q, k = s["q"].float(), s["k"].float()
    if s["rotary"] is not None:
        cs = s["rotary"][pos]
        q, k = _rotated(q, cs, s["case"]["paired"]), _rotated(k, cs, s["case"]["paired"])
    _quantised_into(k, s["k_cache"], s["k_scale"], s, seq, pos)
    _quantised_into(s["v"].float(), s["v_cache"], s["v_scale"], s, seq, pos)
    return q.to(s["q"].dtype), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _plain_attention(s):
    q, table, window = s["q"], s["table"].long(), s["case"]["window"]
    B, page, D, Hkv = table.shape[0], s["k_cache"].shape[2], q.shape[2], s["k_cache"].shape[1]
    G, most = q.shape[1] // Hkv, s["max_rows"]
    seq, pos = _rows(s)
    row = torch.arange(q.shape[0], device=q.device) - s["row_start"].long()[seq]
    padded = q.new_zeros(B, most, Hkv, G, D, dtype=torch.float32)
    padded[seq, row] = q.float().view(-1, Hkv, G, D)
    padded = padded.permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * most, D)
    at = table.clamp(min=0)

    def keys(cache, scale):
        x = cache[at].float() * scale[at][..., None, None]                      # [B][pages][heads][page][dim]
        return x.permute(0, 2, 1, 3, 4).reshape(B * Hkv, -1, D)

    k = keys(s["k_cache"], s["k_scale"])
    score = torch.bmm(padded, k.transpose(1, 2)).mul_(D ** -0.5).view(B, Hkv, G, most, -1)
    del k
    length = s["kv_len"].long()
    n = s["row_start"].long().diff()
    place = (length - n)[:, None] + torch.arange(most, device=q.device)         # [B][most]
    j = torch.arange(score.shape[-1], device=q.device)
    hidden = (j > place[..., None]) | (j >= length[:, None, None])
    if window:
        hidden |= j <= place[..., None] - window
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0]
    score = score.view(B * Hkv, G * most, -1)
    out = torch.bmm(score, keys(s["v_cache"], s["v_scale"])).view(B, Hkv, G, most, D) / total
    out = out.permute(0, 3, 1, 2, 4)[seq, row].reshape(q.shape).to(q.dtype)
    return out, lse.permute(0, 3, 1, 2)[seq, row].reshape(q.shape[:2])


def _plain_logits(s):
    x = s["logits"].float()
    R, V = x.shape
    start = s["token_start"].long()
    n = start.diff()
    row = torch.repeat_interleave(torch.arange(R, device=x.device), n, output_size=len(s["tokens"]))
    answer = torch.arange(len(s["tokens"]), device=x.device) - start[row] >= s["prompt_len"].long()[row]
    at = row * V + s["tokens"].long()
    seen = torch.zeros(R * V, device=x.device).index_fill_(0, at, 1.0).view(R, V) > 0
    count = torch.zeros(R * V, device=x.device).index_add_(0, at, answer.float()).view(R, V)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_token"] is not None:
        row = torch.repeat_interleave(torch.arange(R, device=x.device), s["bias_start"].long().diff(), output_size=len(s["bias_token"]))
        x = x.view(-1).index_add_(0, row * V + s["bias_token"].long(), s["bias_value"]).view(R, V)
    if s["allowed"] is not None:
        t = torch.arange(V, device=x.device)
        x = torch.where((s["allowed"][:, t // 32] >> (t % 32).int()) & 1 > 0, x, torch.full_like(x, -math.inf))
    return x.to(DTYPE[s["case"]["out"]])


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attention, "logits": _exact_logits}[case["kind"]](case, s)


def _exact_append(case, s):
    page, dtype = case["page"], s["q"].dtype
    new, past = _lengths(case)
    R = case["rotary"]

    def turned(x, p):
        x = x.double()
        if not R:
            return x
        cs = s["rotary"][p:p + x.shape[0]].double()
        z = torch.complex(cs[:, :R // 2], cs[:, R // 2:])[:, None]
        y = x.clone()
        if case["paired"]:
            w = torch.view_as_complex(x[..., :R].reshape(*x.shape[:2], R // 2, 2).contiguous()) * z
            y[..., :R] = torch.view_as_real(w).flatten(-2)
        else:
            w = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * z
            y[..., :R] = torch.cat([w.real, w.imag], -1)
        return y

    q_out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, p) in enumerate(zip(new, past)):
        rows = slice(first, first + n)
        first += n
        q_out[rows] = turned(s["q"][rows], p)
        for cache, scale, x in ((s["k_cache"], s["k_scale"], turned(s["k"][rows], p)), (s["v_cache"], s["v_scale"], s["v"][rows].double())):
            t = p
            while t < p + n:
                end = min(p + n, (t // page + 1) * page)
                at, slot = int(s["table"][b, t // page]), t % page
                part = x[t - p:end - p]
                need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((0, 2)) / E4M3_MAX)))
                if slot:
                    need = torch.maximum(need, scale[at].double())
                    earlier = cache[at, :, :slot].double() * (scale[at].double() / need)[:, None, None]
                    cache[at, :, :slot] = earlier.float().to(cache.dtype)
                    after = cache[at, :, slot + end - t:].double() * (scale[at].double() / need)[:, None, None]
                    cache[at, :, slot + end - t:] = after.float().to(cache.dtype)
                scale[at] = need.float()
                cache[at, :, slot:slot + end - t] = (part / need[:, None]).transpose(0, 1).float().to(cache.dtype)
                t = end
    return q_out, s["k_cache"].double(), s["v_cache"].double(), s["k_scale"].double(), s["v_scale"].double()


def _exact_attention(case, s):
    new, past = _lengths(case)
    D, page, Hkv = case["dim"], case["page"], case["kv_heads"]
    G = case["q_heads"] // Hkv
    if 4 * sum(n * (n + p) for n, p in zip(new, past)) * case["q_heads"] * D > 2e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, p) in enumerate(zip(new, past)):
        at = s["table"][b, :-(-(n + p) // page)].long()
        for h in range(Hkv):
            k = (s["k_cache"][at, h].double() * s["k_scale"][at, h].double()[:, None, None]).reshape(-1, D)[:n + p]
            v = (s["v_cache"][at, h].double() * s["v_scale"][at, h].double()[:, None, None]).reshape(-1, D)[:n + p]
            for g in range(h * G, h * G + G):
                score = (s["q"][first:first + n, g].double() @ k.T) / math.sqrt(D)
                ahead = torch.arange(n + p, device="cuda")[None] - torch.arange(p, p + n, device="cuda")[:, None]
                score[ahead > 0] = -math.inf
                if case["window"]:
                    score[ahead <= -case["window"]] = -math.inf
                lse[first:first + n, g] = torch.logsumexp(score, -1)
                out[first:first + n, g] = torch.softmax(score, -1) @ v
        first += n
    return out, lse


def _exact_logits(case, s):
    out = s["logits"].double()
    V = case["vocab"]
    start = s["token_start"].tolist()
    for r in range(case["rows"]):
        tokens = s["tokens"][start[r]:start[r + 1]].long()
        counts = torch.bincount(tokens[int(s["prompt_len"][r]):], minlength=V).double()
        seen = torch.bincount(tokens, minlength=V) > 0
        x, rep = out[r], s["repetition"][r].double()
        x[seen] = torch.where(x[seen] < 0, x[seen] * rep, x[seen] / rep)
        x -= counts * s["frequency"][r].double() + counts.clamp(max=1) * s["presence"][r].double()
        if case["biases"]:
            at = slice(r * case["biases"], (r + 1) * case["biases"])
            x[s["bias_token"][at].long()] += s["bias_value"][at].double()
        if case["masked"]:
            bits = (s["allowed"][r][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
            x[bits.reshape(-1)[:V] == 0] = -math.inf
    return out
