"""A small language model that answers prompts with the framework's operators, as a server would use them:

    python -m ogle_b200.lm_example [--prompts 5,1,40] [--steps 12] [--layers 2] [--window 0] [--chosen 0] [--beams 0]

Every step is one batch: a product for the queries, keys and values of its rows, `lm.append` (rotation, 8-bit pages),
`lm.attention` over each sequence's pages, a product and an addition behind it, and at the end the logits of each sequence's last
row through `lm.adjust_logits` (repeated tokens, biases, a mask of the tokens that may come). The prompts are the first step, of many
rows to a sequence; each later step has one row. Pages are handed out as sequences grow. The weights are random: what it
prints means nothing, but it does not depend on how the prompts are batched.

With --chosen a row attends so many pages alone: `lm.page_bounds` behind `lm.append`, then `lm.choose_pages` and `lm.sparse_attention`.
With --beams several continuations of a prompt are followed at once: `lm.beam_step` picks them from the logits, `lm.advance_pages` makes
the block tables of the texts that go on - their full pages shared -, `lm.copy_pages` copies the pages that two of them would write to, and
`lm.compact_pages` moves what is in use to the front. Nothing in a step of the search waits for the device.
"""
import argparse

import torch

from . import lm, ops


class Model:
    """Random weights: embedding, layers of attention (no feed-forward part), and the embedding again for the logits."""

    def __init__(self, vocab=1000, width=256, q_heads=8, kv_heads=2, layers=2, positions=4096, window=0, seed=0, chosen=0):
        if window and chosen:
            raise ValueError("a window and chosen pages do not go together")
        g = torch.Generator().manual_seed(seed)
        self.vocab, self.width, self.q_heads, self.kv_heads, self.window, self.chosen = vocab, width, q_heads, kv_heads, window, chosen
        self.head_dim = width // q_heads
        self.qkv_width = (q_heads + 2 * kv_heads) * self.head_dim
        self.embedding = torch.randn(vocab, width, generator=g).cuda()
        self.qkv = [(2 * torch.randn(self.qkv_width, width, generator=g) / width ** 0.5).cuda() for _ in range(layers)]
        self.out = [(torch.randn(width, width, generator=g) / width ** 0.5).cuda() for _ in range(layers)]
        self.rotary = lm.rotary_table(positions, self.head_dim)

    def new_caches(self, pages, page_tokens):
        return [lm.new_cache(pages, self.kv_heads, page_tokens, self.head_dim) for _ in self.qkv]

    def new_bounds(self, caches):
        return [lm.new_bounds(c) for c in caches] if self.chosen else None

    def rows(self, tokens, caches, batch, bounds=None):
        """Activations [rows, width] behind the last layer, the rows' keys and values in the caches. batch: what places the rows
        (block_table, kv_len, max_kv_len, row_start, max_rows of lm.append). bounds: the caches' (new_bounds), where pages are chosen."""
        x = self.embedding[tokens]
        n, h, hk, d = len(tokens), self.q_heads, self.kv_heads, self.head_dim
        for layer, (qkv, out, cache) in enumerate(zip(self.qkv, self.out, caches)):
            y = ops.gemm_ws(x, qkv, None, n, self.width, self.qkv_width, transB=1, beta=0.0, math_mode=ops.MATH_TF32X3)
            q, k, v = y.view(n, h + 2 * hk, d).split([h, hk, hk], 1)
            q = lm.append(k, v, cache, q=q, rotary=self.rotary, **batch)
            if self.chosen:
                lm.page_bounds(cache, bounds[layer], **batch)
                chosen = lm.choose_pages(q, cache, bounds[layer], count=self.chosen, **batch)
                o, _ = lm.sparse_attention(q, cache, chosen, **batch)
            else:
                o, _ = lm.attention(q, cache, window=self.window, **batch)
            o = ops.gemm_ws(o.view(n, self.width), out, None, n, self.width, self.width, transB=1, beta=0.0, math_mode=ops.MATH_TF32X3)
            x = ops.add(x, o)
        return x

    def logits(self, x):
        return ops.gemm_ws(x, self.embedding, None, len(x), self.width, self.vocab, transB=1, beta=0.0,
                           math_mode=ops.MATH_TF32X3)[:, :self.vocab]


class Answers:
    """Texts that grow together: pages, tokens and what lm.adjust_logits is given of them."""

    def __init__(self, model, prompts, page_tokens=16, pages=256, repetition=1.3, presence=0.5, frequency=0.2, forbidden=(0,), favoured=()):
        self.model, self.page_tokens = model, page_tokens
        self.texts, self.prompt_len = [list(p) for p in prompts], [len(p) for p in prompts]
        self.free, self.pages = list(range(pages))[::-1], [[] for _ in prompts]
        self.caches = model.new_caches(pages, page_tokens)
        self.bounds = model.new_bounds(self.caches)
        n = len(prompts)
        self.penalties = [torch.full((n,), v, device="cuda") for v in (repetition, presence, frequency)]
        words = torch.full(((model.vocab + 31) // 32,), -1, dtype=torch.int32)
        for t in forbidden:
            words[t // 32] &= ~(1 << t % 32) if t % 32 < 31 else 0x7fffffff
        self.allowed = words.cuda()
        self.bias = None
        if favoured:
            self.bias = (torch.tensor([t for t, _ in favoured] * n, dtype=torch.int32).cuda(),
                         torch.tensor([v for _, v in favoured] * n, dtype=torch.float32).cuda(),
                         (torch.arange(n + 1) * len(favoured)).int().cuda())

    def _ints(self, v):
        return torch.tensor(v, dtype=torch.int32).cuda()

    def step(self):
        """Appends one token to every text: the prompts' rows if they are not in the cache yet, else the last token's."""
        m = self.model
        first = not self.pages[0]
        new = [len(t) if first else 1 for t in self.texts]
        for text, pages in zip(self.texts, self.pages):
            while len(pages) * self.page_tokens < len(text):
                pages.append(self.free.pop())
        wide = max(len(p) for p in self.pages)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        batch = dict(block_table=self._ints([p + [-1] * (wide - len(p)) for p in self.pages]), kv_len=self._ints([len(t) for t in self.texts]),
                     max_kv_len=max(len(t) for t in self.texts), row_start=self._ints(starts), max_rows=max(new))
        tokens = torch.tensor([t for text, n in zip(self.texts, new) for t in text[len(text) - n:]]).cuda()
        x = m.rows(tokens, self.caches, batch, self.bounds)
        last = x[self._ints([s - 1 for s in starts[1:]]).long()]
        logits = m.logits(last)
        lengths = [len(t) for t in self.texts]
        logits = lm.adjust_logits(logits, self._ints([t for text in self.texts for t in text]), self._ints([sum(lengths[:i]) for i in range(len(lengths) + 1)]),
                                  self._ints(self.prompt_len), *self.penalties, *(self.bias or (None, None, None)), allowed=self.allowed)
        for text, t in zip(self.texts, logits.argmax(1).tolist()):
            text.append(t)
        return logits


MOST_COUNT = 128                                # continuations that lm.beam_step finds for a group


class Search:
    """Beam search over the answers to prompts: `beams` texts of each, whose pages, scores and parents stay on the device."""

    def __init__(self, model, prompts, beams, page_tokens=16, pages=512, ends=(), steps=100):
        if not all(len(p) for p in prompts):
            raise ValueError("a prompt without a token has no next one")
        self.model, self.beams, self.page_tokens, self.prompts, self.steps = model, beams, page_tokens, [list(p) for p in prompts], steps
        self.caches = model.new_caches(pages, page_tokens)
        self.bounds = model.new_bounds(self.caches)
        self.most = max(len(p) for p in prompts) + steps          # tokens of a text
        ends = sorted(set(ends))
        self.ends = torch.tensor(ends, dtype=torch.int32).cuda() if ends else None
        # each beam may have all end tokens among the best
        self.count = min(beams * max(2, 1 + len(ends)), MOST_COUNT)
        none = torch.full((1, -(-self.most // page_tokens)), -1, dtype=torch.int32).cuda()
        lengths = [len(p) for p in prompts]
        self.refs = torch.zeros(pages, dtype=torch.int32).cuda()
        self.table, self.kv_len, self.missing = none, torch.zeros(1, dtype=torch.int32).cuda(), torch.zeros((), dtype=torch.int32).cuda()
        self._advance(torch.full((len(prompts),), -1, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
        starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        batch = dict(block_table=self.table, kv_len=self.kv_len, max_kv_len=self.most, row_start=torch.tensor(starts, dtype=torch.int32).cuda(),
                     max_rows=max(lengths))
        x = model.rows(torch.tensor([t for p in prompts for t in p]).cuda(), self.caches, batch, self.bounds)
        x = x[torch.tensor([s - 1 for s in starts[1:]]).cuda()]
        # the best tokens behind each prompt that are no end token are the first beams
        self.first = score, _, token = lm.beam_step(model.logits(x), None, 1, min(beams + len(ends), MOST_COUNT))[:3]
        goes_on = token >= 0
        if self.ends is not None:
            goes_on &= ~(token[..., None] == self.ends).any(-1)
        place = torch.where(goes_on, goes_on.cumsum(1) - 1, beams).clamp(max=beams)       # those behind the last beam have one place
        row = torch.arange(len(prompts), dtype=torch.int32).cuda()[:, None].expand_as(token)
        self.next = tuple(v.new_full((len(prompts), beams + 1), nothing).scatter(1, place, v)[:, :beams].flatten().contiguous()
                          for v, nothing in ((row, -1), (token, -1), (score, -float("inf"))))
        self.found, self.taken = [], [self.next]

    def _advance(self, row, new):
        self.table, self.kv_len, self.refs, copies, state = lm.advance_pages(self.table, self.kv_len, row, new, self.refs, self.page_tokens)
        lm.copy_pages(self.caches, copies, bounds=self.bounds)
        self.missing = self.missing + state[1]

    def step(self):
        """Appends the chosen tokens and chooses the next ones, `steps` times at most: the tables have no room for more."""
        if len(self.found) == self.steps:
            raise ValueError(f"the search was made for {self.steps} steps")
        row, token, score = self.next
        self._advance(row, (row >= 0).int())
        batch = dict(block_table=self.table, kv_len=self.kv_len, max_kv_len=self.most)
        x = self.model.rows(token.clamp(min=0).long(), self.caches, batch, self.bounds)
        found = lm.beam_step(self.model.logits(x), score, self.beams, self.count, ends=self.ends)
        self.found.append(found[:3])
        self.next = found[3:]
        self.taken.append(self.next)

    def compact(self, most=64):
        """Moves pages in use to the front of the pool, `most` at a time."""
        self.table, self.refs, copies, state = lm.compact_pages(self.table, self.refs, most, self.page_tokens)
        lm.copy_pages(self.caches, copies, bounds=self.bounds)
        return state

    def texts(self):
        """(score, tokens) of the texts that are left, the prompts' in turn; of those that have ended, too. Waits for the device."""
        if int(self.missing):
            raise RuntimeError("the pool has too few pages")
        taken = [[t.tolist() for t in step] for step in self.taken]
        ends = set(self.ends.tolist()) if self.ends is not None else set()

        def tokens(step, i):
            out = []
            for row, token, _ in reversed(taken[:step + 1]):
                out.append(token[i])
                i = row[i]
            return out[::-1]

        left = [[] for _ in self.prompts]
        for i, (row, score) in enumerate(zip(taken[-1][0], taken[-1][2])):
            if row >= 0:
                left[i // self.beams].append((score, tokens(len(taken) - 1, i)))
        ended = [[(s, [t]) for s, t in zip(*found) if t in ends] for found in zip(self.first[0].tolist(), self.first[2].tolist())]
        for step, found in enumerate(self.found):
            score, beam, token = (t.tolist() for t in found)
            for g in range(len(self.prompts)):
                for s, b, t in zip(score[g], beam[g], token[g]):
                    if b >= 0 and t in ends:
                        ended[g].append((s, tokens(step, g * self.beams + b) + [t]))
        return left, ended


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--prompts", default="5,1,40", help="lengths of the (random) prompts")
    p.add_argument("--steps", type=int, default=12)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--window", type=int, default=0)
    p.add_argument("--chosen", type=int, default=0, help="pages that a row attends (0: all)")
    p.add_argument("--beams", type=int, default=0, help="texts of a prompt that a beam search follows (0: no search)")
    a = p.parse_args()
    model = Model(layers=a.layers, window=a.window, chosen=a.chosen)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(1, model.vocab, (int(n),), generator=g).tolist() for n in a.prompts.split(",")]
    if a.beams:
        search = Search(model, prompts, a.beams, ends=(0,), steps=a.steps)
        for _ in range(a.steps - 1):
            search.step()
        search.compact()
        for prompt, left in zip(prompts, search.texts()[0]):
            for score, text in left:
                print("prompt of", len(prompt), "->", *text, "(%.2f)" % score)
        return
    answers = Answers(model, prompts)
    for _ in range(a.steps):
        answers.step()
    for text, n in zip(answers.texts, answers.prompt_len):
        print("prompt of", n, "->", *text[n:])


if __name__ == "__main__":
    main()
