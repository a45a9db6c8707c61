"""A small language model that answers prompts with the framework's operators, as a server would use them:

    python -m ogle_b200.lm_example [--prompts 5,1,40] [--steps 12] [--layers 2] [--window 0]

Every step is one batch: a product for the queries, keys and values of its rows, `lm.append` (rotation, 8-bit pages),
`lm.attention` over each sequence's pages, a product and an addition behind it, and at the end the logits of each sequence's last
row through `lm.adjust_logits` (repeated tokens, biases, a mask of the tokens that may come). The prompts are the first step, of many
rows to a sequence; each later step has one row. Pages are handed out as sequences grow. The weights are random: what it
prints means nothing, but it does not depend on how the prompts are batched.
"""
import argparse

import torch

from . import lm, ops


class Model:
    """Random weights: embedding, layers of attention (no feed-forward part), and the embedding again for the logits."""

    def __init__(self, vocab=1000, width=256, q_heads=8, kv_heads=2, layers=2, positions=4096, window=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.vocab, self.width, self.q_heads, self.kv_heads, self.window = vocab, width, q_heads, kv_heads, window
        self.head_dim = width // q_heads
        self.qkv_width = (q_heads + 2 * kv_heads) * self.head_dim
        self.embedding = torch.randn(vocab, width, generator=g).cuda()
        self.qkv = [(2 * torch.randn(self.qkv_width, width, generator=g) / width ** 0.5).cuda() for _ in range(layers)]
        self.out = [(torch.randn(width, width, generator=g) / width ** 0.5).cuda() for _ in range(layers)]
        self.rotary = lm.rotary_table(positions, self.head_dim)

    def new_caches(self, pages, page_tokens):
        return [lm.new_cache(pages, self.kv_heads, page_tokens, self.head_dim) for _ in self.qkv]

    def rows(self, tokens, caches, batch):
        """Activations [rows, width] behind the last layer, the rows' keys and values in the caches. batch: what places the rows
        (block_table, kv_len, max_kv_len, row_start, max_rows of lm.append)."""
        x = self.embedding[tokens]
        n, h, hk, d = len(tokens), self.q_heads, self.kv_heads, self.head_dim
        for qkv, out, cache in zip(self.qkv, self.out, caches):
            y = ops.gemm_ws(x, qkv, None, n, self.width, self.qkv_width, transB=1, beta=0.0, math_mode=ops.MATH_TF32X3)
            q, k, v = y.view(n, h + 2 * hk, d).split([h, hk, hk], 1)
            q = lm.append(k, v, cache, q=q, rotary=self.rotary, **batch)
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
        x = m.rows(tokens, self.caches, batch)
        last = x[self._ints([s - 1 for s in starts[1:]]).long()]
        logits = m.logits(last)
        lengths = [len(t) for t in self.texts]
        logits = lm.adjust_logits(logits, self._ints([t for text in self.texts for t in text]), self._ints([sum(lengths[:i]) for i in range(len(lengths) + 1)]),
                                  self._ints(self.prompt_len), *self.penalties, *(self.bias or (None, None, None)), allowed=self.allowed)
        for text, t in zip(self.texts, logits.argmax(1).tolist()):
            text.append(t)
        return logits


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--prompts", default="5,1,40", help="lengths of the (random) prompts")
    p.add_argument("--steps", type=int, default=12)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--window", type=int, default=0)
    a = p.parse_args()
    model = Model(layers=a.layers, window=a.window)
    g = torch.Generator().manual_seed(1)
    answers = Answers(model, [torch.randint(1, model.vocab, (int(n),), generator=g).tolist() for n in a.prompts.split(",")])
    for _ in range(a.steps):
        answers.step()
    for text, n in zip(answers.texts, answers.prompt_len):
        print("prompt of", n, "->", *text[n:])


if __name__ == "__main__":
    main()
