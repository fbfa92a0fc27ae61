"""Chat sessions over a paged cache that is kept to a budget: the cache operators
and the sampler around a small random-weight attention model.

    python examples/paged_decode.py [--sessions 8] [--tokens 200] [--budget 128]

Prompts of different lengths go through in chunks; then every step writes its tokens'
keys and values (kv_append), attends over the cache with a window and sinks
(paged_attention), adds what each key drew to its score (kv_add_scores), applies
the penalties (adjust_logits) and samples.  A session whose cache has grown past
twice its budget is cut back to it (kv_evict), and its old pages are free again.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np
import torch

import tensormark_amd as tm

DEV = "cuda:0"


class Cache:
    """One layer's pools, and the pages and lengths of all sessions."""

    def __init__(self, sessions, pages, heads, dim, page, budget, window, sinks):
        self.page, self.budget, self.window, self.sinks = page, budget, window, sinks
        self.k = torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=DEV)
        self.v = torch.zeros_like(self.k)
        self.scores = torch.zeros(pages, heads, page, device=DEV)
        self.free = list(range(pages))[::-1]
        self.pages = [[] for _ in range(sessions)]
        self.length = [0] * sessions
        self.most = -(-(2 * budget + 512) // page)

    def _table(self, rows):
        host = np.full((len(rows), self.most), -1, np.int32)
        for i, r in enumerate(rows):
            host[i, :len(r)] = r
        return torch.from_numpy(host).to(DEV)

    def grow(self, counts):
        """Room for counts[i] more tokens of session i; the call's tables, lengths and starts."""
        for s, n in enumerate(counts):
            self.length[s] += n
            while len(self.pages[s]) * self.page < self.length[s]:
                self.pages[s].append(self.free.pop())
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        return (self._table(self.pages), torch.tensor(self.length, dtype=torch.int32, device=DEV),
                torch.from_numpy(starts).to(DEV))

    def attend(self, q, k, v, counts):
        """The new tokens' keys and values in, their attention out, the keys' scores up to date."""
        where, bounds = self.grow(counts), dict(max_q=max(counts))
        tm.kv_append(k, v, self.k, self.v, *where, scores=self.scores, **bounds)
        bounds.update(max_kv=max(self.length), window=self.window, sinks=self.sinks)
        out, lse = tm.paged_attention(q, self.k, self.v, *where, **bounds)
        tm.kv_add_scores(q, lse, self.k, self.scores, *where, **bounds)
        return out

    def cut(self):
        """Sessions past twice the budget go back to it, on pages of their own."""
        long = [s for s, n in enumerate(self.length) if n > 2 * self.budget]
        if not long:
            return 0
        new = [[self.free.pop() for _ in range(-(-self.budget // self.page))] for _ in long]
        lengths = torch.tensor([self.length[s] for s in long], dtype=torch.int32, device=DEV)
        tm.kv_evict(self.k, self.v, self.scores, self._table([self.pages[s] for s in long]), lengths, self._table(new),
                    budget=self.budget, max_kv=max(self.length), sinks=self.sinks, recent=self.budget // 4)
        for s, pages in zip(long, new):
            self.free += self.pages[s]   # (the next use of these pages is on the same stream)
            self.pages[s], self.length[s] = pages, self.budget
        return len(long)


class Model:
    """An embedding, attention layers and an output matrix, all random."""

    def __init__(self, sessions, budget, vocab=4000, layers=2, heads=4, group=2, dim=64, seed=0):
        g = torch.Generator(DEV).manual_seed(seed)
        self.heads, self.group, self.dim = heads, group, dim
        hidden = heads * group * dim

        def matrix(a, b):
            return (torch.randn(a, b, generator=g, device=DEV) / a ** 0.5).to(torch.bfloat16)

        self.embed = torch.randn(vocab, hidden, generator=g, device=DEV).to(torch.bfloat16)
        self.head = matrix(hidden, vocab)
        self.qkv = [matrix(hidden, (group + 2) * heads * dim) for _ in range(layers)]
        self.proj = [matrix(hidden, hidden) for _ in range(layers)]
        pages = sessions * (-(-(2 * budget + 512) // 16) + -(-budget // 16))
        self.caches = [Cache(sessions, pages, heads, dim, 16, budget, window=budget, sinks=4) for _ in range(layers)]

    def __call__(self, tokens, counts):
        """Logits of each session's last new token."""
        x = self.embed[tokens]
        H, G, D = self.heads, self.group, self.dim
        for w, proj, cache in zip(self.qkv, self.proj, self.caches):
            y = (x / x.float().square().mean(-1, keepdim=True).sqrt().to(x.dtype)) @ w
            q, k, v = y.view(-1, (G + 2) * H, D).split([G * H, H, H], 1)
            x = x + cache.attend(q, k, v, counts).reshape(x.shape) @ proj
        last = torch.tensor(np.cumsum(counts) - 1, device=DEV)
        return x[last] @ self.head


def run(sessions=8, tokens=200, budget=128, chunk=96, seed=0):
    """Decodes; returns the sampled ids [sessions, tokens], the cuts made and the cache lengths."""
    rng = np.random.default_rng(seed)
    model, vocab = Model(sessions, budget, seed=seed), 4000
    prompts = [rng.integers(0, vocab, n) for n in rng.integers(1, 2 * budget, sessions)]
    params = tm.make_params(sessions, tm.Opts(0.8, 40, 0.95), repeat_penalty=1.1, repeat_last_n=64, frequency_penalty=0.1,
                            seed=np.arange(sessions))
    records = torch.from_numpy(params.view(np.uint8)).to(DEV)
    plain = params.copy()   # the penalties are applied before
    plain["repeat_penalty"], plain["frequency_penalty"] = 1.0, 0.0
    sampler = tm.Sampler(sessions, vocab)
    history = torch.zeros(sessions, 2 * budget + tokens, dtype=torch.int32, device=DEV)
    n_history = torch.zeros(sessions, dtype=torch.int32, device=DEV)
    logits = torch.zeros(sessions, vocab, device=DEV)
    for at in range(0, max(len(p) for p in prompts), chunk):   # a chunk of every prompt that has one left
        part = [p[at:at + chunk] for p in prompts]
        y = model(torch.from_numpy(np.concatenate(part)).to(DEV), [len(p) for p in part]).float()
        has = torch.tensor([len(p) > 0 for p in part], device=DEV)
        logits = torch.where(has[:, None], y, logits)
    for s, p in enumerate(prompts):
        history[s, :len(p)] = torch.from_numpy(p)
        n_history[s] = len(p)
    ids, cuts = [], 0
    row = torch.arange(sessions, device=DEV)
    for step in range(tokens):
        tm.adjust_logits(logits, records, recent=history, n_recent=n_history, out=logits)
        plain["offset"] = step
        token = sampler.sample(logits, plain, topk_cap=40)["tokens"]
        history[row, n_history.long()] = token
        n_history += 1
        ids.append(token.clone())
        cuts += sum(c.cut() for c in model.caches)
        logits = model(token.long(), [1] * sessions).float()
    torch.cuda.synchronize()
    sampler.close()
    return torch.stack(ids, 1), cuts, [c.length for c in model.caches]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--budget", type=int, default=128)
    a = ap.parse_args()
    ids, cuts, lengths = run(a.sessions, a.tokens, a.budget)
    print(f"{ids.numel()} tokens, {cuts} caches cut; lengths now {lengths[0]}; first session: {ids[0, :16].tolist()}")
