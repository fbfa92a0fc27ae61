"""Speculative decoding with trees of drafts over a paged cache: a small random-weight
attention model with rotary positions, and a draft that looks at the last token alone.

    python examples/tree_decode.py [--sessions 8] [--steps 60] [--drawn]

Every step drafts a tree for each session from its last token, runs the model over all
nodes at once (kv_append_rotary, tree_attention), keeps the drafts that the target's
probabilities accept and draws one token more (verify_tree), and leaves the accepted path in
the cache (kv_compact).  With --drawn the drafts are drawn from the draft's distribution,
else they are its best.  Prompts go through paged_attention.
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
TREE = [-1, 0, 0, 0, 1, 1, 2, 4, 4, 6, 7]   # the parents of a step's nodes


class Cache:
    """The pools of all layers, and the pages and lengths of all sessions."""

    def __init__(self, sessions, layers, pages, heads, dim, page):
        shape = (pages, heads, page, dim)
        self.page, self.free = page, list(range(pages))[::-1]
        self.k = [torch.zeros(shape, dtype=torch.bfloat16, device=DEV) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.bfloat16, device=DEV) for _ in range(layers)]
        self.pages, self.length = [[] for _ in range(sessions)], [0] * sessions
        self.most = pages // sessions

    def grow(self, counts):
        """Room for counts[s] more tokens of session s; the calls' tables, lengths and starts."""
        host = np.full((len(counts), self.most), -1, np.int32)
        for s, n in enumerate(counts):
            self.length[s] += n
            while len(self.pages[s]) * self.page < self.length[s]:
                self.pages[s].append(self.free.pop())
            host[s, :len(self.pages[s])] = self.pages[s]
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEV)
        return torch.from_numpy(host).to(DEV), torch.tensor(self.length, dtype=torch.int32, device=DEV), starts

    def keep(self, where, path, kept):
        """The paths to the front of the trees, in every layer; the lengths follow."""
        tables, kv_len, starts = where
        for k, v in zip(self.k, self.v):
            new = tm.kv_compact(k, v, tables, kv_len, path, kept, q_start=starts)
        self.length = new.tolist()
        for s, n in enumerate(self.length):   # pages that hold nothing now
            while (len(self.pages[s]) - 1) * self.page >= n:
                self.free.append(self.pages[s].pop())


class Model:
    """An embedding, attention layers with rotary positions and an output matrix, all random."""

    def __init__(self, vocab=2000, layers=2, heads=4, group=2, dim=64, seed=0):
        g = torch.Generator(DEV).manual_seed(seed)
        self.vocab, self.heads, self.group, self.dim = vocab, heads, group, dim
        hidden = heads * group * dim

        def matrix(a, b):
            return (torch.randn(a, b, generator=g, device=DEV) / a ** 0.5).to(torch.bfloat16)

        self.embed = torch.randn(vocab, hidden, generator=g, device=DEV).to(torch.bfloat16)
        self.head = matrix(hidden, vocab)
        self.qkv = [matrix(hidden, (group + 2) * heads * dim) for _ in range(layers)]
        self.proj = [matrix(hidden, hidden) for _ in range(layers)]
        self.freqs = tm.rotary_frequencies(dim, device=DEV)

    def __call__(self, tokens, positions, where, cache, counts, parents=None):
        """The probabilities of what follows each token."""
        x, H, G = self.embed[tokens], self.heads, self.group
        bounds = dict(max_q=max(counts), max_kv=max(cache.length))
        for w, proj, k_cache, v_cache in zip(self.qkv, self.proj, cache.k, cache.v):
            y = (x / x.float().square().mean(-1, keepdim=True).sqrt().to(x.dtype)) @ w
            q, k, v = y.view(-1, (G + 2) * H, self.dim).split([G * H, H, H], 1)
            q = tm.kv_append_rotary(q, k, v, k_cache, v_cache, *where, positions, self.freqs, max_q=max(counts))
            if parents is None:
                out, _ = tm.paged_attention(q, k_cache, v_cache, *where, **bounds)
            else:
                out, _ = tm.tree_attention(q, k_cache, v_cache, *where, parents, **bounds)
            x = x + 0.5 * (out.reshape(x.shape) @ proj)
        return torch.softmax((x @ self.head).float() * 2.0, -1)

    def draft(self, tokens):
        """What follows a token by the token alone."""
        return torch.softmax((self.embed[tokens] @ self.head).float() * 2.0, -1)


def drafts(model, roots, drawn, g):
    """A tree for each session: tokens [sessions, nodes] and the draft's rows."""
    S, n = roots.shape[0], len(TREE)
    tokens = torch.zeros(S, n, dtype=torch.long, device=DEV)
    rows = torch.zeros(S, n, model.vocab, device=DEV)
    tokens[:, 0] = roots
    for i in range(n):
        if i:
            p = TREE[i]
            if drawn:
                tokens[:, i] = torch.multinomial(rows[:, p], 1, generator=g)[:, 0]
            else:
                tokens[:, i] = torch.topk(rows[:, p], 8, -1).indices[:, TREE[:i].count(p)]
        rows[:, i] = model.draft(tokens[:, i])
    return tokens, rows


def run(sessions=8, steps=60, drawn=False, greedy=False, seed=0):
    """Decodes; returns each session's tokens, the prompts, the model and the drafts accepted a step."""
    rng, g = np.random.default_rng(seed), torch.Generator(DEV).manual_seed(seed)
    model = Model(seed=seed)
    n, depth = len(TREE), []
    for p in TREE:
        depth.append(0 if p < 0 else depth[p] + 1)
    prompts = [rng.integers(0, model.vocab, k) for k in rng.integers(1, 200, sessions)]
    most = 200 + steps * (max(depth) + 1) + n
    cache = Cache(sessions, len(model.qkv), sessions * -(-most // 16), model.heads, model.dim, 16)
    counts = [len(p) for p in prompts]
    where = cache.grow(counts)
    positions = torch.tensor(np.concatenate([np.arange(k) for k in counts]), dtype=torch.int32, device=DEV)
    p = model(torch.from_numpy(np.concatenate(prompts)).to(DEV), positions, where, cache, counts)
    last = p[(where[2][1:] - 1).long()]
    roots = last.argmax(-1) if greedy else torch.multinomial(last, 1, generator=g)[:, 0]
    out, accepted = [[r] for r in roots.tolist()], 0
    parents = torch.tensor(TREE * sessions, dtype=torch.int32, device=DEV)
    for _ in range(steps):
        draft, rows = drafts(model, roots, drawn, g)
        first = torch.tensor(cache.length, dtype=torch.int32, device=DEV)
        positions = (first[:, None] + torch.tensor(depth, dtype=torch.int32, device=DEV)).flatten()
        where = cache.grow([n] * sessions)
        target = model(draft.flatten(), positions, where, cache, [n] * sessions, parents)
        if greedy:
            target = torch.nn.functional.one_hot(target.argmax(-1), model.vocab).float()
        u = torch.rand(sessions * n, generator=g, device=DEV, dtype=torch.float64)
        path, kept, token = tm.verify_tree(target, draft.flatten().int(), parents, where[2], u, max_q=n,
                                           draft=rows.flatten(0, 1) if drawn else None)
        cache.keep(where, path, kept)
        chosen = torch.gather(draft, 1, path.clamp(min=0).long()).tolist()
        for s, (k, t) in enumerate(zip(kept.tolist(), token.tolist())):
            out[s] += chosen[s][1:k] + [t]
            accepted += k - 1
        roots = token.long()
    return out, prompts, model, accepted / (steps * sessions)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=8)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--drawn", action="store_true")
    a = ap.parse_args()
    out, _, _, rate = run(a.sessions, a.steps, a.drawn)
    print(f"{sum(map(len, out))} tokens in {a.steps} steps, {rate:.2f} drafts accepted a step; first session: {out[0][:16]}")
