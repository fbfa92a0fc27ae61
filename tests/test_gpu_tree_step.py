"""The tree calls as one step after another: on given streams, captured and replayed, two at once,
past 32-bit offsets, and the example."""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF
from test_gpu_tree_attention import TreeBatch, some_tree
from test_gpu_verify_tree import Trees

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Step:
    """A step's tensors; the last nodes' keys are appended by the step itself."""

    def __init__(self, kv, q, *, seed=0, V=3000, drawn=True, G=2, D=64, dt=BF):
        self.bt = TreeBatch(kv, q, H=2, G=G, D=D, dt=dt, seed=seed)
        self.trees = Trees(q, V, drawn=drawn, seed=seed)
        g = torch.Generator(DEV).manual_seed(seed)
        T = sum(q)
        self.x = torch.randn(T, 2 * G + 4, D, generator=g, device=DEV).to(dt)
        depth = [len(line) - 1 for b in range(len(kv)) for line in self.bt.lines(b)]
        p0 = np.repeat([a - b for a, b in zip(kv, q)], q)
        self.positions = torch.tensor(p0 + depth, dtype=torch.int32, device=DEV)
        self.freqs = tm.rotary_frequencies(D, device=DEV)
        (self.target, self.tokens, _, _, self.u), self.more = self.trees.device()
        self.G = G
        self.pools = [self.bt.k, self.bt.v, self.bt.scores]
        for t in self.pools:
            t.nan_to_num_(0.0)

    def run(self, stream=None):
        b = self.bt
        q, k, v = self.x.split([2 * self.G, 2, 2], 1)
        where = (b.tables, b.kv_len, b.q_start)
        q = tm.kv_append_rotary(q, k, v, b.k, b.v, *where, self.positions, self.freqs, max_q=b.max_q, scores=b.scores, stream=stream)
        out, lse = tm.tree_attention(q, b.k, b.v, *where, b.parents, max_q=b.max_q, max_kv=b.max_kv, stream=stream)
        path, kept, token = tm.verify_tree(self.target, self.tokens, b.parents, b.q_start, self.u, stream=stream, **self.more)
        new_len = tm.kv_compact(b.k, b.v, b.tables, b.kv_len, path, kept, q_start=b.q_start, scores=b.scores, stream=stream)
        back = tm.rotary(q, -self.positions, self.freqs, stream=stream)
        return [q, out, lse, path, kept, token, new_len, back]

    def state(self):
        return [t.clone() for t in self.pools]

    def reset(self, state):
        for t, s in zip(self.pools, state):
            t.copy_(s)


def bits(tensors):
    return [t.contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()]).clone() for t in tensors]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


CASES = [([700, 90], [8, 20], {}), ([1500, 300, 40], [40, 64, 9], {}), ([60] * 9, [7] * 9, dict(drawn=False)),
         ([400, 333], [33, 12], dict(V=20000, dt=HF, D=128, G=4))]


@pytest.mark.parametrize("kv, q, kw", CASES)
def test_a_step_on_a_given_stream(kv, q, kw):
    results = []
    for given in (False, True):
        s = Step(kv, q, seed=3, **kw)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        got = s.run(side.cuda_stream if given else None)   # (the tensors are held past the end)
        side.synchronize()
        torch.cuda.synchronize()
        results.append(bits(got) + bits(s.pools))
    assert same(*results)


@pytest.mark.parametrize("kv, q, kw", CASES)
def test_a_step_captured_and_replayed(kv, q, kw):
    """One capture; replays with other inputs and lengths between the program's own eager work, each
    checked against the eager calls."""
    s = Step(kv, q, seed=4, **kw)
    start = s.state()
    s.run()
    s.reset(start)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = s.run()
    for replay in range(4):
        g = torch.Generator(DEV).manual_seed(replay)
        s.x.copy_(torch.randn(s.x.shape, generator=g, device=DEV))
        s.u.copy_(torch.rand(s.u.shape, generator=g, device=DEV, dtype=torch.float64))
        if replay > 1:   # shorter sequences: their trees lie before
            s.bt.kv_len -= 3
        s.reset(start)
        graph.replay()
        got = bits(outs) + bits(s.pools)
        s.reset(start)
        want = bits(s.run())
        assert same(got, want + bits(s.pools)), replay
        torch.randn(1000, 1000, device=DEV).sum().item()


def test_two_captures_share_nothing():
    """Two graphs with workspaces of their own, replayed in turn and on two streams."""
    steps = [Step([900, 200], [40, 30], seed=s, V=30000) for s in (5, 6)]
    starts, graphs, outs, want = [], [], [], []
    for s in steps:
        starts.append(s.state())
        want.append(bits(s.run()))
        s.reset(starts[-1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for s, st in zip(steps, starts):
            s.reset(st)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert same(bits(o), w)


def test_many_verifies_at_once():
    """Calls on several streams at once, whose parts wait for each other beside the others' workgroups."""
    jobs = [Trees([9] * 24, 60000, drawn=drawn, seed=s, sharp=3.0) for s, drawn in enumerate((True, False, True, True))]
    want = [t.want() for t in jobs]
    args = [t.device() for t in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for (a, more), stream in zip(args, streams):
            with torch.cuda.stream(stream):
                for _ in range(4):
                    out = tm.verify_tree(*a, **more)
                got.append(out)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(np.array_equal(x.cpu().numpy(), y) for x, y in zip(g, w))


def test_the_same_bits_on_every_call():
    s = Step([5000, 700, 90], [50, 20, 64], seed=7, V=40000)
    start, first = s.state(), None
    for _ in range(4):
        s.reset(start)
        got = bits(s.run()) + bits(s.pools)
        first = first or got
        assert same(got, first)


def test_offsets_past_32_bits():
    """Pages whose bytes lie past 2^32 in both pools, rows of probabilities past 2^32, against the same on
    small tensors, bit for bit."""
    kv, q, H, D, page = [200, 130], [20, 33], 4, 128, 64
    small = TreeBatch(kv, q, H=H, G=2, D=D, page=page, seed=8, extra=9)
    small.k.nan_to_num_(0.0)
    small.v.nan_to_num_(0.0)
    pages = (9 << 30) // (2 * H * D * page)
    big_k, big_v = (torch.empty(pages, H, page, D, dtype=BF, device=DEV) for _ in range(2))
    far = pages - small.k.shape[0]
    big_k[far:], big_v[far:] = small.k, small.v
    tables = torch.where(small.tables >= 0, small.tables + far, small.tables)
    assert far * H * page * D * 2 > 2 ** 32
    freqs, g = tm.rotary_frequencies(D, device=DEV), torch.Generator(DEV).manual_seed(1)
    x = torch.randn(sum(q), 2 * H + 2 * H, D, generator=g, device=DEV).to(BF)
    qq, kn, vn = x.split([2 * H, H, H], 1)
    kept = torch.tensor([[0, 3, 9, 15], [0, 2, 30, 31]], dtype=torch.int32, device=DEV)
    n_kept = torch.tensor([4, 3], dtype=torch.int32, device=DEV)
    for k, v, t in ((small.k, small.v, small.tables), (big_k, big_v, tables)):
        where = (t, small.kv_len, small.q_start)
        turned = tm.kv_append_rotary(qq, kn, vn, k, v, *where, None, freqs, max_q=33)
        out = tm.tree_attention(turned, k, v, *where, small.parents, max_q=33, max_kv=200)
        tm.kv_compact(k, v, t, small.kv_len, kept, n_kept, q_start=small.q_start)
        long = torch.arange(100, 180, dtype=torch.int32, device=DEV).expand(2, 80).contiguous()
        tm.kv_compact(k, v, t, small.kv_len, long, torch.tensor([80, 20], dtype=torch.int32, device=DEV))
        if k is small.k:
            want = bits([turned, *out, k, v])
    assert same(bits([turned, *out, big_k[far:], big_v[far:]]), want)
    del big_k, big_v
    t = Trees([5, 7], 500000, drawn=True, seed=9, sharp=4.0)
    (target, tokens, parents, starts, u), more = t.device()
    rows, at = 2300, 2300 - 12
    assert at * 500000 * 4 > 2 ** 32
    wide = [torch.empty(rows, 500000, device=DEV) for _ in range(2)]
    wide[0][at:], wide[1][at:] = target, more["draft"]
    pad = lambda x: torch.cat([torch.zeros(at, dtype=x.dtype, device=DEV), x])
    starts = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), starts + at])
    got = tm.verify_tree(wide[0], pad(tokens), pad(parents), starts, pad(u), max_q=7, draft=wide[1])
    for g_, w in zip(got, t.want()):
        assert np.array_equal(g_[1:].cpu().numpy(), w)


def test_a_greedy_example_follows_the_model():
    """With probabilities of one for the best token, every token of the example is the model's best after the
    tokens before it, but for ties within the attention's rounding: a whole pass over prompt and tokens, without
    trees, gives it a probability near the row's largest.  bf16 activations are off by some 2^-8 of themselves a layer;
    logits of a few units by 0.1 at most, which is allowed for."""
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import tree_decode

    out, prompts, model, rate = tree_decode.run(sessions=4, steps=20, greedy=True, seed=1)
    assert rate > 0
    for tokens, prompt in zip(out, prompts):
        ids = np.concatenate([prompt, tokens[:-1]])
        cache = tree_decode.Cache(1, len(model.qkv), -(-len(ids) // 16), model.heads, model.dim, 16)
        where = cache.grow([len(ids)])
        p = model(torch.from_numpy(ids).to(DEV), torch.arange(len(ids), dtype=torch.int32, device=DEV), where, cache, [len(ids)])
        p = p[len(prompt) - 1:].log()
        mine = p[torch.arange(len(tokens), device=DEV), torch.tensor(tokens, device=DEV)]
        assert (mine >= p.amax(-1) - 0.2).all(), (p.amax(-1) - mine).max()   # (log-probabilities are twice the logits)


@pytest.mark.parametrize("drawn", [False, True])
def test_the_example_runs(drawn):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import tree_decode

    out, _, model, rate = tree_decode.run(sessions=3, steps=8, drawn=drawn)
    assert all(len(o) >= 9 and all(0 <= t < model.vocab for t in o) for o in out)
