"""Attention of drafted trees over the paged cache, against a plain implementation in 64 bits
with the tolerances of test_gpu_cache.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch, check

pytestmark = pytest.mark.gpu


def some_tree(rng, n, kind="random"):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    if kind == "roots":
        return [-1] * n
    return ([-1] + [int(rng.integers(max(0, i - 9), i)) for i in range(1, n)])[:n]


class TreeBatch(Batch):
    def __init__(self, kv, q, *, kind="random", seed=0, parents=None, **kw):
        super().__init__(kv, q, seed=seed, **kw)
        rng = np.random.default_rng(seed + 1000)
        self.trees = parents or [some_tree(rng, n, kind) for n in q]
        flat = np.array([p for t in self.trees for p in t], np.int32)
        self.parents = torch.from_numpy(flat).to(DEV)

    def lines(self, b):
        """Each node's ancestors and itself, from itself up."""
        out = []
        for i in range(self.q[b]):
            line, a = [], i
            while a >= 0:
                line.append(a)
                p = self.trees[b][a]
                a = p if 0 <= p < a else -1
            out.append(line)
        return out

    def seen(self, b, window, sinks):
        n, L = self.q[b], self.kv[b]
        p0 = L - n
        ok = np.zeros((n, L), bool)
        for i, line in enumerate(self.lines(b)):
            at = p0 + len(line) - 1   # where the node stands in the text
            if i >= self.max_q:
                continue
            for j in range(max(p0, 0)):
                ok[i, j] = not window or j > at - window or j < sinks
            for back, a in enumerate(line):
                if p0 + a >= 0:
                    ok[i, p0 + a] = not window or back < window or at - back < sinks
        page = self.host[b][np.arange(L) // self.page] if L else np.zeros(0, np.int32)
        return ok & ((page >= 0) & (page < self.k.shape[0]))[None]

    def attend(self, q=None, **kw):
        return tm.tree_attention(self.qs.to(DEV) if q is None else q, self.k, self.v, self.tables, self.kv_len, self.q_start, self.parents,
                                 max_q=self.max_q, max_kv=self.max_kv, **kw)


@pytest.mark.parametrize("dt", [HF, BF])
@pytest.mark.parametrize("kv, q, H, G, D", [([1], [1], 1, 1, 64), ([8], [8], 2, 2, 64), ([40, 17, 300], [8, 17, 1], 2, 4, 128),
                                            ([600, 90], [25, 40], 1, 3, 80), ([70], [33], 1, 1, 96), ([200, 64, 31], [64, 60, 31], 1, 8, 64),
                                            ([1200], [70], 2, 2, 256), ([2500, 41], [6, 3], 1, 5, 128)])
def test_trees(dt, kv, q, H, G, D):
    check(TreeBatch(kv, q, H=H, G=G, D=D, dt=dt, seed=len(kv) + D))


@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
@pytest.mark.parametrize("q", [[5, 9], [40, 64], [100, 3]])
def test_kinds(kind, q):
    bt = TreeBatch([150, 131], q, H=1, G=2, D=64, kind=kind, seed=3)
    check(bt)
    if kind == "chain":   # what paged_attention sees too, within the same bounds
        check(bt, got=Batch.attend(bt))


@pytest.mark.parametrize("window, sinks", [(1, 0), (2, 0), (3, 5), (16, 0), (40, 4), (64, 130), (1000, 3)])
@pytest.mark.parametrize("q, G, page", [([7, 3], 2, 16), ([60, 33], 2, 8), ([40, 40], 1, 64)])
def test_windows(window, sinks, q, G, page):
    for kind in ("random", "chain"):
        check(TreeBatch([157, 64], q, H=1, G=G, D=64, page=page, kind=kind, seed=window), window=window, sinks=sinks)


@pytest.mark.parametrize("G", [1, 4])
def test_the_largest_trees(G):
    rng = np.random.default_rng(5)
    n = 512
    wide = [-1] + [int(rng.integers(0, i)) for i in range(1, n)]
    check(TreeBatch([530], [n], H=1, G=G, D=64, parents=[wide], seed=1))
    check(TreeBatch([512], [n], H=1, G=G, D=64, kind="chain", seed=1))
    check(TreeBatch([700], [n], H=1, G=G, D=64, kind="chain", seed=1), window=300, sinks=2)


@pytest.mark.parametrize("q", [[6], [45]])
def test_parents_that_are_none(q):
    """Parents at or above the node itself, or below -1, count as none."""
    n = q[0]
    parents = some_tree(np.random.default_rng(1), n)
    parents[1], parents[2], parents[3], parents[5] = 1, 5, -7, 2 ** 31 - 1
    parents[4] = -2 ** 31
    check(TreeBatch([60], q, H=2, G=2, D=64, parents=[parents], seed=2))


@pytest.mark.parametrize("q", [[4, 9], [40, 50]])
def test_unmapped_pages_and_empty_rows(q):
    bt = TreeBatch([100, 90], q, H=1, G=2, D=64, seed=4)
    bt.host[0][:] = -1          # the first sequence sees nothing at all
    bt.host[1][1] = 10 ** 6
    bt.host[1][4] = -5
    bt.tables.copy_(torch.from_numpy(bt.host))
    check(bt)
    check(bt, window=30, sinks=2)


@pytest.mark.parametrize("q", [[5, 4], [40, 36]])
def test_max_q_and_short_sequences(q):
    """Nodes past max_q are left out and rows behind the last sequence are left as they were; a
    sequence shorter than its tree has its first nodes before position 0, and they do not exist."""
    bt = TreeBatch([3, 60], q, H=1, G=2, D=64, seed=6, parents=[list(range(-1, q[0] - 1)), some_tree(np.random.default_rng(3), q[1])])
    bt.kv[0] = 3
    bt.max_q = max(q) - 2
    T = sum(q)
    out = torch.full((T + 2, 2, 64), 9.0, dtype=BF, device=DEV)
    lse = torch.full((T + 2, 2), 9.0, device=DEV)
    qs = torch.cat([bt.qs, bt.qs[:2]]).to(DEV)
    parents = torch.cat([bt.parents, bt.parents[:2]])
    tm.tree_attention(qs, bt.k, bt.v, bt.tables, bt.kv_len, bt.q_start, parents, max_q=bt.max_q, max_kv=bt.max_kv, out=out, lse=lse)
    left = [b for a, n in zip(bt.starts[:-1], q) for b in range(a + min(n, bt.max_q), a + n)] + [T, T + 1]
    assert (out[left] == 9.0).all() and (lse[left] == 9.0).all()
    done = [i for i in range(T) if i not in left]
    want, wl, tol, ltol, _, _ = bt.reference()
    o, l = out.double().cpu().numpy(), lse.double().cpu().numpy()
    empty = np.isneginf(wl[done])
    assert np.array_equal(np.isneginf(l[done]), empty) and (empty.any() == (q[0] > 3))
    assert np.all(np.abs(o[done] - want[done]) <= tol[done])
    assert np.all(np.abs(l[done][~empty] - wl[done][~empty]) <= ltol[done][~empty])


@pytest.mark.parametrize("q", [[6, 5], [40, 33]])
def test_garbage_that_no_row_sees(q):
    """Infinite and NaN values of nodes that a row does not see do not reach it."""
    bt = TreeBatch([80, 70], q, H=1, G=2, D=64, kind="star", seed=7)
    for b, n in enumerate(q):
        last = bt.kv[b] - 1
        bt.keys[b][last], bt.values[b][last] = float("nan"), float("inf")
        bt.values[b][last - 1, :, 5] = float("nan")
    bt.fill()
    out, lse = bt.attend()
    own = [x for a, n in zip(bt.starts[:-1], q) for x in (a + n - 1, a + n - 2)]
    others = [i for i in range(sum(q)) if i not in own]
    for b in range(2):
        bt.keys[b] = torch.nan_to_num(bt.keys[b], nan=0.0, posinf=0.0)
        bt.values[b] = torch.nan_to_num(bt.values[b], nan=0.0, posinf=0.0)
    want, wl, tol, ltol, _, _ = bt.reference()
    assert np.all(np.abs(out.double().cpu().numpy() - want)[others] <= tol[others])
    assert np.all(np.abs(lse.double().cpu().numpy() - wl)[others] <= ltol[others])
    assert torch.isnan(out[bt.starts[1] - 1]).all()


@pytest.mark.parametrize("q, page", [([9, 5, 30], 16), ([40, 33, 64], 128)])
def test_strides_and_in_place(q, page):
    bt = TreeBatch([300, 157, 90], q, H=2, G=3, D=80, page=page, dt=HF, seed=8, slot_major=True)
    packed = torch.zeros(sum(q), 11, 80, dtype=HF, device=DEV)
    packed[:, 2:8] = bt.qs.to(DEV)
    view = packed[:, 2:8]
    want = bt.attend()
    check(bt, got=want)
    out, lse = bt.attend(q=view, out=view)
    assert torch.equal(packed[:, 2:8], want[0]) and torch.equal(lse, want[1])
    assert (packed[:, :2] == 0).all() and (packed[:, 8:] == 0).all()
    check(bt, scale=-0.03, got=bt.attend(scale=-0.03))
    check(bt, scale=0.0, got=bt.attend(scale=0.0))


@pytest.mark.parametrize("kv, q, kw", [([9000, 300], [6, 2], {}), ([9000, 5000], [24, 30], {}), ([20000], [64], dict(window=700, sinks=4))])
def test_long_caches(kv, q, kw):
    check(TreeBatch(kv, q, H=1, G=4, D=128, page=64, seed=9), **kw)


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("kw", [{}, dict(window=900, sinks=3)])
def test_many_rows_over_long_caches(D, kw):
    check(TreeBatch([3000, 700, 1300], [64, 60, 33], H=2, G=4, D=D, page=32, seed=D), **kw)


def test_more_sequences_than_threads():
    """A long sequence among hundreds of short ones: shares that hold many of them, and none, whole."""
    rng = np.random.default_rng(14)
    q = [int(x) for x in rng.integers(0, 41, 300)]
    kv = [n + int(x) for n, x in zip(q, rng.integers(0, 90, 300))]
    q[170], kv[170] = 40, 2900
    check(TreeBatch(kv, q, H=1, G=1, D=64, seed=15))


def test_many_sequences_of_any_lengths():
    rng = np.random.default_rng(11)
    q = [int(x) for x in rng.integers(1, 9, 40)]
    kv = [n + int(x) for n, x in zip(q, rng.integers(0, 1500, 40))]
    check(TreeBatch(kv, q, H=2, G=2, D=64, seed=12))
    q[7], kv[7], q[9] = 0, 5, 0
    check(TreeBatch(kv, q, H=1, G=1, D=64, seed=13))


@pytest.mark.parametrize("q", [[6, 2, 1], [40, 60, 33]])
def test_positions_past_max_kv(q):
    """max_kv sizes workspaces and grids; positions past it are attended all the same."""
    for told in (1, 100, 2000):
        bt = TreeBatch([3000, 90, 700], q, H=1, G=2, D=64, seed=14)
        bt.max_kv = told
        check(bt)
        check(bt, window=1500, sinks=4)


@pytest.mark.parametrize("q", [[6, 5], [40, 33]])
def test_lengths_past_the_table(q):
    """Positions past the table do not exist: a tree that lies there partly or wholly."""
    bt = TreeBatch([70, 80], q, H=1, G=2, D=64, seed=15)
    cap = bt.host.shape[1] * bt.page
    for b, past in ((0, 3), (1, 200)):
        bt.kv[b] = cap + past
        bt.kv_len[b] = bt.kv[b]
        grow = bt.kv[b] - bt.keys[b].shape[0]
        for t in (bt.keys, bt.values):
            t[b] = torch.cat([t[b], torch.zeros(grow, 1, 64, dtype=BF)])
    bt.k.nan_to_num_(0.0)   # (slots of the last pages that hold positions now)
    bt.v.nan_to_num_(0.0)
    bt.host = np.concatenate([bt.host, np.full((2, 40), -1, np.int32)], 1)   # (the reference's view of what is not there)
    check(bt)
