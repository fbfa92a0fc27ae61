"""The verify of drafted trees against the walk in 64 bits, written out one sequence at a time.
All outputs are whole numbers and have to be equal: sums of another order differ by 10^-16 of
themselves, and the given random numbers do not come that near to a border."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import DEV
from test_gpu_tree_attention import some_tree

pytestmark = pytest.mark.gpu

F32, HF, BF = torch.float32, torch.float16, torch.bfloat16


def clean(row):
    row = row.astype(np.float64)
    return np.where(np.isfinite(row) & (row > 0), row, 0.0)


def walk(target, draft, tokens, parents, u, max_q):
    """Path, token of one tree (numpy arrays of its nodes)."""
    n = min(len(tokens), max_q)
    if n == 0:
        return [], -1
    V, c, line = target.shape[1], 0, [0]
    while True:
        p = clean(target[c])
        q = None if draft is None else clean(draft[c])
        r, S, j = p.copy(), 1.0, None
        for i in range(c + 1, n):
            if parents[i] != c:
                continue
            x = tokens[i]
            there = 0 <= x < V
            rx, qx = (r[x] if there else 0.0), (1.0 if q is None else q[x] if there else 0.0)
            if u[i] * qx * S < rx:
                j = i
                break
            if q is None:
                S -= rx
                if there:
                    r[x] = 0.0
            else:
                r = np.maximum(r - S * q, 0.0)
                S = math.fsum(r)
        if j is None:
            break
        c = j
        line.append(j)
    if not r.any():
        r = p
    if not r.any():
        return line, -1
    upto = np.cumsum(r)
    over = np.flatnonzero((upto > max(u[0] * upto[-1], 0.0)) & (r > 0))
    return line, int(over[0]) if len(over) else int(np.flatnonzero(r)[-1])


class Trees:
    def __init__(self, q, V, *, drawn, dt=F32, seed=0, noise=0.7, sharp=2.0, kind="random", max_q=None):
        rng = np.random.default_rng(seed)
        T = sum(q)
        self.q, self.V, self.max_q = q, V, max(q + [0]) if max_q is None else max_q
        self.parents = np.array([p for n in q for p in some_tree(rng, n, kind)], np.int32)
        x = rng.normal(0, sharp, (T, V))
        y = x + rng.normal(0, noise, (T, V))
        self.target = torch.from_numpy(np.exp(x) / np.exp(x).sum(1, keepdims=True)).to(dt)
        self.draft = torch.from_numpy(np.exp(y) / np.exp(y).sum(1, keepdims=True)).to(dt) if drawn else None
        self.starts = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        self.tokens, self.u = np.zeros(T, np.int32), rng.random(T)
        for a, n in zip(self.starts[:-1], q):
            for i in range(1, n):
                c = self.parents[a + i]
                if drawn:
                    d = self.draft[a + c].double().numpy()
                    self.tokens[a + i] = rng.choice(V, p=d / d.sum())
                else:
                    rank = int((self.parents[a:a + i] == c).sum())
                    self.tokens[a + i] = np.argsort(-y[a + c])[min(rank, V - 1)]

    def device(self, pad=0, offset=0):
        """The tensors; rows `pad` elements longer, `offset` from an aligned address."""
        def rows(t):
            if t is None:
                return None
            w = torch.full((t.shape[0], t.shape[1] + pad + offset), float("nan"), dtype=t.dtype, device=DEV)
            w[:, offset:offset + t.shape[1]] = t.to(DEV)
            return w[:, offset:offset + t.shape[1]]

        ints = [torch.from_numpy(x).to(DEV) for x in (self.tokens, self.parents, self.starts, self.u)]
        return (rows(self.target), *ints), dict(max_q=self.max_q, draft=rows(self.draft))

    def want(self):
        target = self.target.double().numpy()
        draft = None if self.draft is None else self.draft.double().numpy()
        path = np.full((len(self.q), self.max_q), -1, np.int32)
        kept, token = np.zeros(len(self.q), np.int32), np.zeros(len(self.q), np.int32)
        for b, (a, n) in enumerate(zip(self.starts[:-1], self.q)):
            s = np.s_[a:a + n]
            line, token[b] = walk(target[s], None if draft is None else draft[s], self.tokens[s], self.parents[s], self.u[s], self.max_q)
            path[b, :len(line)], kept[b] = line, len(line)
        return path, kept, token

    def check(self, got=None, **kw):
        if got is None:
            args, more = self.device(**kw)
            got = tm.verify_tree(*args, **more)
        want = self.want()
        for g, w, name in zip(got, want, ("path", "kept", "token")):
            assert np.array_equal(g.cpu().numpy(), w), (name, g.cpu().numpy(), w)
        return want


@pytest.mark.parametrize("dt", [F32, HF, BF])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("q, V", [([1], 1), ([2], 2), ([5, 1, 9], 50), ([8] * 20, 300), ([25, 3], 2048), ([7, 12], 5001), ([16] * 6, 33000)])
def test_walks(dt, drawn, q, V):
    kept = [Trees(q, V, drawn=drawn, dt=dt, seed=s).check()[1] for s in range(3)]
    if len(q) > 5:   # drafts are accepted and refused
        assert (np.concatenate(kept) > 1).any() and (np.concatenate(kept) < 4).any()


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
def test_kinds_of_trees(drawn, kind):
    for seed in range(3):
        Trees([6, 20, 2], 700, drawn=drawn, seed=seed, kind=kind, sharp=1.0).check()


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("V", [257, 4099, 20001])
def test_rows_of_any_stride_and_alignment(drawn, dt, V):
    t = Trees([6, 9], V, drawn=drawn, dt=dt, seed=V)
    for pad, offset in ((0, 0), (1, 0), (3, 1), (8, 5)):
        t.check(pad=pad, offset=offset)


@pytest.mark.parametrize("dt", [F32, HF, BF])
@pytest.mark.parametrize("V", [8193, 16385, 32767, 32768, 32769, 70003])
def test_given_drafts_around_whole_parts(dt, V):
    """A workgroup a sequence (in 16 bits up to 32768 ids), and several."""
    t = Trees([6, 1, 9], V, drawn=False, dt=dt, seed=V, sharp=3.0)
    for pad, offset in ((0, 0), (3, 1), (8, 5)):
        t.check(pad=pad, offset=offset)


@pytest.mark.parametrize("drawn", [False, True])
def test_large_vocabularies(drawn):
    for V, q in ((128256, [9, 4]), (256000, [5]), (1048576, [3])):
        Trees(q, V, drawn=drawn, seed=1, sharp=4.0).check()
    Trees([4] * 3, 151936, drawn=drawn, dt=BF, seed=2, sharp=4.0).check()


@pytest.mark.parametrize("drawn", [False, True])
def test_the_largest_trees(drawn):
    for kind in ("random", "star", "chain"):
        Trees([512, 30], 600, drawn=drawn, seed=4, kind=kind, sharp=0.3, noise=2.0).check()
    Trees([100], 9000, drawn=drawn, seed=4, kind="star", sharp=0.3, noise=2.0).check()


@pytest.mark.parametrize("drawn", [False, True])
def test_many_sequences(drawn):
    rng = np.random.default_rng(8)
    Trees([int(n) for n in rng.integers(0, 7, 700)], 97, drawn=drawn, seed=9).check()
    Trees([3] * 300, 4500, drawn=drawn, seed=9).check()


@pytest.mark.parametrize("drawn", [False, True])
def test_empty_sequences_and_max_q(drawn):
    t = Trees([0, 6, 0, 9, 0], 120, drawn=drawn, seed=3)
    want = t.check()
    assert want[1][0] == 0 and want[2][0] == -1
    t.max_q = 4   # nodes past it are left out
    t.check()
    t.max_q = 1
    assert (t.check()[1] <= 1).all()
    args, more = t.device()
    path, kept, token = tm.verify_tree(*args, **dict(more, max_q=0))
    assert path.shape == (5, 0) and (kept == 0).all() and (token == -1).all()
    none = tm.verify_tree(args[0][:0], args[1][:0], args[2][:0], torch.zeros(4, dtype=torch.int32, device=DEV), args[4][:0], max_q=3)
    assert (none[0] == -1).all() and (none[1] == 0).all() and (none[2] == -1).all()
    assert tm.verify_tree(args[0], args[1], args[2], args[3][:1], args[4], max_q=3)[0].shape == (0, 3)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [60, 9000])
def test_drafts_outside_the_vocabulary_and_twice(drawn, V):
    t = Trees([9, 9, 9], V, drawn=drawn, seed=5, kind="star", sharp=0.5)
    t.tokens[[2, 11, 20]] = [V, -1, 2 ** 31 - 1]
    t.tokens[[4, 5, 13, 14]] = t.tokens[[3, 3, 12, 12]]   # the same token several times
    t.tokens[22:27] = t.tokens[21]
    for u in (0.0, 0.3, 1 - 2.0 ** -53):
        t.u[:] = u
        t.check()


@pytest.mark.parametrize("drawn", [False, True])
def test_parents_that_are_none(drawn):
    """A node whose parent is not below it, and what hangs from it, is never tried."""
    t = Trees([8], 40, drawn=drawn, seed=6)
    t.parents[:] = [5, 1, 0, 2, -9, 7, 5, 2 ** 31 - 1]
    t.u[1:] = 0.0
    assert set(t.check()[0][0][:3]) <= {0, 2, 3, -1}


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [33, 7000])
def test_what_is_no_probability(drawn, V):
    t = Trees([5, 5, 5, 5], V, drawn=drawn, seed=7)
    x = t.target
    x[0, ::3], x[1, 1::2], x[2, :] = float("nan"), -1.0, 0.0
    x[5, 4], x[6, :] = float("inf"), float("nan")
    x[10, :], x[15] = 0.0, 0.0
    x[10, V - 1] = 0.5     # a single entry, the last
    if drawn:
        t.draft[0, ::2], t.draft[5, 3] = float("nan"), float("inf")
    want = t.check()
    assert want[2][3] == -1 and want[2][2] == V - 1 or want[1][2] > 1


def test_drafts_of_the_target_itself_are_all_accepted():
    """p = q: every first child is accepted for any number below 1, and a last refusal of nothing leaves the row."""
    t = Trees([6, 6], 500, drawn=True, seed=8, kind="chain")
    t.draft = t.target.clone()
    t.u[:] = 1 - 2.0 ** -53
    assert (t.check()[1] == 6).all()
    t.u[1] = t.u[7] = 2.0   # no number below 1: refused, and nothing is left of the target
    assert (t.check()[1] == 1).all()


def test_the_target_with_all_its_mass_refused():
    t = Trees([4], 10, drawn=False, seed=9, kind="star")
    t.target[0] = 0
    t.target[0, [2, 7]] = 0.5
    t.tokens[1:] = [2, 7, 2]
    t.u[:] = [0.9, 2.0, 2.0, 2.0]
    assert t.check()[2][0] == 7


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -53, 1.0, -0.5, math.inf, math.nan])
def test_numbers_at_the_ends(drawn, u):
    for V in (70, 6000):
        t = Trees([4, 1], V, drawn=drawn, seed=10, sharp=6.0)
        t.u[[0, 4]] = u
        args, more = t.device()
        got = tm.verify_tree(*args, **more)
        if math.isnan(u):
            t.u[[0, 4]] = 0.0
        t.check(got=got)


def test_tokens_follow_the_target():
    """First tokens of many trees with drafts drawn anew: their shares are the target's (chi-squared, 5
    degrees of freedom; a value above 40 has a chance of 1.5e-7)."""
    rng, V, n = np.random.default_rng(11), 6, 40000
    p, q = np.array([0.3, 0.05, 0.25, 0.2, 0.15, 0.05]), np.array([0.1, 0.4, 0.1, 0.1, 0.1, 0.2])
    for drawn in (True, False):
        ids = rng.choice(V, (n, 3), p=q) if drawn else np.tile([1, 0, 3], (n, 1))
        tokens = np.concatenate([np.zeros((n, 1), int), ids], 1).astype(np.int32).ravel()
        dev = [torch.from_numpy(x).to(DEV) for x in (tokens, np.tile([-1, 0, 0, 0], n).astype(np.int32),
                                                     (4 * np.arange(n + 1)).astype(np.int32), rng.random(4 * n))]
        target = torch.from_numpy(p).to(DEV).expand(4 * n, V).contiguous()
        draft = torch.from_numpy(q).to(DEV).expand(4 * n, V).contiguous()
        path, kept, token = tm.verify_tree(target.float(), *dev, max_q=4, draft=draft.float() if drawn else None)
        path, kept, token = path.cpu().numpy(), kept.cpu().numpy(), token.cpu().numpy()
        first = np.where(kept > 1, tokens.reshape(n, 4)[np.arange(n), path[:, 1].clip(0)], token)
        count = np.bincount(first, minlength=V)
        assert ((count - n * p) ** 2 / (n * p)).sum() < 40, count / n


@pytest.mark.parametrize("drawn", [False, True])
def test_a_wait_that_runs_out(drawn):
    """The parts of a sequence wait for each other's sums; without any wait each works the missing ones out
    itself, to the same answer."""
    lib = tm.load_library()
    lib.tms_debug_verify_polls.argtypes = [C.c_int]
    t = Trees([9, 12, 5], 40000, drawn=drawn, seed=12, sharp=3.0)
    try:
        for polls in (0, 1, 2):
            lib.tms_debug_verify_polls(polls)
            t.check()
    finally:
        lib.tms_debug_verify_polls(-1)
