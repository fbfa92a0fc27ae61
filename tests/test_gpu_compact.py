"""Chosen entries of the paged cache moved: bits against a plain implementation that reads all before it writes."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch

pytestmark = pytest.mark.gpu


def pools(bt):
    return [bt.k.contiguous().view(torch.int16).cpu().numpy().copy(), bt.v.contiguous().view(torch.int16).cpu().numpy().copy(),
            bt.scores.view(torch.int32).cpu().numpy().copy()]


def moved(bt, kept, n_kept, base, dst=None):
    """The pools' bits after the call, and the new lengths."""
    was, now = pools(bt), pools(bt)
    P, S = bt.k.shape[0], bt.page
    cap = bt.host.shape[1] * S
    to = bt.host if dst is None else dst
    new = []
    for b, L in enumerate(bt.kv):
        n = min(max(n_kept[b], 0), kept.shape[1])
        if dst is None:
            n = min(n, L - base[b])
        new.append(max(base[b] + n, 0))
        for i in range(n):
            j, z = base[b] + int(kept[b][i]), base[b] + i
            if kept[b][i] < 0 or (dst is None and kept[b][i] < i) or not 0 <= j < min(L, cap) or z < 0 or z // S >= to.shape[1]:
                continue
            a, c = bt.host[b][j // S], to[b][z // S]
            if 0 <= a < P and 0 <= c < P:
                for x, y in zip(now, was):
                    x[c, :, z % S] = y[a, :, j % S]
    return now, new


def check(bt, kept, n_kept, *, tree=True, dst=None, scores=True, new_len=None):
    kept = np.asarray(kept, np.int32)
    base = [L - n if tree else 0 for L, n in zip(bt.kv, bt.q)]
    want, lengths = moved(bt, kept, n_kept, base, dst)
    if not scores:
        want[2] = pools(bt)[2]
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEV)
    got = tm.kv_compact(bt.k, bt.v, bt.tables, bt.kv_len, dev(kept), dev(n_kept), q_start=bt.q_start if tree else None,
                        dst_tables=None if dst is None else dev(dst), scores=bt.scores if scores else None, new_len=new_len)
    assert got.tolist() == lengths
    for g, w in zip(pools(bt), want):
        assert np.array_equal(g, w)


def paths(rng, q, most):
    n_kept = [int(rng.integers(0, min(most, n) + 1)) for n in q]
    kept = np.full((len(q), most), -1, np.int32)
    for b, (n, k) in enumerate(zip(q, n_kept)):
        kept[b, :k] = np.sort(rng.choice(n, k, replace=False))
    return kept, n_kept


@pytest.mark.parametrize("dt", [HF, BF])
@pytest.mark.parametrize("kv, q, H, D, page", [([1], [1], 1, 8, 8), ([60, 33, 5], [9, 30, 5], 2, 64, 16), ([300], [64], 3, 80, 8),
                                               ([100, 512], [50, 512], 1, 256, 64), ([40] * 30, [17] * 30, 2, 128, 16)])
def test_paths(dt, kv, q, H, D, page):
    rng = np.random.default_rng(D)
    for most in (1, 8, 64, 200):
        bt = Batch(kv, q, H=H, G=1, D=D, page=page, dt=dt, seed=most, slot_major=most == 8)
        check(bt, *paths(rng, q, most), scores=most != 64)


@pytest.mark.parametrize("page", [8, 128])
def test_long_lists_in_place(page):
    rng = np.random.default_rng(3)
    kv = [5000, 1, 2077, 900, 64]
    for share in (1.0, 0.98, 0.5, 0.03):
        bt = Batch(kv, [1] * 5, H=2, G=1, D=64, page=page, seed=4)
        kept, n_kept = np.full((5, 5000), -1, np.int32), []
        for b, n in enumerate(kv):
            at = np.flatnonzero(rng.random(n) < share)
            kept[b, :len(at)] = at
            n_kept.append(len(at))
        check(bt, kept, n_kept, tree=False)
    # Shifted by one, by a page, and to the end of the sequence.
    for by in (1, page, 3000):
        bt = Batch([5000], [1], H=1, G=1, D=128, page=page, seed=5)
        at = np.concatenate([np.arange(4), np.arange(4 + by, 5000)])
        check(bt, at[None], [len(at)], tree=False)


def test_lists_that_are_not_ascending():
    """Any kept[i] >= i: twice the same, and in other orders."""
    bt = Batch([200], [1], H=1, G=1, D=64, seed=6)
    kept = [[5, 3, 2, 9, 9, 9, 6, 150, 8, 100]]
    check(bt, kept, [10], tree=False)
    rng = np.random.default_rng(7)
    kept = [np.array([int(rng.integers(i, 190)) for i in range(150)])]
    check(bt, kept, [150], tree=False)


@pytest.mark.parametrize("tree", [False, True])
def test_entries_that_are_left_out(tree):
    """Below their own place, outside the sequence, counts of any size, unmapped pages on either side."""
    for most in (10, 80):
        bt = Batch([90, 100, 40], [30, 90, 40], H=2, G=1, D=64, seed=8)
        bt.host[1][3], bt.host[1][1], bt.host[0][4] = -1, 10 ** 6, -7
        bt.tables.copy_(torch.from_numpy(bt.host))
        rng = np.random.default_rng(9)
        kept = rng.integers(-3, 110, (3, most)).astype(np.int32)
        kept[0, 1], kept[1, 2], kept[2, 0] = 2 ** 31 - 1, -2 ** 31, 2 ** 29
        check(bt, kept, [2 ** 31 - 1, most, -5], tree=tree)
        check(bt, kept, [0, 3, 2 ** 30], tree=tree, scores=False)


def test_sequences_shorter_than_their_trees_and_tables():
    bt = Batch([3, 60], [5, 10], H=1, G=1, D=64, seed=10)
    kept = np.tile(np.arange(1, 6, dtype=np.int32), (2, 1))
    check(bt, kept, [4, 5])
    bt.kv_len[1] = bt.kv[1] = 10 ** 6   # past the table
    check(bt, kept, [2, 5])


@pytest.mark.parametrize("dt, page, D", [(BF, 16, 128), (HF, 64, 80)])
def test_to_other_pages(dt, page, D):
    kv = [500, 33, 129]
    each = -(-500 // page) + 1
    bt = Batch(kv, [1] * 3, H=2, G=1, D=D, page=page, dt=dt, seed=11, extra=3 * each)
    used = set(bt.host[bt.host >= 0].tolist())
    dst = np.array([p for p in range(bt.k.shape[0]) if p not in used][:3 * each], np.int32).reshape(3, each)
    kept = np.tile(np.arange(500, dtype=np.int32), (3, 1))
    check(bt, kept, kv, tree=False, dst=dst)          # a copy
    kept[0, :200] = np.random.default_rng(1).integers(0, 500, 200)   # any list, entries twice
    check(bt, kept, [200, 20, 0], tree=False, dst=dst)
    dst[1, 0], dst[2, 1] = -1, 10 ** 6
    check(bt, kept, [10, 33, 129], tree=False, dst=dst, scores=False)
    check(bt, kept, [500, 500, 500], tree=False, dst=dst[:, :2].copy())   # a table that is too short


def test_to_other_pages_with_trees():
    bt = Batch([40, 50], [10, 20], H=1, G=1, D=64, seed=12, extra=20)
    used = set(bt.host[bt.host >= 0].tolist())
    dst = np.array([p for p in range(bt.k.shape[0]) if p not in used][:8], np.int32).reshape(2, 4)
    check(bt, [[0, 4, 9], [0, 1, 19]], [3, 3], dst=dst)


def test_new_lengths_into_a_tensor():
    bt = Batch([40, 50], [10, 20], H=1, G=1, D=64, seed=13)
    out = torch.zeros(2, dtype=torch.int32, device=DEV)
    check(bt, [[0, 4, 9], [0, 1, 19]], [3, 2], new_len=out)
    assert out.tolist() == [33, 32]
    check(bt, np.zeros((2, 0), np.int32), [0, 0])
