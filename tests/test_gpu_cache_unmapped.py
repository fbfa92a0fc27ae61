"""Eviction of sequences of which some pages have been given back: what is not there
is not kept, and attention over the cut cache is attention over what was."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch, check

pytestmark = pytest.mark.gpu


def kept_of(bt, budget, sinks, recent):
    """Kept positions [B][H] by the definition."""
    kept = []
    for b, L in enumerate(bt.kv):
        page = bt.host[b][np.arange(L) // bt.page] if L else np.zeros(0, np.int32)
        there = np.flatnonzero((page >= 0) & (page < bt.k.shape[0]))
        row = []
        for h in range(bt.H):
            s = bt.sums[b][:, h].double().numpy()
            rank = sorted(there.tolist(), key=lambda j: (0, 0.0, j) if j < sinks or j >= L - recent else
                          (2, 0.0, j) if math.isnan(s[j]) else (1, -s[j], j))
            row.append(np.array(sorted(rank[:budget]), np.int64))
        kept.append(row)
    return kept


CASES = [   # kv, entries given back (of sequence 0), budget, sinks, recent, page
    ([100], [2], 200, 4, 8, 16),                          # all fits the budget
    ([3000, 300], list(range(1, 155)), 1024, 4, 64, 16),  # a window's pages left, fewer than the budget
    ([3000, 300], list(range(1, 155)), 200, 4, 64, 16),
    ([400], [0, 3, 24], 100, 20, 40, 16),                 # holes among the sinks and the last
    ([400], [1, 2, 3], 100, 4, 40, 64),
    ([400], [0, 1, 2, 3, 4, 5, 6], 100, 4, 40, 64),       # nothing there
    ([77, 90], [1, 2], 60, 30, 30, 8),                    # guarded positions fill the budget
    ([20000, 17000], [0, 3, 70], 900, 4, 300, 64),        # past what registers hold
    ([20000], list(range(1, 310)), 900, 4, 300, 64),
    ([20000], list(range(1, 250)), 8000, 1, 30, 64),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("values", ["spread", "ties", "nan"])
@pytest.mark.parametrize("kv, gone, budget, sinks, recent, page", CASES)
def test_positions_without_a_page_are_not_kept(kv, gone, budget, sinks, recent, page, values, in_place):
    each = -(-min(budget, max(kv)) // page)
    bt = Batch(kv, [0] * len(kv), H=2, D=64, page=page, dt=HF if page == 64 else BF, seed=budget, extra=len(kv) * each + 1)
    rng = np.random.default_rng(budget)
    for b, L in enumerate(kv):
        if values == "ties":
            bt.sums[b] = torch.from_numpy(rng.integers(0, 2, (L, 2)).astype(np.float32))
        elif values == "nan":
            bt.sums[b][torch.from_numpy(rng.random((L, 2)) < 0.7)] = float("nan")
    bt.fill()
    used = set(bt.host[bt.host >= 0].tolist())
    free = [p for p in range(bt.k.shape[0]) if p not in used]
    dst = np.array(free[:len(kv) * each], np.int32).reshape(len(kv), each)
    bt.host[0, gone] = [-1, 10 ** 7, -5][:1] * len(gone) if len(gone) < 3 else ([-1, 10 ** 7, -5] * len(gone))[:len(gone)]
    bt.tables = torch.from_numpy(bt.host).to(DEV)
    want = kept_of(bt, budget, sinks, recent)
    new_len, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, torch.from_numpy(dst).to(DEV), budget=budget,
                                max_kv=bt.max_kv, sinks=sinks, recent=recent, new_len=bt.kv_len if in_place else None)
    lengths = [len(w[0]) for w in want]
    assert new_len.tolist() == lengths
    kept = kept.cpu().numpy()
    for b, n in enumerate(lengths):
        for h in range(2):
            assert np.array_equal(kept[b, h, :n], want[b][h]) and np.all(kept[b, h, n:] == -1)
    # the cut cache: the pools hold NaN wherever nothing was put
    after = Batch(lengths, [min(n, 1) for n in lengths], H=2, G=2, D=64, page=page, dt=bt.dt, seed=1)
    after.host, after.tables, after.k, after.v = dst, torch.from_numpy(dst).to(DEV), bt.k, bt.v
    for b, n in enumerate(lengths):
        for h in range(2):
            after.keys[b][:, h], after.values[b][:, h] = bt.keys[b][want[b][h], h], bt.values[b][want[b][h], h]
        p, s = after.where(b, np.arange(n))
        for h in range(2):
            got = bt.scores[p, h, s].cpu()
            assert torch.equal(got.view(torch.int32), bt.sums[b][want[b][h], h].view(torch.int32))
    check(after)


@pytest.mark.parametrize("budget", [2 ** 31 - 1, 2 ** 31 - 1024, 2 ** 31 - 1025])
def test_a_budget_that_is_no_limit(budget):
    """All is kept; every place of `kept` past that says so, up to the last of 8 GiB."""
    bt = Batch([50], [0], H=1, D=64, page=16, seed=3, extra=4)
    used = set(bt.host[bt.host >= 0].tolist())
    dst = torch.tensor([[p for p in range(bt.k.shape[0]) if p not in used][:4]], dtype=torch.int32, device=DEV)
    kept = torch.full((1, 1, budget), 7, dtype=torch.int32, device=DEV)
    new_len, _ = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, dst, budget=budget, max_kv=50, sinks=4, recent=8, kept=kept)
    assert new_len.tolist() == [50] and kept[0, 0, :50].tolist() == list(range(50))
    assert all(bool((part == -1).all()) for part in kept[0, 0, 50:].split(1 << 28))
    p, s = bt.where(0, np.arange(50))
    to, at = dst[0][torch.arange(50, device=DEV) // 16].long(), torch.arange(50, device=DEV) % 16
    assert torch.equal(bt.k[to, 0, at], bt.k[p, 0, s]) and torch.equal(bt.scores[to, 0, at], bt.scores[p, 0, s])
