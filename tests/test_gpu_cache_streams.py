"""Every cache call on a stream that is not the current one, and evictions in full: each head's
keys, values and scores."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch, evicted

pytestmark = pytest.mark.gpu


def destinations(bt, each):
    used = set(bt.host[bt.host >= 0].tolist())
    free = [p for p in range(bt.k.shape[0]) if p not in used]
    return np.array(free[:len(bt.kv) * each], np.int32).reshape(len(bt.kv), each)


def bits(*tensors):
    return [t.view({2: torch.int16, 4: torch.int32}[t.element_size()]) for t in tensors]


def step(bt, qd, kn, vn, dst, x, stream=None):
    """A decode step's calls one after another."""
    where = (bt.tables, bt.kv_len, bt.q_start)
    kw = dict(max_q=bt.max_q, stream=stream)
    tm.kv_append(kn, vn, bt.k, bt.v, *where, scores=bt.scores, **kw)
    kw["max_kv"] = bt.max_kv
    out, lse = tm.paged_attention(qd, bt.k, bt.v, *where, **kw)
    tm.kv_add_scores(qd, lse, bt.k, bt.scores, *where, **kw)
    new_len, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, dst, budget=64, max_kv=bt.max_kv, sinks=4, recent=8,
                                stream=stream)
    return out, lse, new_len, kept, tm.adjust_logits(x, stream=stream)


@pytest.mark.parametrize("kv, q", [([1500, 90], [1, 1]), ([700, 300], [9, 40])])
def test_a_step_on_a_given_stream(kv, q):
    results = []
    for given in (False, True):
        bt = Batch(kv, q, H=2, G=2, D=64, seed=8, extra=9)
        dst = torch.from_numpy(destinations(bt, 4)).to(DEV)
        g = torch.Generator(DEV).manual_seed(1)
        kn, vn, qd = (torch.randn(sum(q), h, 64, generator=g, device=DEV).to(BF) for h in (2, 2, 4))
        x = torch.randn(2, 5000, generator=g, device=DEV)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        got = step(bt, qd, kn, vn, dst, x, side.cuda_stream if given else None)   # (the tensors are held past the end)
        side.synchronize()
        torch.cuda.synchronize()
        results.append(bits(*got, bt.k, bt.v, bt.scores))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("kv, budget, H, D, page, dt", [([5000, 4096, 700], 1000, 3, 64, 64, BF), ([20000], 1500, 4, 8, 16, HF),
                                                        ([3000, 2000], 777, 2, 256, 16, HF), ([2500], 1200, 5, 80, 32, BF)])
def test_an_eviction_in_full(kv, budget, H, D, page, dt, slot_major):
    each = -(-budget // page)
    bt = Batch(kv, [0] * len(kv), H=H, D=D, page=page, dt=dt, slot_major=slot_major, seed=budget, extra=len(kv) * each + 1)
    want, dst = evicted(bt, budget, 4, 64), destinations(bt, each)
    pools = [bt.k.clone(), bt.v.clone(), bt.scores.clone()]
    for b in range(len(kv)):
        for h in range(H):
            old, new = want[b][h], np.arange(len(want[b][h]))
            sp, ss, dp, ds = (torch.from_numpy(np.asarray(i).astype(np.int64)).to(DEV)
                              for i in (bt.host[b][old // page], old % page, dst[b][new // page], new % page))
            for pool, source in zip(pools, (bt.k, bt.v, bt.scores)):
                pool[dp, h, ds] = source[sp, h, ss]
    _, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, torch.from_numpy(dst).to(DEV), budget=budget,
                          max_kv=bt.max_kv, sinks=4, recent=64)
    kept = kept.cpu().numpy()
    assert all(np.array_equal(kept[b, h, :len(want[b][h])], want[b][h]) for b in range(len(kv)) for h in range(H))
    for got, w in zip((bt.k, bt.v, bt.scores), pools):
        assert torch.equal(*bits(got.contiguous(), w.contiguous()))
