"""The host's bounds: what lies past max_q and max_kv is left out, to the position."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("less", [1, 50, 127, 290])
@pytest.mark.parametrize("q, G, D, dt", [([1, 1], 4, 128, BF), ([9, 2], 2, 256, HF), ([60, 40], 2, 80, HF), ([0, 0], 1, 64, BF)])
def test_scores_past_max_kv_are_left(q, G, D, dt, less):
    kv = [300, 200]
    bt = Batch(kv, q, H=2, G=G, D=D, page=16, dt=dt, seed=less)
    lse = bt.attend()[1]
    args = (bt.qs.to(DEV), lse, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start)
    whole, part = torch.full_like(bt.scores, 7.0), torch.full_like(bt.scores, 7.0)
    tm.kv_add_scores(*args, max_q=bt.max_q, max_kv=300, out=whole)
    tm.kv_add_scores(*args, max_q=bt.max_q, max_kv=300 - less, out=part)
    for b, n in enumerate(kv):
        p, s = bt.where(b, np.arange(n))
        want = whole[p, :, s]
        want[300 - less:] = 7.0
        assert torch.equal(part[p, :, s], want)


@pytest.mark.parametrize("q, most", [([9, 3], 4), ([60, 200], 50), ([60, 2], 20), ([5, 7], 0)])
def test_tokens_past_max_q_are_left(q, most):
    kv = [300, 250]
    bt = Batch(kv, q, H=2, G=2, D=64, seed=most)
    first = np.concatenate([np.arange(n) < most for n in q])
    qd = bt.qs.to(DEV)
    want, lse = bt.attend(q=qd)
    out, l = torch.full_like(want, 7.0), torch.full_like(lse, 7.0)
    where = (bt.tables, bt.kv_len, bt.q_start)
    tm.paged_attention(qd, bt.k, bt.v, *where, max_q=most, max_kv=300, out=out, lse=l)
    got, per_row = out[first].float(), want[first].float()
    # (another split of the keys, other roundings: a step of each output)
    assert torch.all((got - per_row).abs() <= 2 * torch.finfo(BF).eps * (1 + per_row.abs()))
    assert torch.all(out[~first] == 7) and torch.all(l[~first] == 7)
    none = lse.clone()
    none[~torch.from_numpy(first).to(DEV)] = float("-inf")   # rows that add nothing
    a, b = torch.full_like(bt.scores, 7.0), torch.full_like(bt.scores, 7.0)
    tm.kv_add_scores(qd, none, bt.k, bt.scores, *where, max_q=bt.max_q, max_kv=300, out=a)
    tm.kv_add_scores(qd, lse, bt.k, bt.scores, *where, max_q=most, max_kv=300, out=b)
    held = a != 7
    assert torch.equal(held, b != 7) and torch.allclose(a[held], b[held], rtol=300 * 2.0 ** -24, atol=0, equal_nan=True)
    new = torch.randn(sum(q), 2, 64, device=DEV).to(BF)
    k0 = bt.k.clone()
    tm.kv_append(new, new, bt.k, bt.v, *where, max_q=most)
    for s, n in enumerate(q):
        p, at = bt.where(s, np.arange(kv[s] - n, kv[s]))
        rows = new[bt.starts[s]:bt.starts[s + 1]]
        m = min(n, most)
        assert torch.equal(bt.k[p[:m], :, at[:m]], rows[:m]) and torch.equal(bt.k[p[m:], :, at[m:]], k0[p[m:], :, at[m:]])


def test_evictions_end_with_max_kv():
    """As sequences of that length."""
    got = []
    for kv, most in (([300, 120], 200), ([200, 120], 200)):
        bt = Batch([300, 120], [0, 0], H=2, D=64, seed=4, extra=8)
        used = set(bt.host[bt.host >= 0].tolist())
        dst = torch.tensor([p for p in range(bt.k.shape[0]) if p not in used][:8], dtype=torch.int32, device=DEV).view(2, 4)
        bt.kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
        n, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, dst, budget=64, max_kv=most, sinks=2, recent=9)
        got.append((n, kept, bt.k.view(torch.int16), bt.scores.view(torch.int32)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
