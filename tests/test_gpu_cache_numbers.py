"""Numbers at the edges of the cache operators' types: weights far below a row's
largest, rows and keys that are no numbers."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, U, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("q, G, D, copies", [(1, 1, 64, 1), (1, 4, 128, 128), (2, 2, 256, 128), (40, 1, 64, 1), (40, 1, 64, 512),
                                             (34, 1, 128, 512), (33, 1, 256, 512)])
def test_many_small_weights_beside_a_large_one(q, G, D, copies, dt):
    """One key takes nearly all of a row's weight and 150,000 others some 2^-25 of it
    each, 0.4 percent together: they all count, in the output as in its sum.  Many
    sequences share the pages, so that the card does not share out one's keys."""
    L, low = 150_000, -17.375
    bt = Batch([L], [q], H=1, G=G, D=D, page=64, dt=dt, seed=1)
    bt.qs[:] = 0
    bt.qs[..., 0] = 1
    bt.keys[0][:, 0, 0] = low
    bt.keys[0][3, 0, 0] = 0
    bt.values[0][:] = 1 + torch.arange(D) / 64
    bt.values[0][3] = 0
    bt.fill()
    o, l = tm.paged_attention(bt.qs.to(DEV).repeat(copies, 1, 1), bt.k, bt.v, bt.tables.repeat(copies, 1), bt.kv_len.repeat(copies),
                              q * torch.arange(copies + 1, dtype=torch.int32, device=DEV), max_q=q, max_kv=L, scale=1.0)
    o, l = o.double().cpu(), l.double().cpu()
    n = (L - q + torch.arange(q, dtype=torch.float64)).repeat(copies)[:, None, None]   # small weights of each token
    w = math.exp(low)
    want = n * w / (1 + n * w) * bt.values[0][0, 0].double()
    # A weight is off by half a step of the type and by its argument's error in fp32 (some steps of
    # 25); running sums by a step for every 16 keys; the output by half a step.
    err = 16 * 25 * U + L // 16 * U
    half = torch.finfo(dt).eps / 2
    tiny = torch.finfo(dt).smallest_normal * half if dt == HF else 0.0   # half a step of an output below the normal ones
    assert torch.all((o - want).abs() <= (2 * half + 2 * err) * want + tiny)
    assert torch.all((l - (1 + n * w).log()[..., 0]).abs() <= err + 8 * U)


def added(bt, lse, window=0, sinks=0, odd=None):
    """kv_add_scores onto sums of its own, checked where the definition gives a number: what rows
    without one add is none, to the keys they see and to no others."""
    with np.errstate(invalid="ignore"):
        weights, wtol = bt.reference(window, sinks)[4:]
    out = torch.full_like(bt.scores, 7.0)
    tm.kv_add_scores(bt.qs.to(DEV), lse, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q, max_kv=bt.max_kv,
                     window=window, sinks=sinks, out=out)
    most = lse[torch.isfinite(lse)].abs().max().item()
    for b, n in enumerate(bt.kv):
        p, s = bt.where(b, np.arange(n))
        new = out[p, :, s].double().cpu().numpy()
        for h in range(bt.H):
            w, had = weights[b * bt.H + h], bt.sums[b][:, h].double().numpy()
            none = np.isnan(w)
            # paged_attention's lse is off by what its own sums and exponentials are (as the weights) and a rounding
            slack = 2 * wtol[b * bt.H + h] + w * U * 10 * most + 2 * U * np.abs(had + w)
            assert np.array_equal(np.isnan(new[:, h]), none), (h, np.flatnonzero(np.isnan(new[:, h]) != none)[:9])
            assert np.all(np.abs(new[:, h] - had - w)[~none] <= slack[~none])
    return out


@pytest.mark.parametrize("window, sinks", [(0, 0), (30, 4)])
@pytest.mark.parametrize("q, G, D, dt", [(9, 2, 64, BF), (60, 2, 80, HF), (150, 1, 128, BF), (100, 3, 64, HF), (5, 70, 256, BF)])
def test_a_query_that_is_no_number_reaches_the_keys_it_sees(q, G, D, dt, window, sinks):
    bt = Batch([200], [q], H=1, G=G, D=D, dt=dt, seed=q)
    bt.qs[q // 2, G - 1, 3] = float("nan")
    lse = bt.attend(window=window, sinks=sinks)[1]
    assert torch.isnan(lse[q // 2, G - 1]) and int(torch.isnan(lse).sum()) == 1
    added(bt, lse, window, sinks)


@pytest.mark.parametrize("q, G, D, dt", [(9, 2, 64, BF), (60, 2, 80, HF), (70, 3, 64, HF), (45, 1, 128, BF), (5, 70, 256, BF)])
def test_a_key_that_every_row_scores_minus_infinity(q, G, D, dt):
    """Its weight is zero in attention, and so is what its score grows by; the others' are right."""
    bt = Batch([300], [q], H=1, G=G, D=D, dt=dt, seed=q)
    bt.qs[..., 2] = bt.qs[..., 2].abs() + 0.25
    low = [1, 40, 130, 220]
    bt.keys[0][low, 0, 2] = float("-inf")
    bt.fill()
    lse = bt.attend()[1]
    assert torch.isfinite(lse).all()
    out = torch.full_like(bt.scores, 7.0)
    tm.kv_add_scores(bt.qs.to(DEV), lse, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=q, max_kv=300, out=out)
    p, s = bt.where(0, np.arange(300))
    grown = (out[p, 0, s].double() - bt.scores[p, 0, s].double()).cpu()
    assert torch.all(grown[low] == 0)
    # every row's weights sum to one: (kv + rows + 32) steps of fp32, and a step of each sum so far
    assert abs(float(grown.sum()) - q * G) <= q * G * (300 + 32) * U + U * float(out[p, 0, s].double().sum())


@pytest.mark.parametrize("scale", [3e38, -3e38, 1e-45, -1e-38])
@pytest.mark.parametrize("q, D", [(3, 64), (50, 128), (40, 256)])
def test_a_scale_at_the_type_s_ends(q, D, scale):
    """Rows that score every key 0 weigh all alike, whatever the scale."""
    bt = Batch([130], [q], H=1, G=2, D=D, dt=HF, seed=q)
    bt.qs[:] = 0
    out, lse, tol, ltol, weights, wtol = bt.reference(scale=1.0)
    o, l = bt.attend(scale=scale)
    assert np.all(np.abs(o.double().cpu().numpy() - out) <= tol) and np.all(np.abs(l.double().cpu().numpy() - lse) <= ltol)
    zero = torch.zeros_like(bt.scores)
    tm.kv_add_scores(bt.qs.to(DEV), l, bt.k, zero, bt.tables, bt.kv_len, bt.q_start, max_q=q, max_kv=130, scale=scale)
    p, s = bt.where(0, np.arange(130))
    want = weights[0]
    assert np.all(np.abs(zero[p, 0, s].double().cpu().numpy() - want) <= 2 * wtol[0] + want * U * 10 * np.abs(lse).max() + 2 * U * want)
