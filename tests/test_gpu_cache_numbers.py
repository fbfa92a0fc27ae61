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
