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
