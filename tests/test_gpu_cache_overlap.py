"""Outputs in the inputs' own memory: the same tensor where the header allows it, refused where they overlap otherwise."""
from __future__ import annotations

import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv, q, D", [([900, 70], [1, 1], 64), ([5000, 60], [2, 1], 128), ([300, 260], [200, 260], 128), ([9000], [50], 256)])
def test_attention_over_its_queries(kv, q, D):
    bt = Batch(kv, q, H=2, G=4, D=D, seed=8)
    want, lse = bt.attend()
    qd = bt.qs.to(DEV)
    got, l = bt.attend(q=qd, out=qd)
    assert got is qd and torch.equal(got, want) and torch.equal(l, lse)


def test_partial_overlap_is_refused():
    bt = Batch([90], [4], H=2, G=2, D=64, dt=HF, seed=1)
    wide = torch.zeros(5, 4, 64, dtype=HF, device=DEV)
    with pytest.raises(ValueError, match="out"):
        bt.attend(q=wide[:4], out=wide[1:])
    with pytest.raises(ValueError, match="out"):
        bt.attend(out=wide[:1].expand(4, 4, 64))
    pages = bt.scores.shape[0]
    sums = torch.zeros(pages + 1, 2, 16, device=DEV)
    lse = torch.zeros(4, 4, device=DEV)
    with pytest.raises(ValueError, match="out"):
        tm.kv_add_scores(bt.qs.to(DEV), lse, bt.k, sums[:pages], bt.tables, bt.kv_len, bt.q_start, max_q=4, max_kv=90, out=sums[1:])
    x = torch.randn(4, 1000, device=DEV)
    with pytest.raises(ValueError, match="out"):
        tm.adjust_logits(x[:3], out=x[1:])
    with pytest.raises(ValueError, match="out"):
        tm.adjust_logits(x, out=torch.zeros(1, 1000, device=DEV).expand(4, 1000))
    both = torch.randn(3, 2000, device=DEV)   # rows next to each other do not overlap
    assert torch.equal(tm.adjust_logits(both[:, :1000], out=both[:, 1000:]), both[:, :1000])
