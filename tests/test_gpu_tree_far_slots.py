"""Trees of more than 32 rows a key head where the kernel of few rows has them, in tiles of 32: pools
whose slots span 2^32 bytes.  And heads past 128 dimensions under a window."""
from __future__ import annotations

import pytest
import torch

from test_gpu_cache import BF, DEV, HF, check
from test_gpu_tree_attention import TreeBatch

pytestmark = pytest.mark.gpu


def far_apart(bt):
    """The batch's one sequence on a page whose slots lie 64 KB apart."""
    step, page, n = 32768, bt.page, bt.kv[0]
    buf = torch.zeros(step * page + 128, dtype=bt.dt, device=DEV)
    k, v = (buf.as_strided((1, 1, page, 64), (step * page, step * page, step, 1), at) for at in (0, 64))
    k[:, :, :n], v[:, :, :n] = bt.k[:, :, :n], bt.v[:, :, :n]
    bt.k, bt.v = k, v
    return bt


@pytest.mark.parametrize("kind", ["random", "chain"])
@pytest.mark.parametrize("kv", [300, 1500])   # an item a workgroup, and shares with a join
@pytest.mark.parametrize("q, G", [(40, 3), (100, 1), (47, 7)])   # a token's heads in two tiles, and not
def test_slots_far_apart(q, G, kv, kind):
    bt = far_apart(TreeBatch([kv], [q], H=1, G=G, D=64, page=65536, extra=0, kind=kind, seed=q))
    for window, sinks in ((0, 0), (33, 2), (5, 0), (700, 3)):
        check(bt, window, sinks)


@pytest.mark.parametrize("q", [[40, 25], [140, 90], [7, 3]])
@pytest.mark.parametrize("window, sinks", [(1, 0), (16, 0), (64, 5), (200, 130)])
@pytest.mark.parametrize("D, dt", [(256, BF), (136, HF)])
def test_windows_past_128_dimensions(q, window, sinks, D, dt):
    for kind in ("random", "chain"):
        check(TreeBatch([400, 190], q, H=1, G=2, D=D, dt=dt, page=32, kind=kind, seed=window), window, sinks)
