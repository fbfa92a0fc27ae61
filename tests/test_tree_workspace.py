"""The tree attention's workspace at the largest bounds serves every smaller call: it does not shrink
with more positions, sequences, nodes or query heads."""
from __future__ import annotations

import ctypes as C

import pytest

from tensormark_amd import cache, tree
from test_cache_args import a_cache, rows_args

KV = (1, 100, 256, 257, 512, 513, 1000, 1025, 5000, 40000)
BATCH = (1, 2, 8, 33, 200)
NODES = (1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 257, 512)
GROUP = (1, 2, 4, 8)


def need(D, H, kv, batch, q, group, window):
    c = a_cache(max_kv=kv, table_stride=40000, batch=batch, tokens=q * batch, max_q=q, head_dim=D, kv_heads=H)
    for s in (c.k_stride, c.v_stride):
        s[:] = [16 * D * H, 16 * D, D]
    a = rows_args(cache.AttentionArgs, q_heads=group * H, window=window, sinks=4)
    a.q_stride[:] = a.out_stride[:] = [group * H * D, D]
    return tree._fns().tms_tree_attention_workspace(C.byref(c), C.byref(a))


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("D", [64, 128, 136, 256])
@pytest.mark.parametrize("H", [1, 8])
def test_workspaces_grow_with_every_bound(D, H, window):
    sizes = {at: need(D, H, *at, window) for at in
             ((kv, b, q, g) for kv in KV for b in BATCH for q in NODES for g in GROUP)}
    assert min(sizes.values()) >= 0
    for axis, steps in enumerate((KV, BATCH, NODES, GROUP)):
        for at, size in sizes.items():
            i = steps.index(at[axis])
            if i:
                below = at[:axis] + (steps[i - 1],) + at[axis + 1:]
                assert sizes[below] <= size, (below, at, sizes[below], size)
