"""Forward-mode derivatives: no call carries a tangent, so a dual tensor that a call would take one
from is refused, whatever the gradient mode."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

import test_cache_autograd as paged
import test_tree_args as tree

TAKES = [(paged.some, paged.calls, call, name) for call, names in paged.TAKES.items() for name in names]
TAKES += [(tree.some, tree.calls, call, name) for call, names in tree.TAKES.items() for name in names]


@pytest.mark.parametrize("some, calls, call, name", TAKES, ids=lambda x: x if isinstance(x, str) else x.__module__)
def test_a_tensor_with_a_tangent_is_refused(some, calls, call, name):
    with fw.dual_level():
        x = some("cpu")
        x[name] = fw.make_dual(x[name], torch.ones_like(x[name]))
        for mode in (torch.enable_grad, torch.no_grad):   # (no_grad leaves tangents on)
            with mode(), pytest.raises(ValueError, match="tangent"):
                calls(x)[call]()
        x[name] = fw.unpack_dual(x[name]).primal
        with pytest.raises(ValueError) as e:   # (a host tensor is refused all the same)
            calls(x)[call]()
        assert "tangent" not in str(e.value)


@pytest.mark.gpu
def test_calls_under_a_level_without_tangents_run():
    with fw.dual_level():
        for module in (paged, tree):
            for call in module.TAKES:
                module.calls(module.some("cuda:0"))[call]()
