"""The example that runs the cache operators and the sampler together."""
from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_decode.py")


def example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_sessions_are_the_same_on_every_run_and_stay_within_their_budget():
    ex = example()
    a, cuts, lengths = ex.run(sessions=5, tokens=60, budget=32, chunk=20, seed=1)
    b, again, _ = ex.run(sessions=5, tokens=60, budget=32, chunk=20, seed=1)
    assert a.shape == (5, 60) and torch.equal(a, b) and cuts == again > 0
    assert int(a.min()) >= 0 and int(a.max()) < 4000
    assert all(n <= 2 * 32 + 1 for layer in lengths for n in layer)


def test_a_cache_layer_attends_like_its_definition():
    """Chunks and single tokens through the cache, against all tokens at once in fp64."""
    ex = example()
    g = torch.Generator(ex.DEV).manual_seed(0)
    cache = ex.Cache(2, 64, 2, 64, 16, 64, window=24, sinks=3)
    counts = [[30, 7], [1, 1], [5, 0], [1, 1]]
    T = [sum(c[s] for c in counts) for s in (0, 1)]
    q, k, v = ([torch.randn(n, h, 64, generator=g, device=ex.DEV).to(torch.bfloat16) for n in T] for h in (4, 2, 2))
    got, at = [[], []], [0, 0]
    for c in counts:
        cut = [torch.cat([x[s][at[s]:at[s] + c[s]] for s in (0, 1)]) for x in (q, k, v)]
        out = cache.attend(*cut, c)
        got[0].append(out[:c[0]])
        got[1].append(out[c[0]:])
        at = [a + n for a, n in zip(at, c)]
    for s in (0, 1):
        p, j = torch.arange(T[s])[:, None], torch.arange(T[s])[None]
        seen = ((j <= p) & ((j > p - 24) | (j < 3)))[None]
        qs, ks, vs = (x[s].double().cpu().transpose(0, 1) for x in (q, k, v))
        ks, vs = ks.repeat_interleave(2, 0), vs.repeat_interleave(2, 0)
        w = (qs @ ks.transpose(1, 2).contiguous() / 8).masked_fill(~seen, float("-inf")).softmax(-1)
        want, size = (w @ vs).transpose(0, 1), (w @ vs.abs()).transpose(0, 1)
        # a weight rounded to bf16 and the output once more, and some steps of fp32
        err = (torch.cat(got[s]).double().cpu() - want).abs()
        assert torch.all(err <= 2.0 ** -8 * (size + want.abs()) + 1e-4 * size)
