"""The verify of trees where a sequence has several parts and none waits for another: each works all
the others' sums out itself, in every type, for vocabularies and rows of odd sizes, and where nothing is left
of a target row."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import tensormark_amd as tm
from test_gpu_verify_tree import BF, F32, HF, Trees

pytestmark = pytest.mark.gpu


@pytest.fixture
def polls():
    lib = tm.load_library()
    lib.tms_debug_verify_polls.argtypes = [C.c_int]
    yield lib.tms_debug_verify_polls
    lib.tms_debug_verify_polls(-1)


@pytest.mark.parametrize("dt", [F32, HF, BF])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [40000, 70003])
def test_no_part_waits(dt, drawn, V, polls):
    t = Trees([9, 1, 12], V, drawn=drawn, dt=dt, seed=V, sharp=3.0)
    for n in (0, 1, -1):
        polls(n)
        for pad, offset in ((0, 0), (3, 1), (8, 5)):
            t.check(pad=pad, offset=offset)


@pytest.mark.parametrize("dt", [F32, HF, BF])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [40000, 70003])
def test_nothing_is_left(dt, drawn, V, polls):
    """All of a row's mass is refused (rows that sum to less than 1): the token is the target row's own."""
    t = Trees([4, 7], V, drawn=drawn, dt=dt, seed=V + 1, kind="star", sharp=3.0)
    t.u[:] = 0.9
    if drawn:
        t.target = t.draft * 0.5
    else:
        t.target[:] = 0
        for first, n in zip(t.starts[:-1], t.q):
            for i in range(1, n):
                t.tokens[first + i] = V - 1 - 5000 * (i - 1)
                t.target[first, int(t.tokens[first + i])] = 2.0 ** -4
    for n in (0, -1):
        polls(n)
        path, kept, token = t.check(offset=1, pad=2)
        assert (kept == 1).all() and (token >= 0).all()
        if not drawn:   # one of the refused
            assert all(x in t.tokens[a + 1:a + m] for x, a, m in zip(token, t.starts[:-1], t.q))


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("V", [33, 7000])
def test_rows_of_nothing_and_of_a_single_entry(drawn, V):
    t = Trees([5, 5], V, drawn=drawn, seed=7)
    t.target[0], t.target[5] = 0.0, 0.0
    t.target[5, V - 1] = 0.5
    path, kept, token = t.check()
    assert kept[0] == 1 and token[0] == -1
    assert np.array_equal(path[0], [0, -1, -1, -1, -1])
    assert token[1] == V - 1 or kept[1] > 1
