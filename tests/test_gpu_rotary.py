"""Rotary positions against the formula in 64 bits.

Bounds, an element: cos and sin are off by 2^-25 (the series' end) and some roundings of fp32: 4 U of
them, U = 2^-24, and the reduced angle by its own rounding, U pi / 4; the sum of two products by 3 U of their
sizes; all rounded once to the type (half a step)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, U, Batch

pytestmark = pytest.mark.gpu

F32 = torch.float32


def formula(x, positions, freqs, interleaved=False, scale=1.0):
    """The turned values in 64 bits and bounds of the errors (numpy)."""
    x = x.double().cpu().numpy()
    R = 2 * freqs.shape[0]
    a = np.outer(positions.double().cpu().numpy(), freqs.double().cpu().numpy())[:, None]
    lo, hi = (np.s_[..., 0:R:2], np.s_[..., 1:R:2]) if interleaved else (np.s_[..., :R // 2], np.s_[..., R // 2:R])
    out, tol = x.copy(), np.zeros_like(x)
    c, s = np.cos(a) * scale, np.sin(a) * scale
    out[lo], out[hi] = x[lo] * c - x[hi] * s, x[hi] * c + x[lo] * s
    # an angle of n quarter turns in 53 bits besides: 2^-52 of it
    tol[lo] = tol[hi] = abs(scale) * (np.abs(x[lo]) + np.abs(x[hi])) * (10 * U + np.abs(a) * 2.0 ** -51)
    return out, tol


def check(got, x, positions, freqs, dt, **kw):
    want, tol = formula(x, positions, freqs, **kw)
    got = got.double().cpu().numpy()
    R = 2 * freqs.shape[0]
    assert np.array_equal(got[..., R:], want[..., R:])
    eps = torch.finfo(dt).eps / 2
    tol = tol + eps * (np.abs(want) + tol) + torch.finfo(dt).smallest_normal * eps
    bad = np.abs(got - want)[..., :R] > tol[..., :R]
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want)[..., :R][bad][:4], tol[..., :R][bad][:4])


@pytest.mark.parametrize("dt", [F32, HF, BF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T, H, D, R", [(1, 1, 8, 2), (1, 40, 128, 128), (3, 5, 64, 20), (17, 3, 80, 80), (5, 2, 96, 24), (2, 9, 256, 32),
                                        (700, 40, 128, 64), (1, 3, 1024, 1024), (9, 1, 8, 8), (33, 7, 64, 48)])
def test_rotary(dt, interleaved, T, H, D, R):
    g = torch.Generator(DEV).manual_seed(T + H)
    x = torch.randn(T, H, D, generator=g, device=DEV).to(dt)
    positions = torch.randint(0, 5000, (T,), generator=g, device=DEV, dtype=torch.int32)
    freqs = tm.rotary_frequencies(R, device=DEV)
    check(tm.rotary(x, positions, freqs, interleaved=interleaved), x, positions, freqs, dt, interleaved=interleaved)


def test_positions_of_any_size_and_scales():
    g = torch.Generator(DEV).manual_seed(1)
    positions = torch.tensor([0, 1, -1, 10 ** 6, -123456789, 2 ** 31 - 1, -2 ** 31, 77], dtype=torch.int32, device=DEV)
    x = torch.randn(8, 2, 64, generator=g, device=DEV)
    for freqs in (tm.rotary_frequencies(64, device=DEV), torch.linspace(-3, 3, 32, device=DEV), torch.zeros(32, device=DEV)):
        for scale in (1.0, -0.25, 0.0, 3.5):
            check(tm.rotary(x, positions, freqs, scale=scale), x, positions, freqs, F32, scale=scale)
    # Quarter turns, on the border of the reduction.
    freqs = torch.full((32,), float(np.pi / 4), device=DEV)
    positions = torch.arange(-4, 4, dtype=torch.int32, device=DEV)
    check(tm.rotary(x, positions, freqs), x, positions, freqs, F32)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_strides_and_back(dt, interleaved):
    g = torch.Generator(DEV).manual_seed(2)
    packed = torch.randn(50, 9, 64, generator=g, device=DEV).to(dt)
    positions, freqs = torch.arange(50, dtype=torch.int32, device=DEV) * 1000, tm.rotary_frequencies(32, device=DEV)
    before = packed.clone()
    view = packed[:, 2:7]
    want = tm.rotary(view, positions, freqs, interleaved=interleaved)
    assert torch.equal(packed, before)
    got = tm.rotary(view, positions, freqs, interleaved=interleaved, out=view)
    assert got is view or got.data_ptr() == view.data_ptr()
    assert torch.equal(packed[:, 2:7], want) and torch.equal(packed[:, :2], before[:, :2]) and torch.equal(packed[:, 7:], before[:, 7:])
    back = tm.rotary(want, -positions, freqs, interleaved=interleaved)
    # twice the rounding to the type, of values of up to |x| + |y|
    eps = torch.finfo(dt).eps
    assert float((back.float() - before[:, 2:7].float()).abs().max()) <= 2 * eps * 2 * float(before.float().abs().max())
    heads_first = torch.randn(9, 50, 64, generator=g, device=DEV).to(dt).transpose(0, 1)
    check(tm.rotary(heads_first, positions, freqs, interleaved=interleaved), heads_first, positions, freqs, dt, interleaved=interleaved)
    assert tm.rotary(packed[:0], positions[:0], freqs).shape == (0, 9, 64)
    assert tm.rotary(packed[:, :0], positions, freqs).shape == (50, 0, 64)


def test_infinities_stay_in_their_pair():
    x = torch.ones(1, 2, 64, device=DEV)
    x[0, 0, 3], x[0, 1, 40] = float("inf"), float("nan")
    y = tm.rotary(x, torch.tensor([7], dtype=torch.int32, device=DEV), tm.rotary_frequencies(32, device=DEV))
    odd = ~torch.isfinite(y[0])
    assert odd[0].nonzero().flatten().tolist() == [3, 19] and odd[1].nonzero().flatten().tolist() == [40]


def test_the_gradient_is_the_turn_back():
    """y = A x with a rotation A: the gradient of sum(w y) is A^T w, against differences too."""
    g = torch.Generator(DEV).manual_seed(3)
    x, w = (torch.randn(4, 1, 16, generator=g, device=DEV) for _ in range(2))
    positions, freqs = torch.tensor([0, 3, 90, 7000], dtype=torch.int32, device=DEV), tm.rotary_frequencies(16, device=DEV)
    grad = tm.rotary(w, -positions, freqs)
    for e in range(16):
        step = torch.zeros_like(x)
        step[..., e] = 1.0   # (linear: a step of one loses nothing)
        d = ((tm.rotary(x + step, positions, freqs).double() - tm.rotary(x - step, positions, freqs).double()) * w.double()).sum((1, 2)) / 2
        assert torch.allclose(d, grad[:, 0, e].double(), rtol=0, atol=16 * 8 * 12 * U)


def appended(bt, Q, freqs, dt, *, interleaved=False, positions=None, seed=5, scores=True, **kw):
    """A packed projection through kv_append_rotary: the calls' tensors and what came out."""
    T, g = sum(bt.q), torch.Generator(DEV).manual_seed(seed)
    x = torch.randn(T, Q + 2 * bt.H, bt.D, generator=g, device=DEV).to(dt)
    q, k, v = x.split([Q, bt.H, bt.H], 1)
    out = tm.kv_append_rotary(q if Q else None, k, v, bt.k, bt.v, bt.tables, bt.kv_len, bt.q_start, positions, freqs, max_q=bt.max_q,
                              interleaved=interleaved, scores=bt.scores if scores else None, **kw)
    return q, k, v, out


@pytest.mark.parametrize("dt", [HF, BF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kv, q, H, Q, D, R, given", [([9], [1], 1, 1, 64, 64, False), ([40, 3, 17, 1], [1, 1, 1, 1], 2, 8, 128, 128, True),
                                                      ([90, 200], [31, 180], 2, 6, 80, 40, True), ([50, 33], [7, 2], 3, 0, 64, 24, False),
                                                      ([300, 0, 12], [5, 0, 12], 1, 7, 256, 20, True)])
def test_append(dt, interleaved, kv, q, H, Q, D, R, given):
    bt = Batch(kv, q, H=H, G=1, D=D, dt=dt, seed=3)
    freqs = tm.rotary_frequencies(R, device=DEV)
    places = np.concatenate([np.arange(n - m, n) for n, m in zip(kv, q)])
    positions = torch.from_numpy((places * 3 + 100000 if given else places).astype(np.int32)).to(DEV)
    before = [t.clone() for t in (bt.k, bt.v, bt.scores)]
    qs, ks, vs, out = appended(bt, Q, freqs, dt, interleaved=interleaved, positions=positions if given else None)
    if Q:
        check(out, qs, positions, freqs, dt, interleaved=interleaved)
    else:
        assert out is None
    at = 0
    for b, (n, m) in enumerate(zip(kv, q)):
        if m:
            p, s = bt.where(b, np.arange(n - m, n))
            check(bt.k[p, :, s], ks[at:at + m], positions[at:at + m], freqs, dt, interleaved=interleaved)
            assert torch.equal(bt.v[p, :, s], vs[at:at + m]) and (bt.scores[p, :, s] == 0).all()
            for t, old in zip((bt.k, bt.v, bt.scores), before):
                t[p, :, s] = old[p, :, s]
        at += m
    for t, old in zip((bt.k, bt.v, bt.scores), before):   # and nothing else
        assert torch.equal(t.view(torch.int16 if t.element_size() == 2 else torch.int32), old.view(torch.int16 if t.element_size() == 2 else torch.int32))


def test_append_rows_of_no_token_and_unmapped_pages():
    bt = Batch([40, 20], [4, 3], H=2, G=1, D=64, seed=1)
    bt.host[0][2] = -1   # positions 32 to 47 of the first
    bt.tables.copy_(torch.from_numpy(bt.host))
    freqs, T = tm.rotary_frequencies(64, device=DEV), 9
    g = torch.Generator(DEV).manual_seed(4)
    q, k = (torch.randn(T, 2, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    out = torch.full_like(q, 7.0)
    pools = [t.clone() for t in (bt.k, bt.v)]
    positions = torch.arange(T, dtype=torch.int32, device=DEV)
    tm.kv_append_rotary(q, k, k, bt.k, bt.v, bt.tables, bt.kv_len, bt.q_start, positions, freqs, max_q=2, out=out)
    done = [0, 1, 4, 5]   # max_q leaves out tokens 2, 3 and 6; 7 and 8 are of no sequence
    check(out[done], q[done], positions[done], freqs, BF)
    left = [2, 3, 6, 7, 8]
    assert (out[left] == 7.0).all()
    p, s = bt.where(1, np.arange(17, 19))
    check(bt.k[p, :, s], k[4:6], positions[4:6], freqs, BF)
    for t, old in zip((bt.k, bt.v), pools):
        t[p, :, s] = old[p, :, s]
        assert torch.equal(t.view(torch.int16), old.view(torch.int16))


def test_append_in_place_agrees_with_its_parts():
    """Queries turned where they lie, and the same as rotary and kv_append one after the other, bit for bit."""
    for R, interleaved in ((64, False), (32, True), (20, False)):
        a, b = (Batch([70, 33], [8, 5], H=2, G=2, D=64, dt=HF, seed=6) for _ in range(2))
        freqs = tm.rotary_frequencies(R, device=DEV)
        positions = torch.arange(13, dtype=torch.int32, device=DEV) + 40
        g = torch.Generator(DEV).manual_seed(9)
        x = torch.randn(13, 8, 64, generator=g, device=DEV).to(HF)
        q, k, v = x.clone().split([4, 2, 2], 1)
        got = tm.kv_append_rotary(q, k, v, a.k, a.v, a.tables, a.kv_len, a.q_start, positions, freqs, max_q=8, interleaved=interleaved,
                                  scores=a.scores, out=q)
        turned = tm.rotary(x[:, :6], positions, freqs, interleaved=interleaved)
        tm.kv_append(turned[:, 4:], x[:, 6:], b.k, b.v, b.tables, b.kv_len, b.q_start, max_q=8, scores=b.scores)
        assert torch.equal(got, turned[:, :4])
        for s, t in ((a.k, b.k), (a.v, b.v), (a.scores.view(torch.int32), b.scores.view(torch.int32))):
            assert torch.equal(s.view(torch.int16), t.view(torch.int16))
