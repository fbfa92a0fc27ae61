"""The cache operators where their kernels change hands: shares that cut
sequences, long lists of parts, groups and strides out of the ordinary, lengths
that change between a graph's replays.  Tolerances are test_gpu_cache's bounds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tensormark_amd as tm
from test_gpu_cache import BF, DEV, HF, U, Batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0])
@pytest.mark.parametrize("q, D", [([1, 3], 128), ([60, 90], 128), ([50, 1], 256)])
def test_any_finite_scale(q, D, scale):
    """A scale of zero weighs all alike, one below zero turns the order; masked keys stay masked."""
    bt = Batch([150, 90], q, H=2, G=2, D=D, seed=21)
    check(bt, scale=scale)
    check(bt, 20, 3, scale)


@pytest.mark.parametrize("dt, D, G", [(BF, 64, 3), (BF, 128, 4), (HF, 80, 1), (HF, 256, 2)])
def test_shares_cut_sequences(dt, D, G):
    """Lengths from nothing to 70 tiles, sequences without tokens, tokens that see
    nothing, and more sequences than a workgroup has threads to look through them."""
    kv = [2200, 1, 0, 33, 1500, 700, 0, 64, 1029, 31, 5, 1200]
    q = [1, 1, 1, 2, 1, 0, 0, 3, 1, 1, 2, 4]
    check(Batch(kv, q, H=2, G=G, D=D, dt=dt, seed=D))
    check(Batch(kv, q, H=2, G=G, D=D, dt=dt, seed=D), 300, 5)


def test_more_sequences_than_threads():
    rng = np.random.default_rng(0)
    kv = [1100] + rng.integers(0, 60, 700).tolist()
    check(Batch(kv, [1] * len(kv), H=1, G=2, D=64, seed=1))


def test_one_long_sequence():
    """Hundreds of parts to a row."""
    check(Batch([70000], [2], H=1, G=2, D=16, seed=2))


def test_chunk_in_splits():
    """Few tokens over many keys: the chunk kernel's shares of the keys."""
    for D in (64, 128, 256):
        check(Batch([5000, 40], [50, 40], H=1, G=1, D=D, page=32, seed=D))


def test_slots_far_apart():
    """Strides past the chunk kernel's 32 bits: more than 32 rows in tiles of 32."""
    step, page = 32768, 65536
    buf = torch.zeros(step * page + 128, dtype=BF, device=DEV)
    bt = Batch([300], [40], H=1, G=2, D=64, page=page, extra=0, seed=4)
    k = buf.as_strided((1, 1, page, 64), (step * page, step * page, step, 1))
    v = buf.as_strided((1, 1, page, 64), (step * page, step * page, step, 1), 64)
    k[:, :, :300], v[:, :, :300] = bt.k[:, :, :300], bt.v[:, :, :300]
    bt.k, bt.v = k, v
    check(bt)
    check(bt, 33, 2)


@pytest.mark.parametrize("what", [float("inf"), float("nan")])
@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("q", [5, 70])
def test_odd_values_reach_no_row_that_does_not_see_them(q, D, what):
    L = 200
    bt = Batch([L], [q], H=1, G=2, D=D, dt=HF, seed=D + q)
    p, s = bt.where(0, [L - 1])
    bt.v[p, :, s, 3:7] = what
    bt.k[p, :, s, 0] = what
    out, lse, tol, ltol, _, _ = bt.reference()
    o, l = (x.double().cpu().numpy() for x in bt.attend())
    assert np.all(np.abs(o[:-1] - out[:-1]) <= tol[:-1]) and np.all(np.abs(l[:-1] - lse[:-1]) <= ltol[:-1])
    # the last row sees the key: a score of minus infinity takes its weight, all else shows
    shows = np.isnan(what) | (bt.qs[-1, :, 0].double().numpy() > 0)
    assert not np.isfinite(o[-1, shows, 3:7]).any()


def added(bt, window=0, sinks=0):
    """Checks kv_add_scores for the batch."""
    _, lse, _, _, weights, wtol = bt.reference(window, sinks)
    l32 = torch.from_numpy(lse).to(DEV, torch.float32)
    out = torch.full_like(bt.scores, 7.0)
    tm.kv_add_scores(bt.qs.to(DEV), l32, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q, max_kv=bt.max_kv,
                     window=window, sinks=sinks, out=out)
    for b, n in enumerate(bt.kv):
        if not n:
            continue
        p, s = bt.where(b, np.arange(n))
        new = out[p, :, s].double().cpu().numpy()
        for h in range(bt.H):
            w = weights[b * bt.H + h]
            want = bt.sums[b][:, h].double().numpy() + w
            slack = wtol[b * bt.H + h] + w * U * 2 * np.nanmax(np.abs(np.where(np.isinf(lse), 0, lse)), initial=0)
            assert np.all(np.abs(new[:, h] - want) <= slack + 2 * U * np.abs(want))


@pytest.mark.parametrize("G, q", [(70, [3, 1]), (64, [2, 2]), (65, [1, 4]), (33, [1, 0]), (3, [100, 21]), (7, [50, 9]), (1, [128, 65])])
@pytest.mark.parametrize("window, sinks", [(0, 0), (30, 4)])
def test_scores_of_any_group(G, q, window, sinks):
    """Tiles of whole tokens, groups that a tile does not divide or hold."""
    added(Batch([300, 129], q, H=1, G=G, D=64, dt=HF, seed=G), window, sinks)


def test_scores_of_odd_keys_stay_theirs():
    """A key of NaN at a position that only the last token sees: every other key's sum is right."""
    for q in (9, 60):
        bt = Batch([200], [q], H=1, G=4, D=80, seed=q)
        lse = torch.from_numpy(bt.reference()[1]).to(DEV, torch.float32)
        args = dict(max_q=bt.max_q, max_kv=bt.max_kv)
        zero = torch.zeros_like(bt.scores)
        want = tm.kv_add_scores(bt.qs.to(DEV), lse, bt.k, zero, bt.tables, bt.kv_len, bt.q_start, out=zero.clone(), **args)
        p, s = bt.where(0, [199])
        bt.k[p, :, s] = float("nan")
        got = tm.kv_add_scores(bt.qs.to(DEV), lse, bt.k, zero, bt.tables, bt.kv_len, bt.q_start, out=zero.clone(), **args)
        want[p, :, s], got[p, :, s] = 0, 0
        assert torch.equal(got, want)


def test_lengths_change_between_replays():
    """One capture with the host's bounds serves every later length."""
    bt = Batch([1900, 1500, 40, 700], [1, 1, 1, 1], H=2, G=4, D=128, seed=31)
    qd = bt.qs.to(DEV)
    out, lse = torch.zeros_like(qd), torch.zeros(qd.shape[:2], device=DEV)
    bt.attend(q=qd)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bt.attend(q=qd, out=out, lse=lse)
    for lens in ([1900, 1500, 40, 700], [1, 900, 0, 699], [1024, 33, 40, 64]):
        bt.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want, wl = bt.attend(q=qd)
        assert torch.equal(out, want) and torch.equal(lse, wl)
        short = Batch([1900, 1500, 40, 700], [1, 1, 1, 1], H=2, G=4, D=128, seed=31)
        short.kv = lens
        short.keys = [k[:n] for k, n in zip(short.keys, lens)]
        short.values = [v[:n] for v, n in zip(short.values, lens)]
        check(short, got=(out, lse))


def test_results_on_a_given_stream():
    bt = Batch([1500, 90], [1, 1], H=2, G=2, D=64, seed=8)
    want, wl = bt.attend()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    o, l = bt.attend(stream=side.cuda_stream)
    dst = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    x = torch.randn(2, 5000, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    y = tm.adjust_logits(x, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(o, want) and torch.equal(l, wl) and torch.equal(x, y)
    del dst


@pytest.mark.parametrize("values", ["spread", "ties"])
def test_evict_writes_the_length_in_place(values):
    """new_len in kv_len's own place gives what a place of its own gives."""
    rng = np.random.default_rng(5)
    pools = []
    for own in (False, True):
        bt = Batch([9000, 6000, 300], [0, 0, 0], H=4, D=64, page=32, seed=6, extra=3 * 32)
        if values == "ties":
            bt.sums = [(s * 2).round() for s in bt.sums]
            bt.fill()
        used = set(bt.host[bt.host >= 0].tolist())
        free = np.array([p for p in range(bt.k.shape[0]) if p not in used][:96], np.int32).reshape(3, 32)
        new_len, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, torch.from_numpy(free).to(DEV), budget=1000,
                                    max_kv=9000, sinks=4, recent=100, new_len=bt.kv_len if own else None)
        assert new_len.tolist() == [1000, 1000, 300]
        pools.append([bt.k.view(torch.int16), bt.v.view(torch.int16), bt.scores.view(torch.int32), kept])
    assert all(torch.equal(a, b) for a, b in zip(*pools))
    kept = pools[0][3].cpu().numpy()
    for b, L in enumerate([9000, 6000]):
        for h in range(4):
            k = kept[b, h]
            assert np.all(np.diff(k) > 0) and np.array_equal(k[:4], np.arange(4)) and np.array_equal(k[-100:], np.arange(L - 100, L))
            s = bt.sums[b][:, h].numpy()
            rest = np.setdiff1d(np.arange(4, L - 100), k)
            mid = k[4:-100]
            assert s[mid].min() >= s[rest].max()
            edge = s[mid].min()   # of equal scores the lowest positions stay
            tied = np.flatnonzero(s[4:L - 100] == edge) + 4
            stay = np.isin(tied, mid)
            assert np.all(stay[:stay.sum()])
    del rng


def test_many_rows_in_place():
    """Several chunks a workgroup, results written over the logits."""
    from test_gpu_adjust import dev, plain, records, some

    R, V = 850, 20001
    x, p, recent, n_recent, _, bias = some(R, V, 1, 40, 2, 9)
    xd = dev(x).to(BF)
    base = xd.float().cpu().numpy()
    got = tm.adjust_logits(xd, records(p), recent=dev(recent), n_recent=dev(n_recent), bias_ids=dev(bias[0]),
                           bias_values=dev(bias[1]), out=xd)
    assert got is xd
    rows = [0, 1, 411, 849]
    want, err = plain(base[rows], 1, p[rows], recent[rows], n_recent[rows], None, (bias[0][rows], bias[1][rows]), None)
    half = torch.finfo(BF).eps / 2
    assert np.all(np.abs(got[rows].double().cpu().numpy() - want) <= err * (1 + half) + half * np.abs(want))
    same = np.ones((R, V), bool)   # ids that nothing names keep their bits
    np.put_along_axis(same, np.clip(recent, 0, V - 1), False, 1)
    np.put_along_axis(same, np.clip(bias[0], 0, V - 1), False, 1)
    assert np.array_equal(got.float().cpu().numpy()[same], base[same])


def test_long_histories_and_bias_lists():
    """More ids than a workgroup keeps in registers and than it has threads, many of them twice."""
    from test_gpu_adjust import check as check_rules

    rng = np.random.default_rng(7)
    R, V, H, nb = 2, 6000, 5000, 3000
    x = rng.normal(0, 3, (R, V)).astype(np.float32)
    p = tm.make_params(R, repeat_penalty=1.02, repeat_last_n=4500, frequency_penalty=0.01, presence_penalty=0.2)
    recent = rng.integers(0, V, (R, H)).astype(np.int32)
    bias = (rng.integers(0, V, (R, nb)).astype(np.int32), rng.normal(0, 1, (R, nb)).astype(np.float32))
    check_rules(x, 1, p, recent, np.array([H, 3000], np.int32), None, bias, None, "f32")


def test_histories_shared_or_cut_from_wider_rows():
    """The first ids of wider rows count as a history of their own; rows that share one are refused."""
    from test_gpu_adjust import records

    x = torch.randn(3, 500, device=DEV)
    p = records(tm.make_params(3, repeat_penalty=1.5, repeat_last_n=100))
    wide = torch.randint(0, 500, (3, 40), dtype=torch.int32, device=DEV)
    a = tm.adjust_logits(x, p, recent=wide[:, :10])
    assert torch.equal(a, tm.adjust_logits(x, p, recent=wide[:, :10].contiguous()))
    with pytest.raises(ValueError):
        tm.adjust_logits(x, p, recent=wide[:1].expand(3, 40))


def test_strides_of_single_ones_do_not_matter():
    """One token, one head, one page: whatever stride their dimension has."""
    bt = Batch([9], [1], H=1, G=1, D=64, page=16, extra=0, seed=3)
    want, wl = bt.attend()
    k = bt.k.as_strided(bt.k.shape, (7, 3, 64, 1))
    v = bt.v.as_strided(bt.v.shape, (5, 1, 64, 1))
    q = bt.qs.to(DEV)
    q = q.as_strided(q.shape, (11, 13, 1))
    o, l = tm.paged_attention(q, k, v, bt.tables, bt.kv_len, bt.q_start, max_q=1, max_kv=9)
    assert torch.equal(o, want) and torch.equal(l, wl)


def test_windows_past_32_bits():
    bt = Batch([60], [3], seed=3)
    want = bt.attend()
    got = bt.attend(window=2 ** 32 + 1, sinks=2 ** 33)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
