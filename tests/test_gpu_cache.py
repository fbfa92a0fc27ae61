"""The paged cache operators against plain implementations in 64 bits.

Tolerances are bounds, derived per element: a weight is off by the scores' error
(a dot product of D terms in fp32, and the exponential), is rounded once to the
cache's type (half a step, eps / 2), and the output once more."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tensormark_amd as tm

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16
U = 2.0 ** -24


class Batch:
    """Sequences with scattered pages; garbage (NaN) in every slot that holds no position."""

    def __init__(self, kv, q, *, H=2, G=2, D=64, page=16, dt=BF, seed=0, extra=2, slot_major=False, peak=1.0):
        rng = np.random.default_rng(seed)
        self.kv, self.q, self.H, self.G, self.D, self.page, self.dt = kv, q, H, G, D, page, dt
        B, need = len(kv), [-(-n // page) for n in kv]
        pages = sum(need) + extra
        order = rng.permutation(pages)
        self.host = np.full((B, max(need + [1]) + 1), -1, np.int32)
        at = 0
        for b in range(B):
            self.host[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        shape = (pages, page, H, D) if slot_major else (pages, H, page, D)
        self.k = torch.full(shape, float("nan"), dtype=dt, device=DEV)
        self.v = torch.full(shape, float("nan"), dtype=dt, device=DEV)
        if slot_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.scores = torch.full((pages, H, page), float("nan"), device=DEV)
        self.keys, self.values, self.sums = [], [], []
        for b in range(B):
            kk = torch.from_numpy(rng.normal(0, 1, (kv[b], H, D))).to(dt)
            vv = torch.from_numpy(rng.normal(0, 1, (kv[b], H, D))).to(dt)
            ss = torch.from_numpy(rng.exponential(1.0, (kv[b], H)).astype(np.float32))
            self.keys.append(kk)
            self.values.append(vv)
            self.sums.append(ss)
        self.tables = torch.from_numpy(self.host).to(DEV)
        self.fill()
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device=DEV)
        self.starts = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        self.q_start = torch.from_numpy(self.starts).to(DEV)
        self.qs = (peak * torch.from_numpy(rng.normal(0, 1, (sum(q), H * G, D)))).to(dt)
        self.max_q, self.max_kv = max(q + [0]), max(kv + [0])

    def where(self, b, pos):
        pos = np.asarray(pos)
        return (torch.from_numpy(self.host[b][pos // self.page].astype(np.int64)).to(DEV),
                torch.from_numpy(pos % self.page).to(DEV))

    def fill(self):
        for b, n in enumerate(self.kv):
            if n:
                p, s = self.where(b, np.arange(n))
                self.k[p, :, s] = self.keys[b].to(DEV)
                self.v[p, :, s] = self.values[b].to(DEV)
                self.scores[p, :, s] = self.sums[b].to(DEV)

    def seen(self, b, window, sinks):
        """[q, kv] truth of which key each new token sees."""
        n, L = self.q[b], self.kv[b]
        p, j = np.arange(L - n, L)[:, None], np.arange(L)[None]
        ok = j <= p
        if window:
            ok &= (j > p - window) | (j < sinks)
        page = self.host[b][np.arange(L) // self.page] if L else np.zeros(0, np.int32)
        return ok & ((page >= 0) & (page < self.k.shape[0]))[None]

    def reference(self, window=0, sinks=0, scale=None):
        """Per sequence and head: out, lse, bounds of their errors, weights [rows, kv] (fp64)."""
        scale = 1 / math.sqrt(self.D) if scale is None else scale
        T, HQ = self.qs.shape[:2]
        out, tol = np.zeros((T, HQ, self.D)), np.zeros((T, HQ, self.D))
        lse, ltol = np.full((T, HQ), -np.inf), np.zeros((T, HQ))
        eps = torch.finfo(self.dt).eps / 2
        weights, wtol = [], []
        for b in range(len(self.kv)):
            L, n, at = self.kv[b], self.q[b], self.starts[b]
            seen = self.seen(b, window, sinks)
            for h in range(self.H):
                kk = np.nan_to_num(self.keys[b][:, h].double().numpy(), nan=0, posinf=0, neginf=0)
                vv = self.values[b][:, h].double().numpy()
                total, ttol = np.zeros(L), np.zeros(L)
                for a in range(h * self.G, (h + 1) * self.G):
                    qq = self.qs[at:at + n, a].double().numpy()
                    s = np.where(seen, scale * (qq @ kk.T), -np.inf)
                    # fp32: D products and sums, the scaling and the base-2 argument
                    serr = (self.D + 8) * U * abs(scale) * (np.abs(qq) @ np.abs(kk).T) + 8 * U * np.abs(np.where(seen, s, 0))
                    for i in range(n):
                        ok = seen[i]
                        if not ok.any():
                            continue
                        top = s[i][ok].max()
                        e = np.exp(s[i][ok] - top)
                        l = e.sum()
                        err = 2 * serr[i][ok].max() + (ok.sum() + 16) * U + 8 * U * abs(top)
                        w = e / l
                        lse[at + i, a] = top + math.log(l)
                        ltol[at + i, a] = err + 8 * U * abs(lse[at + i, a])
                        out[at + i, a] = w @ vv[ok]
                        size = w @ np.abs(vv[ok])
                        tol[at + i, a] = (eps + 2 * err) * size + eps * np.abs(out[at + i, a]) + 1e-30
                        if self.dt == HF:   # weights and outputs below the smallest normal number
                            tol[at + i, a] += 2.0 ** -25 * (np.abs(vv[ok]).sum(0) + 1)
                        total[ok] += w
                        ttol[ok] += w * 3 * err + 2.0 ** -126
                weights.append(total)
                wtol.append(ttol + (n * self.G + 4) * U * total)
        return out, lse, tol, ltol, weights, wtol

    def attend(self, q=None, **kw):
        return tm.paged_attention(self.qs.to(DEV) if q is None else q, self.k, self.v, self.tables, self.kv_len, self.q_start,
                                  max_q=self.max_q, max_kv=self.max_kv, **kw)


def check(bt, window=0, sinks=0, scale=None, got=None):
    out, lse, tol, ltol, _, _ = bt.reference(window, sinks, scale)
    o, l = got or bt.attend(window=window, sinks=sinks, scale=scale)
    o, l = o.double().cpu().numpy(), l.double().cpu().numpy()
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(l), empty)
    assert np.all(o[empty] == 0)
    assert np.all(np.abs(l[~empty] - lse[~empty]) <= ltol[~empty])
    bad = np.abs(o - out) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], o[bad][:4], out[bad][:4], tol[bad][:4])


SHAPES = [   # kv, q, H, G, D, page
    ([1], [1], 1, 1, 64, 16),
    ([17, 1, 500], [1, 1, 1], 8, 4, 128, 16),
    ([31, 32, 33, 127, 128, 129], [1] * 6, 2, 3, 128, 16),
    ([5, 0, 40, 9], [5, 0, 0, 12], 2, 2, 64, 8),           # no tokens, no keys, tokens before position 0
    ([700, 300], [9, 9], 2, 4, 128, 16),                   # drafts
    ([100, 77], [17, 8], 1, 7, 80, 32),
    ([260, 64], [64, 64], 2, 2, 96, 64),
    ([64], [33], 4, 1, 8, 8),
    ([90, 200], [1, 3], 2, 8, 256, 16),
    ([150], [40], 1, 2, 192, 128),
    ([333, 1000, 5], [333, 129, 5], 2, 2, 128, 16),        # prompts
    ([400], [200], 1, 4, 72, 16),
    ([300], [300], 1, 8, 64, 16),
    ([270], [150], 1, 3, 256, 32),
    ([4500], [1], 1, 16, 128, 16),
    ([2100], [2], 1, 32, 64, 64),                          # 64 rows of one key head
]


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("kv, q, H, G, D, page", SHAPES)
def test_attention(kv, q, H, G, D, page, dt):
    check(Batch(kv, q, H=H, G=G, D=D, page=page, dt=dt, seed=len(kv) + D))


@pytest.mark.parametrize("window, sinks", [(1, 0), (5, 0), (16, 4), (33, 13), (64, 1), (100, 40), (1000, 4), (7, 1000),
                                           (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("kv, q, G, D", [([260, 31, 900, 1], [1, 1, 1, 1], 4, 128), ([300, 64, 20], [9, 9, 9], 2, 64),
                                         ([700, 333], [333, 200], 2, 128)])
def test_attention_window_and_sinks(kv, q, G, D, window, sinks):
    check(Batch(kv, q, G=G, D=D, seed=window % 1000 + D), window, sinks)


@pytest.mark.parametrize("q", [[3, 1], [150, 90]])
def test_attention_strides_and_scale(q):
    """Slots before heads in the pool, queries cut out of a wider tensor, an
    output with gaps, another scale."""
    bt = Batch([200, 90], q, H=2, G=3, D=64, slot_major=True, dt=HF, seed=5)
    T = sum(q)
    wide = torch.randn(T, 6 + 4, 72, device=DEV).to(HF)
    wide[:, 2:8, :64] = bt.qs.to(DEV)
    gaps = torch.zeros(T, 6, 128, dtype=HF, device=DEV)
    o, l = bt.attend(q=wide[:, 2:8, :64], scale=0.31, out=gaps[:, :, :64])
    assert not gaps[:, :, 64:].any()
    check(bt, scale=0.31, got=(o, l))


@pytest.mark.parametrize("q", [[1, 2], [160, 2]])
def test_attention_unmapped_pages(q):
    """Entries outside the pool hide their positions; a row left with none gives zero."""
    bt = Batch([260, 45], q, page=16, seed=3)
    bt.host[0, [0, 3, 15]] = [-1, 10 ** 6, -(2 ** 31)]
    bt.host[1, :] = -7
    bt.tables = torch.from_numpy(bt.host).to(DEV)
    check(bt)
    check(bt, 20, 4)


@pytest.mark.parametrize("q", [9, 200])
@pytest.mark.parametrize("what", [float("inf"), float("nan")])
def test_attention_masked_keys_reach_no_row(q, what):
    """Infinities and NaN at positions that a row does not see: later tokens'
    keys and values, and values and keys behind the window."""
    L = 320
    bt = Batch([L], [q], H=1, G=2, D=128, dt=BF, seed=9)
    p, s = bt.where(0, [L - 1, L - 2])
    bt.v[p, :, s] = what
    bt.k[p, :, s] = what
    out, lse, tol, ltol, _, _ = bt.reference()
    o, l = bt.attend()
    o, l = o.double().cpu().numpy(), l.double().cpu().numpy()
    n = q - 2
    assert np.all(np.abs(o[:n] - out[:n]) <= tol[:n]) and np.all(np.abs(l[:n] - lse[:n]) <= ltol[:n])
    bt.fill()
    p, s = bt.where(0, np.arange(10, 30))
    bt.v[p, :, s] = what
    bt.k[p, :, s] = what
    W = 64
    out, lse, tol, ltol, _, _ = bt.reference(W, 4)
    o, l = bt.attend(window=W, sinks=4)
    o, l = o.double().cpu().numpy(), l.double().cpu().numpy()
    rows = np.arange(L - q, L) >= 30 + W - 1
    assert rows.any()
    assert np.all(np.abs(o[rows] - out[rows]) <= tol[rows]) and np.all(np.abs(l[rows] - lse[rows]) <= ltol[rows])


@pytest.mark.parametrize("q", [1, 200])
def test_attention_large_scores(q):
    """Scores of some hundreds: one key takes nearly all."""
    check(Batch([700], [q], H=1, G=2, D=128, peak=40.0, seed=2))


def test_attention_many_splits_and_bounds():
    """A long sequence in many shares, and a host bound below its length."""
    bt = Batch([9000, 300], [1, 1], H=1, G=4, D=64, seed=4)
    check(bt)
    bt.max_kv = 100
    check(bt)


def test_attention_offsets_past_32_bits():
    """A pool of 5 GiB a side; the sequence's pages lie at both ends."""
    pages, H, page, D = 20500, 8, 128, 128
    k = torch.empty(pages, H, page, D, dtype=BF, device=DEV)
    v = torch.empty_like(k)
    bt = Batch([300], [2], H=H, G=1, D=D, page=page, seed=6, extra=0)
    to = [pages - 1, 1, pages - 2]
    for i, p in enumerate(to):
        src = int(bt.host[0, i])
        k[p], v[p] = bt.k[src], bt.v[src]
    bt.k, bt.v = k, v
    bt.host[0, :3] = to
    bt.tables = torch.from_numpy(bt.host).to(DEV)
    check(bt)
    new = torch.randn(2, H, D, device=DEV).to(BF)
    tm.kv_append(new, new, k, v, bt.tables, bt.kv_len, bt.q_start, max_q=2)
    assert torch.equal(k[pages - 2, :, 300 - 2 - 256], new[0]) and torch.equal(v[pages - 2, :, 300 - 1 - 256], new[1])


@pytest.mark.parametrize("kv, q", [([900, 70], [1, 1]), ([300, 260], [200, 260])])
def test_attention_repeats_and_streams(kv, q):
    """The same bits on every call, on another stream, and from a graph's replays."""
    bt = Batch(kv, q, H=2, G=4, D=128, seed=8)
    qd = bt.qs.to(DEV)
    o, l = bt.attend(q=qd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o2, l2 = bt.attend(q=qd)
    side.synchronize()
    assert torch.equal(o, o2) and torch.equal(l, l2)
    out, lse = torch.zeros_like(o), torch.zeros_like(l)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        bt.attend(q=qd, out=out, lse=lse)
        tm.kv_add_scores(qd, lse, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q, max_kv=bt.max_kv)
    for i in range(3):
        bt.fill()
        qd.copy_(bt.qs.to(DEV).roll(i, 0))
        g.replay()
        torch.cuda.synchronize()
        after = bt.scores.clone()
        want, wl = bt.attend(q=qd)
        assert torch.equal(out, want) and torch.equal(lse, wl)
        bt.fill()
        again = tm.kv_add_scores(qd, lse, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q, max_kv=bt.max_kv)
        assert torch.equal(torch.nan_to_num(again, nan=-1.0), torch.nan_to_num(after, nan=-1.0))


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("kv, q, H, G, D, page", SHAPES)
@pytest.mark.parametrize("window, sinks", [(0, 0), (40, 4)])
def test_scores(kv, q, H, G, D, page, window, sinks, dt):
    bt = Batch(kv, q, H=H, G=G, D=D, page=page, dt=dt, seed=len(kv) + D + 1)
    _, lse, _, ltol, weights, wtol = bt.reference(window, sinks)
    l32 = torch.from_numpy(lse).to(DEV, torch.float32)
    before = bt.scores.clone()
    out = torch.full_like(before, 7.0)
    got = tm.kv_add_scores(bt.qs.to(DEV), l32, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q,
                           max_kv=bt.max_kv, window=window, sinks=sinks, out=out)
    assert got is out
    touched = torch.zeros_like(out, dtype=torch.bool)
    for b, n in enumerate(kv):
        if not n:
            continue
        p, s = bt.where(b, np.arange(n))
        touched[p, :, s] = True
        new = out[p, :, s].double().cpu().numpy()
        for h in range(H):
            want = bt.sums[b][:, h].double().numpy() + weights[b * H + h]
            # the given lse is rounded too: half a step of it
            slack = wtol[b * H + h] + weights[b * H + h] * U * 2 * np.nanmax(np.abs(np.where(np.isinf(lse), 0, lse)), initial=0)
            assert np.all(np.abs(new[:, h] - want) <= slack + 2 * U * np.abs(want))
    assert torch.all(out[~touched] == 7.0)
    tm.kv_add_scores(bt.qs.to(DEV), l32, bt.k, bt.scores, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q,
                     max_kv=bt.max_kv, window=window, sinks=sinks)
    assert torch.equal(bt.scores[touched], out[touched])
    assert torch.isnan(bt.scores[~touched]).all()


def test_scores_unmapped_pages_and_lse_of_attention():
    bt = Batch([150], [3], page=16, seed=12)
    bt.host[0, 2] = -1
    bt.tables = torch.from_numpy(bt.host).to(DEV)
    o, l = bt.attend()
    out = torch.zeros_like(bt.scores)
    tm.kv_add_scores(bt.qs.to(DEV), l, bt.k, torch.zeros_like(bt.scores), bt.tables, bt.kv_len, bt.q_start, max_q=3,
                     max_kv=150, out=out)
    # every row's weights sum to one: (kv + rows + 32) steps of fp32
    per_head = out.double().sum((0, 2)).cpu().numpy()
    assert np.all(np.abs(per_head - 3 * bt.G) <= 3 * bt.G * 400 * U)


@pytest.mark.parametrize("dt", [BF, HF], ids=["bf16", "f16"])
@pytest.mark.parametrize("kv, q, D, page, slot_major", [
    ([1], [1], 64, 16, False), ([30, 5, 0, 9], [1, 5, 0, 1], 8, 8, False), ([300, 64], [299, 33], 128, 16, True),
    ([20, 7], [20, 9], 80, 32, False), ([1000, 3], [0, 3], 256, 128, False)])
def test_append(kv, q, D, page, slot_major, dt):
    bt = Batch(kv, q, H=3, D=D, page=page, dt=dt, slot_major=slot_major, seed=1)
    if len(kv) > 1:   # a token of the last sequence on a page that is not there
        bt.host[-1, (kv[-1] - 1) // page] = -1
        bt.tables = torch.from_numpy(bt.host).to(DEV)
    T = sum(q)
    wide = torch.randn(T, 6, D + 8, device=DEV).to(dt)
    kn, vn = wide[:, :3, :D], wide[:, 3:, 8:]
    wk, wv, ws = bt.k.clone(), bt.v.clone(), bt.scores.clone()
    for b, (L, n) in enumerate(zip(kv, q)):
        for i in range(n):
            j, t = L - n + i, bt.starts[b] + i
            if j >= 0 and bt.host[b, j // page] >= 0:
                p = int(bt.host[b, j // page])
                wk[p, :, j % page], wv[p, :, j % page], ws[p, :, j % page] = kn[t], vn[t], 0
    tm.kv_append(kn, vn, bt.k, bt.v, bt.tables, bt.kv_len, bt.q_start, max_q=bt.max_q, scores=bt.scores)
    for got, want in ((bt.k, wk), (bt.v, wv)):
        assert torch.equal(got.contiguous().view(torch.int16), want.contiguous().view(torch.int16))
    assert torch.equal(bt.scores.view(torch.int32), ws.view(torch.int32))


def evicted(bt, budget, sinks, recent):
    """Kept positions [B][H] by the definition."""
    kept = []
    for b, L in enumerate(bt.kv):
        row = []
        for h in range(bt.H):
            if L <= budget:
                row.append(np.arange(L))
                continue
            mapped = bt.host[b][np.arange(L) // bt.page] >= 0
            s = bt.sums[b][:, h].double().numpy()
            rank = [(-2, j) if j < sinks or j >= L - recent else
                    (1, 0.0, j) if not mapped[j] or math.isnan(s[j]) else (0, -s[j], j) for j in range(L)]
            row.append(np.array(sorted(sorted(range(L), key=lambda j: rank[j])[:budget])))
        kept.append(row)
    return kept


@pytest.mark.parametrize("kv, budget, sinks, recent, D, page, slot_major", [
    ([1], 1, 0, 0, 64, 16, False), ([1, 0, 5], 4, 1, 1, 64, 16, False), ([100, 33, 32], 32, 4, 8, 128, 16, False),
    ([1000, 300], 77, 13, 20, 80, 32, True), ([500], 24, 4, 20, 64, 8, False), ([600], 200, 0, 0, 256, 16, False),
    ([5000, 4096], 1000, 4, 64, 64, 64, False), ([20000], 1500, 4, 300, 8, 16, False)])
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
def test_evict(kv, budget, sinks, recent, D, page, slot_major, values):
    bt = Batch(kv, [0] * len(kv), H=2, D=D, page=page, slot_major=slot_major, seed=budget, extra=2 + len(kv) * (-(-budget // page)))
    rng = np.random.default_rng(budget)
    for b, L in enumerate(kv):
        if values == "ties":
            bt.sums[b] = torch.from_numpy(rng.integers(0, 3, (L, 2)).astype(np.float32) * 0.5)
        elif values == "odd" and L:
            pool = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1.5, 2.0, 2.0000002], np.float32)
            bt.sums[b] = torch.from_numpy(rng.choice(pool, (L, 2)))
    bt.fill()
    used = set(bt.host[bt.host >= 0].tolist())
    free = [p for p in range(bt.k.shape[0]) if p not in used]
    each = -(-budget // page)
    dst = np.array([free[b * each:(b + 1) * each] for b in range(len(kv))], np.int32)
    if values == "odd" and kv[0] > 2 * page:
        bt.host[0, 1] = -1
        bt.tables = torch.from_numpy(bt.host).to(DEV)
    want = evicted(bt, budget, sinks, recent)
    wk, wv, ws = bt.k.clone(), bt.v.clone(), bt.scores.clone()
    for b in range(len(kv)):
        for h in range(2):
            for i, j in enumerate(want[b][h]):
                if bt.host[b, j // page] < 0:
                    continue
                sp, ss, dp, ds = int(bt.host[b, j // page]), int(j % page), int(dst[b, i // page]), i % page
                wk[dp, h, ds], wv[dp, h, ds], ws[dp, h, ds] = bt.k[sp, h, ss], bt.v[sp, h, ss], bt.scores[sp, h, ss]
            if len(want[b][h]) > 400:   # (the longest ones' positions say enough)
                break
    long = max(len(w) for r in want for w in r) > 400
    new_len, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, torch.from_numpy(dst).to(DEV), budget=budget,
                                max_kv=bt.max_kv, sinks=sinks, recent=recent)
    assert new_len.tolist() == [min(L, budget) for L in kv]
    kept = kept.cpu().numpy()
    for b in range(len(kv)):
        for h in range(2):
            n = len(want[b][h])
            assert np.array_equal(kept[b, h, :n], want[b][h]) and np.all(kept[b, h, n:] == -1)
    heads = slice(0, 1) if long else slice(0, 2)
    for got, w in ((bt.k, wk), (bt.v, wv)):
        assert torch.equal(got[:, heads].contiguous().view(torch.int16), w[:, heads].contiguous().view(torch.int16))
    assert torch.equal(bt.scores[:, heads].contiguous().view(torch.int32), ws[:, heads].contiguous().view(torch.int32))


def test_evict_in_place_length_and_bad_destinations():
    """new_len may be kv_len; entries for pages outside the pool are not copied."""
    bt = Batch([300, 200], [0, 0], H=4, D=64, seed=3, extra=8)
    used = set(bt.host[bt.host >= 0].tolist())
    free = [p for p in range(bt.k.shape[0]) if p not in used]
    dst = np.array([free[:4], [free[4], 10 ** 7, -3, free[5]]], np.int32)
    want = evicted(bt, 64, 4, 8)
    k0 = bt.k.clone()
    new_len, kept = tm.kv_evict(bt.k, bt.v, bt.scores, bt.tables, bt.kv_len, torch.from_numpy(dst).to(DEV), budget=64,
                                max_kv=300, sinks=4, recent=8, new_len=bt.kv_len)
    assert bt.kv_len.tolist() == [64, 64]
    assert np.array_equal(kept.cpu().numpy(), np.array(want))
    for b in range(2):
        for i in range(64):
            p = dst[b, i // 16]
            if 0 <= p < bt.k.shape[0]:
                j = want[b][1][i]
                assert torch.equal(bt.k[int(p), 1, i % 16], k0[int(bt.host[b, j // 16]), 1, int(j % 16)])
    old = sorted(used)
    assert torch.equal(bt.k[old].view(torch.int16), k0[old].view(torch.int16))
