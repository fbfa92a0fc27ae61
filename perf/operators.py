"""A decode step's work on either side of the sampler: the paged cache of keys
and values (new tokens written, attention over it, the weights each key has
drawn, eviction down to a budget), and the logits rules (mask, penalties,
biases) as an operator of their own, for the rows of a speculative verify.

A case is one call as a serving loop makes it.  Pools, page tables, lengths and
row parameters are device tensors that such a loop has in hand; ``max_q`` and
``max_kv`` are the host's own bounds on the batch.  Pages are scattered over the
pool in random order, as an allocator leaves them after some hours.  Keys of the
first tokens point the way all queries lean, so they draw weight as first tokens
do; the weight sums of an eviction are log-normal with a third of them at zero.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PARAMS = np.dtype([("temperature", "<f4"), ("top_k", "<i4"), ("top_p", "<f4"), ("min_p", "<f4"),
                   ("repeat_penalty", "<f4"), ("repeat_last_n", "<i4"), ("frequency_penalty", "<f4"),
                   ("presence_penalty", "<f4"), ("greedy", "<i4"), ("flags", "<u4"), ("seed", "<u8"),
                   ("offset", "<u8")])

# What a case may say; listed() and draw() give what differs.  kv / q: the
# longest sequence and its new tokens, kv_min / q_min the shortest's; the
# others lie evenly between.
CACHE = dict(batch=1, kv_heads=8, group=4, dim=128, page=16, dtype="bf16", kv=512, kv_min=512, q=1, q_min=1,
             window=0, sinks=0)
EVICT = dict(op="evict", batch=1, kv_heads=8, dim=128, page=16, dtype="bf16", kv=1000, kv_min=1000, budget=512,
             sinks=4, recent=64)
ADJUST = dict(op="adjust", seqs=1, steps=1, vocab=32000, dtype="f32", history=64, window=64, repeat=1.1,
              frequency=0.2, presence=0.1, biases=0, mask="none")


def listed():
    def cache(name, op, **kw):
        return dict(CACHE, op=op, name=name, **kw)

    return [
        # One token of every sequence of a decode batch into the cache.
        cache("append_token", "append", batch=64, kv=4096, kv_min=100),
        # Prompts of several requests, with odd lengths.
        cache("append_prompts", "append", batch=7, kv=2500, kv_min=700, q=2381, q_min=333, dtype="f16"),
        # One chat session's next token after a short prompt.
        cache("attend_row", "attend", kv=500, kv_min=500),
        # A decode batch: ragged lengths, one token each.
        cache("attend_decode", "attend", batch=64, kv=8192, kv_min=257),
        # A verify step, eight drafts and the token before them, over a
        # window with four sinks; the pages left behind are given back.
        cache("attend_verify", "attend", batch=32, kv=16000, kv_min=700, q=9, q_min=9, window=2048, sinks=4,
              dtype="f16"),
        # A chunk of a long prompt over what is cached of it.
        cache("attend_chunk", "attend", kv=16384, kv_min=16384, q=2048, q_min=2048, page=64),
        # The weights that a decode batch's tokens gave to the cached keys.
        cache("scores_decode", "scores", batch=32, kv=4096, kv_min=257),
        # ... and those of a prompt's chunk, with smaller odd-sized heads.
        cache("scores_chunk", "scores", batch=2, kv=6000, kv_min=4097, q=1024, q_min=777, dim=80, group=2,
              dtype="f16", page=32),
        # One session's cache cut to 512 entries.
        dict(EVICT, name="evict_row"),
        # A batch of long caches cut to a quarter.
        dict(EVICT, name="evict_batch", batch=16, kv=8192, kv_min=1500, budget=2048, recent=256),
        # One session's row: penalties and a few biases.
        dict(ADJUST, name="adjust_row", biases=8),
        # The rows of a verify step, with grammar masks.
        dict(ADJUST, name="adjust_verify", seqs=32, steps=9, vocab=128256, dtype="bf16", history=1024, window=256,
             biases=300, mask="dense"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "scores", "scores", "evict", "evict", "adjust", "adjust"])
    if op == "adjust":
        v = rng.choice([32000, 128256, 151936, 256000, _log_int(rng, 32000, 256000)]) + rng.choice([0, 0, 1, 3, -5])
        dtype, steps = rng.choice(["f32", "f16", "bf16"]), rng.choice([1, 1, rng.randint(2, 9)])
        most = max(1, min(64, 70_000_000 // (steps * v * SIZE[dtype])))
        return dict(ADJUST, seqs=_log_int(rng, 1, most), steps=steps, vocab=min(256000, v), dtype=dtype,
                    history=_log_int(rng, 64, 2048), window=_log_int(rng, 64, 1024), repeat=rng.choice([1.0, 1.05, 1.1]),
                    frequency=rng.choice([0.0, 0.2]), presence=rng.choice([0.0, 0.1]),
                    biases=rng.choice([0, 8, _log_int(rng, 1, 300)]), mask=rng.choice(["none", "dense"]))
    c = dict(kv_heads=rng.choice([1, 2, 4, 8, 8]), dim=rng.choice([64, 80, 96, 128, 128, 256]),
             page=rng.choice([16, 16, 32, 64, 128]), dtype=rng.choice(["f16", "bf16"]))
    row = 2 * c["kv_heads"] * c["dim"]   # values a token has in the cache
    if op == "evict":
        c.update(kv=_log_int(rng, 300, 16384))
        c.update(batch=_log_int(rng, 1, max(1, min(64, 250_000_000 // (row * c["kv"])))),
                 kv_min=rng.randint(100, c["kv"]), sinks=rng.choice([0, 1, 4]), recent=rng.choice([0, 16, 64, 128]))
        return dict(EVICT, **dict(c, budget=rng.randint(150, max(151, c["kv"] // 2))))
    c.update(group=rng.choice([1, 2, 3, 4, 7, 8]))
    kind = rng.choice(["token", "token", "verify", "chunk"])
    if kind == "chunk":
        c.update(kv=_log_int(rng, 100, 16384))
        c["q"] = min(c["kv"], _log_int(rng, 20, 2048))
        pairs = c["q"] * c["kv"] * c["kv_heads"] * c["group"]   # of them a pass makes 64 MB to 4 GB in 32 bits
        c["batch"] = rng.randint(1, max(1, min(8, 900_000_000 // pairs, 250_000_000 // (row * c["kv"]))))
        if pairs * c["dim"] > 80_000_000_000:   # a drawn case costs no more than the largest listed one
            c["kv_heads"], c["group"], c["dim"] = 4, 4, 80
        c["q_min"] = rng.randint(1, c["q"])
    else:
        c["q"] = 1 if kind == "token" else rng.randint(2, 17)
        c["q_min"] = rng.choice([1, c["q"]])
        c["kv"] = _log_int(rng, 40, 32768)
        c["batch"] = _log_int(rng, 1, max(1, min(64, 400_000_000 // (row * c["kv"]))))
    c["kv_min"] = rng.randint(c["q"], c["kv"])
    if rng.random() < 0.4:
        c.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 13]))
    return dict(CACHE, op=op, **c)


def _spread(lo, hi, n):
    """n whole numbers evenly from lo to hi, the largest first."""
    return [hi if b == 0 else lo + (hi - lo) * (b - 1) // (n - 1) for b in range(n)]


def _lengths(c):
    kv = _spread(c["kv_min"], c["kv"], c["batch"])
    if "q" not in c:
        return kv, [0] * c["batch"]
    return kv, [min(a, b) for a, b in zip(_spread(c["q_min"], c["q"], c["batch"]), kv)]


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    host = np.random.default_rng(seed)
    if case["op"] == "adjust":
        return _prepare_adjust(case, g, host)
    dt, ps, B, D, H = DTYPES[case["dtype"]], case["page"], case["batch"], case["dim"], case["kv_heads"]
    kv, q = _lengths(case)
    W, S = case.get("window", 0), case["sinks"]
    need = [-(-n // ps) for n in kv]
    there = max(1, -(-case["budget"] // ps)) if case["op"] == "evict" else 0
    pages = sum(need) + B * there + 3
    order = host.permutation(pages).astype(np.int32)
    tables, at = np.full((B, max(need) + 1), -1, np.int32), 0
    dst = np.full((B, max(1, there)), -1, np.int32)
    for b in range(B):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        dst[b, :there] = order[at:at + there]
        at += there
        if W:   # pages that no later token sees are given back
            first = kv[b] - q[b] - W + 1
            lo, hi = -(-S // ps), first // ps
            if hi > lo:
                tables[b, lo:hi] = -1

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    def device(a):
        return torch.from_numpy(np.asarray(a)).to(DEV)

    lean = normal(H, 1, D, dtype=torch.float32) * 0.3
    k_cache, v_cache = normal(pages, H, ps, D), normal(pages, H, ps, D)
    for b in range(B):
        n = min(4, kv[b])
        p, s = tables[b, np.arange(n) // ps], np.arange(n) % ps
        k_cache[device(p.astype(np.int64)), :, device(s)] += (8.0 * lean[:, 0]).to(dt)
    st = dict(case=case, k_cache=k_cache, v_cache=v_cache, tables=device(tables),
              kv_len=device(np.array(kv, np.int32)), max_kv=max(kv))
    scores = torch.exp(2.0 * normal(pages, H, ps, dtype=torch.float32) - 3.0)
    st["scores"] = scores * (torch.rand(pages, H, ps, generator=g, device=DEV) > 0.33)
    if case["op"] == "evict":
        st["dst_tables"] = device(dst)
        return st
    T, G = sum(q), case["group"]
    st["q_start"] = device(np.concatenate([[0], np.cumsum(q)]).astype(np.int32))
    st["max_q"] = max(q)
    if case["op"] == "append":
        st["k_new"], st["v_new"] = normal(T, H, D), normal(T, H, D)
        return st
    heads = normal(T, H, G, D, dtype=torch.float32) + lean
    st["q"] = heads.reshape(T, H * G, D).to(dt)
    if case["op"] == "scores":
        st["lse"] = _attend(st)[1]
        st["new_scores"] = torch.zeros_like(st["scores"])
    return st


def _prepare_adjust(c, g, host):
    S, n, V, H = c["seqs"], c["steps"], c["vocab"], c["history"]
    R = S * n
    words = host.zipf(1.2, (S, H + n)).clip(1, V).astype(np.int64)   # few words often, as in text
    ids = ((words * 7919) % V).astype(np.int32)
    p = np.zeros(S, PARAMS)
    p["temperature"] = 1.0
    p["repeat_penalty"], p["repeat_last_n"] = c["repeat"], c["window"]
    p["frequency_penalty"], p["presence_penalty"] = c["frequency"], c["presence"]

    def device(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    st = dict(case=c, logits=(3.0 * torch.randn(R, V, generator=g, device=DEV)).to(DTYPES[c["dtype"]]),
              params=device(p.view(np.uint8).reshape(S, PARAMS.itemsize)), recent=device(ids[:, :H]),
              n_recent=device(np.array([H - (b * 37) % (H // 2) for b in range(S)], np.int32)),
              drafts=device(ids[:, H:H + n - 1]) if n > 1 else None, bias_ids=None, bias_values=None, mask=None)
    if c["biases"]:
        st["bias_ids"] = device(np.stack([host.choice(V, c["biases"], replace=False) for _ in range(S)]).astype(np.int32))
        st["bias_values"] = device(host.uniform(-10, 10, (S, c["biases"])).astype(np.float32))
    if c["mask"] == "dense":   # about nine ids of ten allowed
        W = (V + 31) // 32
        w = torch.zeros(R, W, dtype=torch.int64, device=DEV)
        for i in range(32):
            w |= (torch.rand(R, W, generator=g, device=DEV) < 0.9).long() << i
        st["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    return st


# ---- plain forms ----------------------------------------------------------------------------------

def _slots(table, j, page):
    """Pages and slots of the positions j [..., n] of sequences with the rows `table` [..., P]."""
    return torch.gather(table, -1, (j // page).long().clamp(0, table.shape[-1] - 1)).long(), (j % page).long()


def _tokens(st, count):
    """Sequence and place in its chunk of every new token."""
    t = torch.arange(count, device=DEV, dtype=torch.int32)
    b = torch.searchsorted(st["q_start"][1:].contiguous(), t, right=True)
    return b, t - st["q_start"][b]


def _weights(st):
    """Scores [B, H, max_q * G, max_kv] in 32 bits, -inf where a key is not seen, and the pages of the keys."""
    c, q = st["case"], st["q"]
    B, H, G, D, ps = c["batch"], c["kv_heads"], c["group"], c["dim"], c["page"]
    n, L = st["max_q"], st["max_kv"]
    j = torch.arange(L, device=DEV, dtype=torch.int32).expand(B, L)
    page, slot = _slots(st["tables"], j, ps)
    keys = st["k_cache"][page.clamp(min=0), :, slot].float().permute(0, 2, 3, 1).contiguous()   # [B, H, D, L]
    r = torch.arange(n, device=DEV, dtype=torch.int32)
    rows = (st["q_start"][:-1, None] + r).clamp(max=q.shape[0] - 1).long()
    qs = q[rows].float().reshape(B, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D)
    s = torch.matmul(qs.contiguous(), keys).mul_(1.0 / math.sqrt(D))
    p = (st["kv_len"] - (st["q_start"][1:] - st["q_start"][:-1]))[:, None] + r
    seen = (j[:, None] <= p[:, :, None]) & (j < st["kv_len"][:, None])[:, None]
    if c["window"]:
        seen &= (j[:, None] > p[:, :, None] - c["window"]) | (j < c["sinks"])[:, None]
    seen &= (page >= 0)[:, None] & (r < (st["q_start"][1:] - st["q_start"][:-1])[:, None])[:, :, None]
    s.view(B, H, n, G, L).masked_fill_(~seen[:, None, :, None], float("-inf"))
    return s, page, slot


def _attend(st):
    c, q = st["case"], st["q"]
    B, H, G, D, n = c["batch"], c["kv_heads"], c["group"], c["dim"], st["max_q"]
    s, page, slot = _weights(st)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    w = s.sub_(top).exp_()
    total = w.sum(-1, keepdim=True)
    values = st["v_cache"][page.clamp(min=0), :, slot].float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(w, values) / total.clamp(min=1e-30)
    b, r = _tokens(st, q.shape[0])
    o = o.view(B, H, n, G, D)[b, :, r.long()].reshape(q.shape).to(q.dtype)
    lse = (top + total.log()).view(B, H, n, G)[b, :, r.long()].reshape(q.shape[:2])
    return o, lse


def _add_scores(st):
    c = st["case"]
    B, H, G, n, L = c["batch"], c["kv_heads"], c["group"], st["max_q"], st["max_kv"]
    s, page, slot = _weights(st)
    rows = (st["q_start"][:-1, None] + torch.arange(n, device=DEV)).clamp(max=st["q"].shape[0] - 1).long()
    lse = st["lse"][rows].view(B, n, H, G).permute(0, 2, 1, 3).reshape(B, H, n * G, 1)
    w = s.sub_(lse.clamp(min=-1e30)).exp_().sum(2)   # [B, H, L]
    new = st["new_scores"]
    held = (torch.arange(L, device=DEV) < st["kv_len"][:, None]) & (page >= 0)
    p, sl = page[held], slot[held]
    new[p, :, sl] = st["scores"][p, :, sl] + w.permute(0, 2, 1)[held]
    return new


def _append(st):
    t, ps = st["k_new"].shape[0], st["case"]["page"]
    b, r = _tokens(st, t)
    at = st["kv_len"][b] - (st["q_start"][b + 1] - st["q_start"][b]) + r
    page, slot = st["tables"][b, (at // ps).long()].long(), (at % ps).long()
    ok = page >= 0
    st["k_cache"][page[ok], :, slot[ok]] = st["k_new"][ok]
    st["v_cache"][page[ok], :, slot[ok]] = st["v_new"][ok]
    st["scores"][page[ok], :, slot[ok]] = 0.0
    return st["k_cache"], st["v_cache"], st["scores"]


def _evict(st):
    c = st["case"]
    B, H, ps, L, N = c["batch"], c["kv_heads"], c["page"], st["max_kv"], c["budget"]
    j = torch.arange(L, device=DEV, dtype=torch.int32).expand(B, L)
    page, slot = _slots(st["tables"], j, ps)
    n = st["kv_len"][:, None]
    s = st["scores"][page.clamp(min=0), :, slot].permute(0, 2, 1)   # [B, H, L]
    s = torch.where(((j < c["sinks"]) | (j >= n - c["recent"]))[:, None], float("inf"), s)
    s = torch.where((j < n)[:, None], s, float("-inf"))
    first = torch.sort(s, dim=-1, descending=True, stable=True).indices[..., :N]
    first = torch.nn.functional.pad(first, (0, max(0, N - L)), value=L)
    kept = torch.where(torch.arange(N, device=DEV) < n[:, None], first, L).sort(-1).values   # past the end: L
    ok = kept < n[:, None]
    sp, ss = _slots(st["tables"][:, None].expand(B, H, -1), kept.clamp(max=L - 1), ps)
    dp, ds = _slots(st["dst_tables"][:, None].expand(B, H, -1), torch.arange(N, device=DEV).expand(B, H, N), ps)
    h = torch.arange(H, device=DEV)[:, None].expand(B, H, N)
    to, of = (dp[ok], h[ok], ds[ok]), (sp[ok], h[ok], ss[ok])
    for pool in (st["k_cache"], st["v_cache"], st["scores"]):
        pool[to] = pool[of]
    new_len = st["kv_len"].clamp(max=N)
    return st["k_cache"], st["v_cache"], st["scores"], new_len, torch.where(ok, kept, -1).to(torch.int32)


def _adjust(st):
    c, x = st["case"], st["logits"].float()
    S, n, V, W, H = c["seqs"], c["steps"], c["vocab"], c["window"], c["history"]
    step = torch.arange(n, device=DEV)[:, None]
    have = st["n_recent"][:, None, None]
    i = torch.arange(H + n - 1, device=DEV)
    ids = st["recent"] if st["drafts"] is None else torch.cat([st["recent"], st["drafts"]], 1)
    place = torch.where(i < H, i, have + i - H)   # [S, 1, .]: where in the row's history
    used = torch.where(i < H, i < have, i - H < step) & (place >= have + step - W)
    ids = ids[:, None].expand(S, n, H + n - 1).reshape(S * n, -1).long()
    count = torch.zeros(S * n, V, dtype=torch.int32, device=DEV).scatter_add_(1, ids, used.reshape(S * n, -1).int())
    factor = torch.pow(float(np.float32(c["repeat"])), count.double())
    x = torch.where(x > 0, x / factor, x * factor)
    x = torch.where(count > 0, x - (count * float(np.float32(c["frequency"])) + float(np.float32(c["presence"]))), x)
    if st["bias_ids"] is not None:
        to = st["bias_ids"].long().repeat_interleave(n, 0)
        x = x.scatter_add_(1, to, st["bias_values"].double().repeat_interleave(n, 0))
    if st["mask"] is not None:
        bit = (st["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = x.masked_fill_(bit.view(S * n, -1)[:, :V] == 0, float("-inf"))
    return x.to(DTYPES[c["dtype"]])


PLAIN = {"append": _append, "attend": _attend, "scores": _add_scores, "evict": _evict, "adjust": _adjust}


def run(st):
    c = st["case"]
    if not own:
        return PLAIN[c["op"]](st)
    import tensormark_amd as tm

    if c["op"] == "append":
        tm.kv_append(st["k_new"], st["v_new"], st["k_cache"], st["v_cache"], st["tables"], st["kv_len"], st["q_start"],
                     max_q=st["max_q"], scores=st["scores"])
        return st["k_cache"], st["v_cache"], st["scores"]
    if c["op"] == "attend":
        return tm.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["tables"], st["kv_len"], st["q_start"],
                                  max_q=st["max_q"], max_kv=st["max_kv"], window=c["window"], sinks=c["sinks"])
    if c["op"] == "scores":
        return tm.kv_add_scores(st["q"], st["lse"], st["k_cache"], st["scores"], st["tables"], st["kv_len"],
                                st["q_start"], max_q=st["max_q"], max_kv=st["max_kv"], window=c["window"],
                                sinks=c["sinks"], out=st["new_scores"])
    if c["op"] == "evict":
        new_len, kept = tm.kv_evict(st["k_cache"], st["v_cache"], st["scores"], st["tables"], st["kv_len"],
                                    st["dst_tables"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"],
                                    max_kv=st["max_kv"])
        return st["k_cache"], st["v_cache"], st["scores"], new_len, kept
    return tm.adjust_logits(st["logits"], st["params"], recent=st["recent"], n_recent=st["n_recent"],
                            drafts=st["drafts"], steps=c["steps"], bias_ids=st["bias_ids"],
                            bias_values=st["bias_values"], mask=st["mask"])


def work(case):
    if case["op"] == "adjust":
        R, V = case["seqs"] * case["steps"], case["vocab"]
        more = case["seqs"] * (4 * min(case["window"], case["history"]) + 8 * case["biases"])
        return {"bytes": 2 * R * V * SIZE[case["dtype"]] + more + (R * 4 * ((V + 31) // 32) if case["mask"] != "none" else 0),
                "flops": R * V}
    kv, q = _lengths(case)
    H, D, e = case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in kv)
        return {"bytes": 4 * H * sum(kv) + H * kept * (4 * D * e + 8), "flops": H * sum(kv)}
    if case["op"] == "append":
        return {"bytes": sum(q) * H * (4 * D * e + 4), "flops": 0}
    G, W, S, pairs, keys = case["group"], case["window"], case["sinks"], 0, 0
    for L, n in zip(kv, q):
        if W:
            pairs += sum(min(p + 1, W + min(S, max(0, p + 1 - W))) for p in range(L - n, L))
            keys += min(L, W + n - 1 + min(S, max(0, L - n + 1 - W)))
        else:
            pairs += n * (L - n) + n * (n + 1) // 2
            keys += L
    rows = sum(q) * H * G
    if case["op"] == "scores":
        return {"bytes": rows * (D * e + 4) + keys * H * D * e + 8 * H * sum(kv), "flops": 2 * D * H * G * pairs}
    return {"bytes": rows * (2 * D * e + 4) + keys * H * 2 * D * e, "flops": 4 * D * H * G * pairs}


# ---- the definitions in 64 bits, one sequence and head at a time -------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "adjust":
        return _exact_adjust(case, st)
    kv, q = _lengths(case)
    H, ps, D = case["kv_heads"], case["page"], case["dim"]
    tables = st["tables"].cpu().numpy().astype(np.int64)
    if case["op"] == "append":
        k, v, sc = st["k_cache"].double(), st["v_cache"].double(), st["scores"].double()
        at = 0
        for b, (L, n) in enumerate(zip(kv, q)):
            pos = np.arange(L - n, L)
            page, slot = torch.from_numpy(tables[b][pos // ps]).to(DEV), torch.from_numpy(pos % ps).to(DEV)
            there = page >= 0
            page, slot = page[there], slot[there]
            k[page, :, slot] = st["k_new"][at:at + n][there].double()
            v[page, :, slot] = st["v_new"][at:at + n][there].double()
            sc[page, :, slot] = 0.0
            at += n
        return k, v, sc
    if case["op"] == "evict":
        return _exact_evict(case, st, kv, tables)
    G, W, S = case["group"], case["window"], case["sinks"]
    T = st["q"].shape[0]
    out = torch.zeros(T, H * G, D, dtype=torch.float64, device=DEV)
    lse = torch.full((T, H * G), float("-inf"), dtype=torch.float64, device=DEV)
    scores = st["new_scores"].double() if case["op"] == "scores" else None
    at = 0
    for b, (L, n) in enumerate(zip(kv, q)):
        pos = np.flatnonzero(tables[b][np.arange(L) // ps] >= 0)
        page = torch.from_numpy(tables[b][pos // ps]).to(DEV)
        slot, j = torch.from_numpy(pos % ps).to(DEV), torch.from_numpy(pos).to(DEV)
        p = torch.arange(L - n, L, device=DEV)[:, None]
        hidden = j > p
        if W:
            hidden |= (j <= p - W) & (j >= S)
        for h in range(H):
            keys, values = st["k_cache"][page, h, slot].double(), st["v_cache"][page, h, slot].double()
            if scores is not None:
                scores[page, h, slot] = st["scores"][page, h, slot].double()
            for a in range(h * G, (h + 1) * G):
                s = (st["q"][at:at + n, a].double() @ keys.t().contiguous()) / math.sqrt(D)
                s[hidden] = float("-inf")
                if scores is not None:
                    scores[page, h, slot] += (s - st["lse"][at:at + n, a, None].double().clamp(min=-1e30)).exp().sum(0)
                    continue
                lse[at:at + n, a] = torch.logsumexp(s, 1)
                out[at:at + n, a] = (s - lse[at:at + n, a, None].clamp(min=-1e300)).exp() @ values
        at += n
    return scores if case["op"] == "scores" else (out, lse)


def _exact_evict(case, st, kv, tables):
    H, ps, N = case["kv_heads"], case["page"], case["budget"]
    dst, sc = st["dst_tables"].cpu().numpy().astype(np.int64), st["scores"].cpu().numpy()
    kept = np.full((len(kv), H, N), -1, np.int32)
    pools = [st["k_cache"].double(), st["v_cache"].double(), st["scores"].double()]
    for b, L in enumerate(kv):
        pos, to = np.arange(L), np.arange(min(L, N))
        guarded = (pos < case["sinks"]) | (pos >= L - case["recent"])
        for h in range(H):
            s = sc[tables[b][pos // ps], h, pos % ps]
            rank = np.lexsort((pos, np.where(guarded, 0, -s.astype(np.float64)), ~guarded))
            keep = np.sort(rank[:N])
            kept[b, h, :len(keep)] = keep
            i = [torch.from_numpy(x).to(DEV) for x in (tables[b][keep // ps], keep % ps, dst[b][to // ps], to % ps)]
            for pool in pools:
                pool[i[2], h, i[3]] = pool[i[0], h, i[1]]
    return (*pools, torch.tensor([min(L, N) for L in kv], dtype=torch.int32, device=DEV), torch.from_numpy(kept).to(DEV))


def _exact_adjust(c, st):
    S, n, V, W = c["seqs"], c["steps"], c["vocab"], c["window"]
    x = st["logits"].double().cpu().numpy()
    recent, have = st["recent"].cpu().numpy(), st["n_recent"].cpu().numpy()
    drafts = st["drafts"].cpu().numpy() if st["drafts"] is not None else np.zeros((S, 0), np.int32)
    rep, freq, pres = (float(np.float32(c[k])) for k in ("repeat", "frequency", "presence"))
    for row in range(S * n):
        b, step = divmod(row, n)
        seen = np.concatenate([recent[b, :have[b]], drafts[b, :step]])[-W:]
        ids, times = np.unique(seen, return_counts=True)
        v = x[row, ids]
        v = np.where(v > 0, v * rep ** -times.astype(np.float64), v * rep ** times.astype(np.float64))
        x[row, ids] = v - (times * freq + pres)
        if st["bias_ids"] is not None:
            np.add.at(x[row], st["bias_ids"][b].cpu().numpy(), st["bias_values"][b].cpu().numpy().astype(np.float64))
    if st["mask"] is not None:
        bits = np.unpackbits(st["mask"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V]
        x[bits == 0] = -np.inf
    return torch.from_numpy(x)
