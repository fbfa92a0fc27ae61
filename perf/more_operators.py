"""A speculative decode step whose drafts form a tree, over the paged cache: keys
and queries turned to their rotary positions (alone, and on the way into the cache),
attention of the tree's nodes, the verify of the drafts against the target's
probabilities, and the cache cut down to the accepted path, or to other entries.

A case is one call as a serving loop makes it.  A sequence's new tokens are its
tree: node 0 is the last token that is settled, every other node a draft whose
parent has a smaller index; trees lie level by level.  Pages are scattered over the
pool in random order.  ``max_q`` and ``max_kv`` are the host's own bounds.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# What a case may say; listed() and draw() give what differs.  kv / q: the
# longest sequence and its new tokens, kv_min / q_min the shortest's; the
# others lie evenly between.  rotary: dimensions that turn; far: added to
# every position; stretch: long-context scaling of the frequencies.
ROTARY = dict(batch=1, q_heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, stretch=1.0, dtype="bf16", q=1,
              q_min=1, far=0, page=16, kv=512, kv_min=512)
TREE = dict(op="tree", batch=1, kv_heads=8, group=4, dim=128, page=16, dtype="bf16", kv=512, kv_min=512, q=8, q_min=8,
            window=0, sinks=0)
VERIFY = dict(op="verify", batch=1, vocab=32000, dtype="f32", q=8, q_min=8, drafts="given")
COMPACT = dict(op="compact", batch=1, kv_heads=8, dim=128, page=16, dtype="bf16", kv=512, kv_min=512, q=0, q_min=0,
               kept=5, kind="path")


def listed():
    return [
        # A decode batch's next tokens, deep in long contexts, into the cache.
        dict(ROTARY, name="append_rotary_token", op="append_rotary", batch=64, kv=4096, kv_min=100, far=500_000, stretch=8.0),
        # Prompts of several requests, with odd lengths; a part of each head turns.
        dict(ROTARY, name="append_rotary_prompts", op="append_rotary", batch=7, kv=2500, kv_min=700, q=2381, q_min=333,
             dtype="f16", rotary=64),
        # Queries and keys of a long prompt, without a cache, in pairs.
        dict(ROTARY, name="rotary_prompt", op="rotary", q=16385, q_min=16385, interleaved=True),
        # One chat session's eight nodes after a short prompt.
        dict(TREE, name="tree_row", kv=508, kv_min=508),
        # A decode batch: ragged lengths, trees of up to 25 nodes.
        dict(TREE, name="tree_decode", batch=32, kv=8192, kv_min=257, q=25, q_min=9),
        # Wide trees over long contexts.
        dict(TREE, name="tree_wide", batch=8, kv=16384, kv_min=9000, q=64, q_min=64, dtype="f16", page=64),
        # One session's drafts, taken from the draft model's best.
        dict(VERIFY, name="verify_row"),
        # A decode batch, drafts drawn from the draft model.
        dict(VERIFY, name="verify_drawn", batch=32, vocab=128256, q=25, q_min=9, drafts="drawn"),
        # ... and with the best taken, and probabilities in 16 bits.
        dict(VERIFY, name="verify_given", batch=64, vocab=151936, q=16, q_min=16, dtype="bf16"),
        # The accepted paths of a decode batch, moved to the front of their trees.
        dict(COMPACT, name="compact_path", batch=32, kv=8192, kv_min=257, q=25, q_min=25),
        # Long sessions cut to their first and last entries, where they lie.
        dict(COMPACT, name="compact_cut", batch=16, kv=8192, kv_min=4600, kept=2200, kind="cut"),
        # Sessions copied to pages of their own.
        dict(COMPACT, name="compact_fork", batch=8, kv=4001, kv_min=500, dtype="f16", page=32, kept=4001, kind="fork"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "append_rotary", "tree", "tree", "tree", "verify", "verify", "compact", "compact"])
    if op == "verify":
        v = rng.choice([32000, 128256, 151936, 256000, _log_int(rng, 32000, 256000)]) + rng.choice([0, 0, 1, 3, -5])
        dtype, drafts, q = rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["given", "drawn"]), _log_int(rng, 2, 64)
        rows = max(1, 100_000_000 // (v * q))   # of up to 400 MB, and as many of the draft's
        return dict(VERIFY, batch=_log_int(rng, 1, max(1, min(64, rows))), vocab=min(256000, v), dtype=dtype, q=q,
                    q_min=rng.randint(1, q), drafts=drafts)
    c = dict(kv_heads=rng.choice([1, 2, 4, 8, 8]), dim=rng.choice([64, 80, 96, 128, 128, 256]),
             page=rng.choice([16, 16, 32, 64, 128]), dtype=rng.choice(["f16", "bf16"]))
    row = 2 * c["kv_heads"] * c["dim"]   # values a token has in the cache
    if op in ("rotary", "append_rotary"):
        c["q_heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 7, 8])
        c["rotary"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, 32, 20])
        c.update(interleaved=rng.choice([False, False, True]), stretch=rng.choice([1.0, 1.0, 4.0, 8.0]),
                 far=rng.choice([0, 0, _log_int(rng, 1000, 1_000_000)]))
        most = 80_000_000 // ((c["q_heads"] + 2 * c["kv_heads"]) * c["dim"])   # new tokens in all
        if op == "rotary":
            c.update(dtype=rng.choice(["f16", "bf16", "f32"]), q=_log_int(rng, 1, min(16385, most // 2)))
            c["batch"] = _log_int(rng, 1, max(1, min(64, most // 2 // c["q"])))
        else:
            c.update(q=rng.choice([1, rng.randint(2, 64), _log_int(rng, 64, 2400)]))
            c["q"] = min(c["q"], most)
            c["batch"] = _log_int(rng, 1, max(1, min(64, most // c["q"])))
            c["kv"] = c["q"] + _log_int(rng, 1, max(2, min(4096, 250_000_000 // (row * c["batch"]))))
            c["kv_min"] = c["q"] + rng.randint(0, c["kv"] - c["q"])
        c["q_min"] = rng.randint(1, c["q"])
        return dict(ROTARY, op=op, **c)
    if op == "compact":
        kind = rng.choice(["path", "path", "cut", "fork"])
        c["kv"] = _log_int(rng, 100, 8192)
        c["batch"] = _log_int(rng, 1, max(1, min(64, 130_000_000 // (row * c["kv"]))))
        if kind == "path":
            c["q"] = rng.randint(4, 64)
            c.update(kept=rng.randint(1, max(1, min(8, c["q"] // 2))), q_min=rng.randint(c["q"] // 2, c["q"]),
                     kv_min=rng.randint(c["q"], c["kv"]))
        else:
            c["kv_min"] = rng.randint(c["kv"] // 2 + 1, c["kv"])
            c["kept"] = rng.randint(1, c["kv_min"] // 2) if kind == "cut" else rng.randint(1, c["kv"])
        return dict(COMPACT, kind=kind, **c)
    c.update(group=rng.choice([1, 2, 3, 4, 7, 8]), q=_log_int(rng, 2, 100), kv=_log_int(rng, 120, 24000))
    pairs = c["q"] * c["kv"] * c["kv_heads"] * c["group"]   # of them a pass makes up to 1 GB in 32 bits
    c["batch"] = _log_int(rng, 1, max(1, min(64, 260_000_000 // pairs, 200_000_000 // (row * c["kv"]))))
    c.update(q_min=rng.randint(1, c["q"]), kv_min=rng.randint(c["q"], c["kv"]))
    if rng.random() < 0.3:
        c.update(window=_log_int(rng, 4, 4096), sinks=rng.choice([0, 1, 4, 13]))
    return dict(TREE, **c)


def _spread(lo, hi, n):
    """n whole numbers evenly from lo to hi, the largest first."""
    return [hi if b == 0 else lo + (hi - lo) * (b - 1) // (n - 1) for b in range(n)]


def _lengths(c):
    q = _spread(c["q_min"], c["q"], c["batch"])
    if c["op"] in ("rotary", "verify"):   # (no cache)
        return q, q
    kv = _spread(c["kv_min"], c["kv"], c["batch"])
    return kv, [min(a, b) for a, b in zip(q, kv)]


def _tree(host, n):
    """Parents of n nodes, level by level: levels of up to sixteen, some nodes with several children and some with none."""
    parents, before, at = [-1], [0], 1
    while at < n:
        level = list(range(at, min(n, at + int(host.integers(1, 17)))))
        parents += sorted(host.choice(before, len(level)).tolist())
        before, at = level, level[-1] + 1
    return np.array(parents[:n], np.int32)


def _paged(c, g, host, st, kv, more=0):
    """Pools and page tables; `more` pages a sequence besides."""
    dt, ps, B, D, H = DTYPES[c["dtype"]], c["page"], c["batch"], c["dim"], c["kv_heads"]
    need = [-(-n // ps) for n in kv]
    order = host.permutation(sum(need) + B * more + 3).astype(np.int32)
    tables, at = np.full((B, max(need) + 1), -1, np.int32), 0
    dst = np.full((B, max(1, more)), -1, np.int32)
    for b in range(B):
        tables[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        dst[b, :more] = order[at:at + more]
        at += more
    if c.get("window"):   # pages that no later token sees are given back
        for b, n in enumerate(kv):
            lo, hi = -(-c["sinks"] // ps), (n - min(c["q"], n) - c["window"] + 1) // ps
            if hi > lo:
                tables[b, lo:hi] = -1
    shape = (len(order), H, ps, D)
    st["k_cache"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)
    st["v_cache"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)
    st["scores"] = torch.rand(shape[:3], generator=g, device=DEV)
    st["tables"], st["kv_len"] = torch.from_numpy(tables).to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV)
    st["dst_tables"], st["max_kv"] = torch.from_numpy(dst).to(DEV), max(kv)


def prepare(case, seed):
    c, g, host = case, torch.Generator(DEV).manual_seed(seed), np.random.default_rng(seed)
    kv, q = _lengths(c)
    T = sum(q)
    st = dict(case=c, max_q=max(q), q_start=torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device=DEV))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    if c["op"] in ("rotary", "append_rotary"):
        R, dt = c["rotary"], DTYPES[c["dtype"]]
        heads = c["q_heads"] + (2 if c["op"] == "append_rotary" else 1) * c["kv_heads"]
        st["x"] = normal(T, heads, c["dim"]).to(dt)   # as the projection leaves them, side by side
        f = 10000.0 ** (-np.arange(0, R, 2) / R)
        if c["stretch"] > 1:   # the slow ones of them slower: those with few turns in 4096 positions
            turns = 4096 * f / (2 * math.pi)
            f *= 1 / c["stretch"] + (1 - 1 / c["stretch"]) * np.clip((turns - 1) / 31, 0, 1)
        st["freqs"] = torch.from_numpy(f.astype(np.float32)).to(DEV)
        where = [np.arange(n - m, n) for n, m in zip(kv, q)] if c["op"] == "append_rotary" else [np.arange(n) for n in q]
        st["positions"] = torch.from_numpy((np.concatenate(where) + c["far"]).astype(np.int32)).to(DEV)
        if c["op"] == "append_rotary":
            _paged(c, g, host, st, kv)
        return st
    if c["op"] == "compact":
        return _prepare_compact(c, g, host, st, kv, q)
    parents = np.concatenate([_tree(host, n) for n in q])
    st["parents"] = torch.from_numpy(parents).to(DEV)
    if c["op"] == "tree":
        _paged(c, g, host, st, kv)
        st["q"] = (1.5 * normal(T, c["kv_heads"] * c["group"], c["dim"])).to(DTYPES[c["dtype"]])
        return st
    # Rows of a vocabulary with some likely words; the draft is a little off.
    V, dt = c["vocab"], DTYPES[c["dtype"]]
    up = torch.from_numpy((parents + np.repeat(np.cumsum([0] + q[:-1]), q)).clip(0)).to(DEV)   # the parents' rows
    lift = normal(V) * 3.0
    logits = normal(T, V).mul_(5.0).add_(lift)
    draft = normal(T, V).add_(logits)
    st["target"], st["draft"] = torch.softmax(logits, 1).to(dt), None
    tokens = torch.zeros(T, dtype=torch.int64, device=DEV)
    if c["drafts"] == "drawn":
        st["draft"] = torch.softmax(draft, 1).to(dt)
        for t in range(T):
            e = torch.empty(V, device=DEV).exponential_(generator=g)
            tokens[t] = (st["draft"][up[t]].float() / e).argmax()
    else:   # the best of the parent's row, its children in turn
        rank = torch.from_numpy(np.concatenate([[int((p[:i] == p[i]).sum()) for i in range(len(p))]
                                                for p in np.split(parents, np.cumsum(q)[:-1])])).to(DEV)
        tokens = torch.topk(draft, 32, 1).indices[up, rank.clamp(max=31)]
    st["tokens"] = tokens.to(torch.int32)
    st["uniforms"] = torch.rand(T, generator=g, device=DEV, dtype=torch.float64)
    return st


def _prepare_compact(c, g, host, st, kv, q):
    """Lists whose entries stay where they are or come from behind the kept ones, so that a call can be made again."""
    if c["kind"] == "path":
        n_kept = [1 + int(host.integers(0, min(c["kept"], max(1, n // 2)))) for n in q]
        lists = [np.concatenate([[0], np.sort(host.choice(np.arange(k, n), k - 1, replace=False))]) if k > 1 else np.zeros(1)
                 for k, n in zip(n_kept, q)]
    elif c["kind"] == "cut":
        n_kept = [min(c["kept"], n // 2) for n in kv]
        lists = [np.concatenate([np.arange(min(4, k)), np.arange(n - k + min(4, k), n)]) for k, n in zip(n_kept, kv)]
    else:
        n_kept = [min(c["kept"], n) for n in kv]
        lists = [np.arange(n - k, n) for k, n in zip(n_kept, kv)]
    _paged(c, g, host, st, kv, more=-(-max(n_kept) // c["page"]) if c["kind"] == "fork" else 0)
    if c["kind"] != "path":
        st["q_start"] = None
    if c["kind"] != "fork":
        st["dst_tables"] = None
    kept = np.full((c["batch"], max(n_kept)), -1, np.int32)
    for b, k in enumerate(lists):
        kept[b, :len(k)] = k
    st["kept"], st["n_kept"] = torch.from_numpy(kept).to(DEV), torch.tensor(n_kept, dtype=torch.int32, device=DEV)
    return st


# ---- plain forms ----------------------------------------------------------------------------------

def _tokens(st, count):
    """Sequence and place in its tree of every new token."""
    t = torch.arange(count, device=DEV, dtype=torch.int32)
    b = torch.searchsorted(st["q_start"][1:].contiguous(), t, right=True)
    return b, t - st["q_start"][b]


def _turn(st, x):
    c = st["case"]
    R, x = c["rotary"], x.float()
    angle = st["positions"].double()[:, None] * st["freqs"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        out[..., 0:R:2], out[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        out[..., :R // 2], out[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    return out.to(st["x"].dtype)


def _append_rotary(st):
    c, ps, Q = st["case"], st["case"]["page"], st["case"]["q_heads"]
    q, k, v = st["x"].split([Q, c["kv_heads"], c["kv_heads"]], 1)
    b, r = _tokens(st, q.shape[0])
    at = st["kv_len"][b] - (st["q_start"][b + 1] - st["q_start"][b]) + r
    page, slot = st["tables"][b, (at // ps).long()].long(), (at % ps).long()
    ok = page >= 0
    turned = _turn(st, st["x"][:, :Q + c["kv_heads"]])
    st["k_cache"][page[ok], :, slot[ok]] = turned[:, Q:][ok]
    st["v_cache"][page[ok], :, slot[ok]] = v[ok]
    st["scores"][page[ok], :, slot[ok]] = 0.0
    return turned[:, :Q].contiguous(), st["k_cache"], st["v_cache"], st["scores"]


def _rotary(st):
    return _turn(st, st["x"])


def _seen(st):
    """[B, max_q, max_q] truth of which nodes a node sees without a window, itself among them, and the nodes' depths."""
    c, n = st["case"], st["max_q"]
    r = torch.arange(n, device=DEV, dtype=torch.int32)
    rows = (st["q_start"][:-1, None] + r).clamp(max=st["q"].shape[0] - 1).long()
    there = r < (st["q_start"][1:] - st["q_start"][:-1])[:, None]
    parents = torch.where(there, st["parents"][rows], -1)
    seen = torch.eye(n, dtype=torch.bool, device=DEV).repeat(c["batch"], 1, 1)
    at = r.expand(c["batch"], n)
    depth = torch.zeros_like(at)
    for _ in range(n - 1):
        at = torch.where(at >= 0, torch.gather(parents, 1, at.clamp(min=0).long()), -1)
        depth = depth + (at >= 0)
        seen |= (at[:, :, None] == r) & (at >= 0)[:, :, None]
    return seen, depth, rows, there


def _attend(st):
    c, q = st["case"], st["q"]
    B, H, G, D, ps = c["batch"], c["kv_heads"], c["group"], c["dim"], c["page"]
    n, L = st["max_q"], st["max_kv"]
    tree, depth, rows, there = _seen(st)
    j = torch.arange(L, device=DEV, dtype=torch.int32).expand(B, L)
    page, slot = torch.gather(st["tables"], 1, (j // ps).long()).long(), (j % ps).long()
    keys = st["k_cache"][page.clamp(min=0), :, slot].float().permute(0, 2, 3, 1).contiguous()
    qs = q[rows].float().reshape(B, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D)
    s = torch.matmul(qs.contiguous(), keys).mul_(1.0 / math.sqrt(D))
    p0 = (st["kv_len"] - (st["q_start"][1:] - st["q_start"][:-1]))[:, None]
    node = (j - p0).clamp(0, n - 1).long()
    prefix = (j < p0)[:, None]
    there = there[:, :, None]
    seen = (prefix | torch.gather(tree, 2, node[:, None].expand(B, n, L))) & (j < st["kv_len"][:, None])[:, None]
    if c["window"]:
        at = torch.where(j < p0, j, p0 + torch.gather(depth, 1, node))[:, None]   # the keys' positions
        seen &= (at > (p0 + depth)[:, :, None] - c["window"]) | (at < c["sinks"])
    seen &= (page >= 0)[:, None] & there
    s.view(B, H, n, G, L).masked_fill_(~seen[:, None, :, None], float("-inf"))
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


def _verify(st):
    """The walk as one pass over the nodes of all sequences, since a child comes after its parent; sums in 64 bits."""
    c, n, T = st["case"], st["max_q"], st["tokens"].shape[0]
    B, V = c["batch"], c["vocab"]
    first = st["q_start"][:-1].long()
    count = (st["q_start"][1:] - st["q_start"][:-1]).long()
    row = torch.arange(B, device=DEV)
    cur = torch.zeros(B, dtype=torch.int64, device=DEV)
    path = torch.full((B, n), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    kept = torch.ones(B, dtype=torch.int64, device=DEV)
    left, total = st["target"][first].double(), torch.ones(B, dtype=torch.float64, device=DEV)
    for j in range(1, n):
        t = (first + j).clamp(max=T - 1)
        x = st["tokens"][t].long()
        tested = (j < count) & (st["parents"][t] == cur)
        draft = st["draft"][first + cur].double() if st["draft"] is not None else None
        have = left[row, x]
        chance = draft[row, x] if draft is not None else torch.ones_like(have)
        taken = tested & (st["uniforms"][t] * chance * total < have)
        refused = tested & ~taken
        if draft is not None:
            less = (left - total[:, None] * draft).clamp_(min=0.0)
            left = torch.where(refused[:, None], less, left)
            total = torch.where(refused, left.sum(1), total)
        else:
            left[row, x] = torch.where(refused, 0.0, have)
            total = torch.where(refused, total - have, total)
        left = torch.where(taken[:, None], st["target"][t].double(), left)
        total = torch.where(taken, 1.0, total)
        path[row, kept.clamp(max=n - 1)] = torch.where(taken, j, path[row, kept.clamp(max=n - 1)])
        kept = kept + taken
        cur = torch.where(taken, j, cur)
    upto = left.cumsum(1)
    some = upto[:, -1] > 0   # else the drafts took all there was
    upto = torch.where(some[:, None], upto, st["target"][first + cur].double().cumsum(1))
    token = torch.searchsorted(upto, (st["uniforms"][first] * upto[:, -1])[:, None], right=True)[:, 0].clamp(max=V - 1)
    return path, kept.to(torch.int32), token.to(torch.int32)


def _compact(st):
    c, ps = st["case"], st["case"]["page"]
    base = torch.zeros_like(st["kv_len"])
    if st["q_start"] is not None:
        base = st["kv_len"] - (st["q_start"][1:] - st["q_start"][:-1])
    i = torch.arange(st["kept"].shape[1], device=DEV, dtype=torch.int32)
    ok = i < st["n_kept"][:, None]
    src, dst = base[:, None] + st["kept"].clamp(min=0), base[:, None] + i
    to = st["tables"] if st["dst_tables"] is None else st["dst_tables"]

    def slots(table, j):
        return torch.gather(table, 1, (j // ps).long().clamp(max=table.shape[1] - 1)).long()[ok], (j % ps).long()[ok]

    (sp, ss), (dp, ds) = slots(st["tables"], src), slots(to, dst)
    for pool in (st["k_cache"], st["v_cache"], st["scores"]):
        pool[dp, :, ds] = pool[sp, :, ss]
    return st["k_cache"], st["v_cache"], st["scores"], base + st["n_kept"]


PLAIN = {"rotary": _rotary, "append_rotary": _append_rotary, "tree": _attend, "verify": _verify, "compact": _compact}


def run(st):
    c = st["case"]
    if not own:
        return PLAIN[c["op"]](st)
    import tensormark_amd as tm

    if c["op"] == "rotary":
        return tm.rotary(st["x"], st["positions"], st["freqs"], interleaved=c["interleaved"])
    if c["op"] == "append_rotary":
        q, k, v = st["x"].split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
        q = tm.kv_append_rotary(q, k, v, st["k_cache"], st["v_cache"], st["tables"], st["kv_len"], st["q_start"],
                                st["positions"], st["freqs"], max_q=st["max_q"], interleaved=c["interleaved"],
                                scores=st["scores"])
        return q, st["k_cache"], st["v_cache"], st["scores"]
    if c["op"] == "tree":
        return tm.tree_attention(st["q"], st["k_cache"], st["v_cache"], st["tables"], st["kv_len"], st["q_start"],
                                 st["parents"], max_q=st["max_q"], max_kv=st["max_kv"], window=c["window"], sinks=c["sinks"])
    if c["op"] == "verify":
        return tm.verify_tree(st["target"], st["tokens"], st["parents"], st["q_start"], st["uniforms"], max_q=st["max_q"],
                              draft=st["draft"])
    new_len = tm.kv_compact(st["k_cache"], st["v_cache"], st["tables"], st["kv_len"], st["kept"], st["n_kept"],
                            q_start=st["q_start"], dst_tables=st["dst_tables"], scores=st["scores"])
    return st["k_cache"], st["v_cache"], st["scores"], new_len


def work(case):
    kv, q = _lengths(case)
    e, T = SIZE[case["dtype"]], sum(q)
    if case["op"] in ("rotary", "append_rotary"):
        turned, D = case["q_heads"] + case["kv_heads"], case["dim"]
        more = case["kv_heads"] if case["op"] == "append_rotary" else 0
        return {"bytes": T * ((turned + more) * 2 * D * e + 4 + 4 * more), "flops": T * turned * case["rotary"] * 3}
    if case["op"] == "verify":
        # The row that the last draw is from, the draft's where one may have been refused, some numbers a node.
        rows = case["batch"] * (2 if case["drafts"] == "drawn" else 1)
        return {"bytes": rows * case["vocab"] * e + T * (16 + 2 * e), "flops": 2 * rows * case["vocab"]}
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "compact":
        most = {"path": lambda n, m: min(case["kept"], m) / 2, "cut": lambda n, m: min(case["kept"], n // 2),
                "fork": lambda n, m: min(case["kept"], n)}[case["kind"]]
        moved = sum(most(n, m) for n, m in zip(kv, q))
        return {"bytes": int(moved * (H * (4 * D * e + 8) + 4)) + 8 * case["batch"], "flops": 0}
    G, W, S, pairs, keys = case["group"], case["window"], case["sinks"], 0, 0
    for L, n in zip(kv, q):
        seen = L - n if not W else min(L - n, W + S)
        pairs += n * (seen + 2)   # (and a few nodes of the tree)
        keys += seen + n
    rows = T * H * G
    return {"bytes": rows * (2 * D * e + 4) + keys * H * 2 * D * e, "flops": 4 * D * H * G * pairs}


# ---- the definitions in 64 bits, one sequence at a time ----------------------------------------------

def exact(case, seed):
    st, (kv, q) = prepare(case, seed), _lengths(case)
    return {"rotary": _exact_rotary, "append_rotary": _exact_rotary, "tree": _exact_tree, "verify": _exact_verify,
            "compact": _exact_compact}[case["op"]](case, st, kv, q)


def _exact_rotary(c, st, kv, q):
    R, Q, H = c["rotary"], c["q_heads"], c["kv_heads"]
    x = st["x"].double()
    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(st["positions"].double(), st["freqs"].double()))
    half = x[:, :Q + H, :R]
    pairs = half.reshape(*half.shape[:2], R // 2, 2) if c["interleaved"] else half.reshape(*half.shape[:2], 2, R // 2).transpose(2, 3)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z[:, None])
    x[:, :Q + H, :R] = (turned if c["interleaved"] else turned.transpose(2, 3)).reshape(half.shape)
    if c["op"] == "rotary":
        return x
    k, v, sc = st["k_cache"].double(), st["v_cache"].double(), st["scores"].double()
    tables, at = st["tables"].cpu().numpy().astype(np.int64), 0
    for b, (L, n) in enumerate(zip(kv, q)):
        pos = np.arange(L - n, L)
        page, slot = torch.from_numpy(tables[b][pos // c["page"]]).to(DEV), torch.from_numpy(pos % c["page"]).to(DEV)
        k[page, :, slot] = x[at:at + n, Q:Q + H]
        v[page, :, slot] = x[at:at + n, Q + H:]
        sc[page, :, slot] = 0.0
        at += n
    return x[:, :Q], k, v, sc


def _exact_tree(c, st, kv, q):
    H, G, D, ps, W, S = c["kv_heads"], c["group"], c["dim"], c["page"], c["window"], c["sinks"]
    T = st["q"].shape[0]
    out = torch.zeros(T, H * G, D, dtype=torch.float64, device=DEV)
    lse = torch.full((T, H * G), float("-inf"), dtype=torch.float64, device=DEV)
    tables, parents, at = st["tables"].cpu().numpy().astype(np.int64), st["parents"].cpu().numpy(), 0
    for b, (L, n) in enumerate(zip(kv, q)):
        hidden = np.ones((n, L), bool)
        for t in range(n):
            line, a = [], t
            while a >= 0:
                line.append(a)
                a = parents[at + a]
            place = L - n + len(line) - 1   # the node's position; the next of its line is one before
            hidden[t, :L - n] = False
            if W:
                hidden[t, max(0, S):max(0, S, min(L - n, place - W + 1))] = True
            for back, a in enumerate(line):
                hidden[t, L - n + a] = W > 0 and back >= W and place - back >= S
        pos = np.flatnonzero(tables[b][np.arange(L) // ps] >= 0)
        page, slot = torch.from_numpy(tables[b][pos // ps]).to(DEV), torch.from_numpy(pos % ps).to(DEV)
        gone = torch.from_numpy(hidden[:, pos]).to(DEV)
        for h in range(H):
            keys, values = st["k_cache"][page, h, slot].double(), st["v_cache"][page, h, slot].double()
            for a in range(h * G, (h + 1) * G):
                s = (st["q"][at:at + n, a].double() @ keys.t().contiguous()) / math.sqrt(D)
                s[gone] = float("-inf")
                lse[at:at + n, a] = torch.logsumexp(s, 1)
                out[at:at + n, a] = (s - lse[at:at + n, a, None].clamp(min=-1e300)).exp() @ values
        at += n
    return out, lse


def _exact_verify(c, st, kv, q):
    tokens, parents, u = (st[k].cpu().numpy() for k in ("tokens", "parents", "uniforms"))
    path = np.full((len(q), max(q)), -1, np.int32)
    kept, out, at = np.zeros(len(q), np.int32), np.zeros(len(q), np.int32), 0
    for b, n in enumerate(q):
        node, line = 0, [0]
        while True:
            p = st["target"][at + node].double().cpu().numpy()
            d = st["draft"][at + node].double().cpu().numpy() if st["draft"] is not None else None
            r, chance, found = p.copy(), 1.0, False
            for j in range(n):
                if parents[at + j] != node:
                    continue
                x = tokens[at + j]
                if u[at + j] * (1.0 if d is None else d[x]) * chance < r[x]:
                    node, found = j, True
                    line.append(j)
                    break
                if d is None:
                    chance -= r[x]
                    r[x] = 0.0
                else:
                    r = np.maximum(r - chance * d, 0.0)
                    chance = math.fsum(r)
            if not found:
                break
        r = r if r.any() else p
        out[b] = np.flatnonzero(np.cumsum(r) > u[at] * np.cumsum(r)[-1])[0]
        path[b, :len(line)], kept[b] = line, len(line)
        at += n
    return tuple(torch.from_numpy(x).to(DEV) for x in (path, kept, out))


def _exact_compact(c, st, kv, q):
    ps, tables = c["page"], st["tables"].cpu().numpy().astype(np.int64)
    to = tables if st["dst_tables"] is None else st["dst_tables"].cpu().numpy().astype(np.int64)
    kept, n_kept = st["kept"].cpu().numpy(), st["n_kept"].cpu().numpy()
    pools = [st["k_cache"].double(), st["v_cache"].double(), st["scores"].double()]
    base = [L - n if st["q_start"] is not None else 0 for L, n in zip(kv, q)]
    for b in range(len(kv)):
        a, z = base[b] + kept[b, :n_kept[b]], base[b] + np.arange(n_kept[b])
        i = [torch.from_numpy(x).to(DEV) for x in (tables[b][a // ps], a % ps, to[b][z // ps], z % ps)]
        for pool in pools:
            pool[i[2], :, i[3]] = pool[i[0], :, i[1]].clone()
    return (*pools, torch.tensor([x + int(y) for x, y in zip(base, n_kept)], dtype=torch.int32, device=DEV))
