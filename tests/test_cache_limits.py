"""Limits of the cache operators that their header names, refused before any device work."""
from __future__ import annotations

import ctypes as C

import pytest

from tensormark_amd import cache
from test_cache_args import CAPACITY, INVALID, P, a_cache, rows_args


def attend(c=None, a=None):
    lib = cache._fns()
    c, a = a_cache(**(c or {})), rows_args(cache.AttentionArgs, **(a or {}))
    need = lib.tms_paged_attention_workspace(C.byref(c), C.byref(a))
    got = lib.tms_paged_attention(C.byref(c), C.byref(a), None)
    assert need == got
    return got


def scores(c=None, a=None):
    c, a = a_cache(**(c or {})), rows_args(cache.ScoreArgs, **(a or {}))
    return cache._fns().tms_kv_add_scores(C.byref(c), C.byref(a), None)


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_a_scale_that_is_no_number(scale):
    assert attend(a=dict(scale=scale)) == INVALID
    assert scores(a=dict(scale=scale)) == INVALID


def test_slots_too_far_apart():
    for s in ("k_stride", "v_stride"):
        assert attend(c={s: (2, 1 << 26)}) == CAPACITY


def test_too_many_rows():
    assert attend(c=dict(tokens=1 << 21, max_q=1 << 21)) == CAPACITY
    assert scores(c=dict(tokens=1 << 21, max_q=1 << 21)) == CAPACITY


def test_too_many_sequences_and_heads():
    assert attend(c=dict(batch=1 << 20)) == CAPACITY


def test_queries_too_far_apart_for_scores():
    assert scores(a=dict(q_stride=(0, (1 << 23) + 8))) == CAPACITY
    assert scores(a=dict(q_stride=(1, 1 << 23))) == CAPACITY


def test_histories_of_logits():
    lib = cache._fns()
    for kw, code in ((dict(n_history=9, recent_stride=8), INVALID), (dict(n_history=-1), INVALID), (dict(reserved=1), INVALID),
                     (dict(n_history=1 << 29, recent_stride=1 << 29), CAPACITY)):
        a = rows_args(cache.AdjustArgs, out=P + 4096, **kw)
        assert lib.tms_adjust_logits(C.byref(a), None) == code


def test_a_workspace_for_every_form():
    """None for whole items, some for shares and for splits; never less for more."""
    lib = cache._fns()
    need = []
    for kv in (100, 1024, 5000, 50000, 500000):
        c, a = a_cache(max_kv=kv, table_stride=40000), rows_args(cache.AttentionArgs)
        need.append(lib.tms_paged_attention_workspace(C.byref(c), C.byref(a)))
    assert need[0] == need[1] == 0 and need[2] > 0 and need == sorted(need)
    c = a_cache(max_kv=50000, table_stride=40000, tokens=90, max_q=30)
    assert lib.tms_paged_attention_workspace(C.byref(c), C.byref(rows_args(cache.AttentionArgs))) > 0


def test_more_items_than_32_bits_count():
    """Strides past the chunk kernel's offsets, and so many sequences and rows that tiles of
    32 rows are past 2^31: refused; the same with ordinary strides is not."""
    def call(batch, heads, far):
        c = a_cache(batch=batch, kv_heads=heads, tokens=1 << 20, max_q=1 << 20, page_size=65536)
        for s in (c.k_stride, c.v_stride):
            s[0], s[1], s[2] = 0, 0, 1 << 25 if far else 64
        return cache._fns().tms_paged_attention_workspace(C.byref(c), C.byref(rows_args(cache.AttentionArgs, q_heads=2 * heads)))

    assert call(1 << 15, 1, True) == CAPACITY and call(1 << 14, 2, True) == CAPACITY
    assert call((1 << 15) - 1, 1, True) > 0 and call(1 << 15, 1, False) >= 0


def test_the_limits_that_the_header_names():
    import os
    import re

    from test_cache_args import ROOT

    with open(os.path.join(ROOT, "include", "tmcache_hip.h")) as f:
        most = {k: int(v) for k, v in re.findall(r"#define (TMS_\w+_MAX_\w+) (\d+)", f.read())}
    lib, n = cache._fns(), most["TMS_APPEND_MAX_BATCH"]
    append = C.byref(rows_args(cache.AppendArgs))
    assert lib.tms_kv_append(C.byref(a_cache(batch=n + 1, kv_heads=1)), append, None) == CAPACITY
    assert lib.tms_kv_append(C.byref(a_cache(batch=n, kv_heads=1, tokens=0)), append, None) == 0
    assert scores(c=dict(max_kv=most["TMS_SCORES_MAX_KV"] + 1)) == CAPACITY
    assert attend(c=dict(batch=most["TMS_CACHE_MAX_PAIRS"] // 2 + 1)) == CAPACITY
    assert attend(c=dict(tokens=most["TMS_CACHE_MAX_TOKENS"] + 1)) == CAPACITY
    evict = C.byref(rows_args(cache.EvictArgs))
    assert lib.tms_kv_evict(C.byref(a_cache(max_kv=most["TMS_EVICT_MAX_KV"] + 1)), evict, None) == CAPACITY
