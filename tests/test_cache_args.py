"""What the cache operators and adjust_logits refuse, and their structs'
layouts, without a GPU: every refusal comes before any device work."""
from __future__ import annotations

import ctypes as C
import os
import shutil
import subprocess

import pytest
import torch

import tensormark_amd as tm
from tensormark_amd import cache

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x1000   # an aligned address that no refused call reads
INVALID, CAPACITY = -1, -2


def a_cache(**kw):
    c = cache.CacheArgs()
    c.k = c.v = c.scores = c.tables = c.kv_len = c.q_start = P
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = 16 * 64 * 2, 16 * 64, 64
    c.dtype, c.pages, c.kv_heads, c.page_size, c.head_dim, c.batch = 2, 10, 2, 16, 64, 3
    c.table_stride, c.tokens, c.max_q, c.max_kv = 4, 3, 1, 64
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(c, k)[v[0]] = v[1]
        else:
            setattr(c, k, v)
    return c


def rows_args(cls, **kw):
    a = cls()
    for name in ("q", "out", "lse", "k_new", "v_new", "dst_tables", "new_len", "kept", "logits"):
        if hasattr(a, name):
            setattr(a, name, P)
    for name in ("q_stride", "out_stride", "k_new_stride", "v_new_stride"):
        if hasattr(a, name) and not isinstance(getattr(a, name), int):
            getattr(a, name)[0], getattr(a, name)[1] = 256, 64
    if hasattr(a, "q_heads"):
        a.q_heads, a.scale = 4, 0.125
    if cls is cache.EvictArgs:
        a.dst_table_stride, a.budget, a.sinks, a.recent = 2, 32, 4, 8
    if cls is cache.AdjustArgs:
        a.seqs, a.steps, a.vocab, a.row_stride, a.out_stride = 2, 3, 100, 100, 100
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


BAD_CACHE = [
    dict(k=None), dict(k=P + 8), dict(dtype=0), dict(dtype=7), dict(pages=0), dict(kv_heads=0), dict(page_size=4),
    dict(page_size=24), dict(page_size=131072), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(batch=-1),
    dict(tables=None), dict(table_stride=0), dict(kv_len=None), dict(k_stride=(2, 63)), dict(k_stride=(0, -8)),
    dict(tokens=-1), dict(max_q=-1), dict(max_kv=-1), dict(reserved=1), dict(scores=P + 4),
]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_every_call_refuses_a_bad_cache(bad):
    lib = cache._fns()
    c = C.byref(a_cache(**bad))
    assert lib.tms_kv_append(c, C.byref(rows_args(cache.AppendArgs)), None) == INVALID
    att = rows_args(cache.AttentionArgs)
    assert lib.tms_paged_attention_workspace(c, C.byref(att)) == INVALID
    assert lib.tms_paged_attention(c, C.byref(att), None) == INVALID
    assert lib.tms_kv_add_scores(c, C.byref(rows_args(cache.ScoreArgs)), None) == INVALID
    assert lib.tms_kv_evict(c, C.byref(rows_args(cache.EvictArgs)), None) == INVALID


def test_null_structs_are_refused():
    lib = cache._fns()
    c = C.byref(a_cache())
    for f in (lib.tms_kv_append, lib.tms_paged_attention, lib.tms_kv_add_scores, lib.tms_kv_evict):
        assert f(None, None, None) == INVALID
        assert f(c, None, None) == INVALID
    assert lib.tms_paged_attention_workspace(None, None) == INVALID
    assert lib.tms_adjust_logits(None, None) == INVALID


@pytest.mark.parametrize("call, kw, code", [
    ("attend", dict(q=None), INVALID), ("attend", dict(q=P + 2), INVALID), ("attend", dict(out=None), INVALID),
    ("attend", dict(q_heads=0), INVALID), ("attend", dict(q_heads=3), INVALID), ("attend", dict(sinks=-1), INVALID),
    ("attend", dict(scale=float("nan")), INVALID), ("attend", dict(q_stride=(0, 4)), INVALID),
    ("attend", dict(out_stride=(1, -64)), INVALID),
    ("scores", dict(lse=None), INVALID), ("scores", dict(q=None), INVALID), ("scores", dict(q_heads=5), INVALID),
    ("scores", dict(out=P + 4), INVALID), ("scores", dict(sinks=-2), INVALID),
    ("append", dict(k_new=None), INVALID), ("append", dict(v_new=P + 4), INVALID), ("append", dict(k_new_stride=(0, 12)), INVALID),
    ("evict", dict(budget=0), INVALID), ("evict", dict(sinks=30), INVALID), ("evict", dict(recent=-1), INVALID),
    ("evict", dict(kept=None), INVALID), ("evict", dict(new_len=None), INVALID), ("evict", dict(dst_table_stride=1), INVALID),
    ("evict", dict(dst_tables=None), INVALID), ("evict", dict(reserved=1), INVALID),
    ("adjust", dict(logits=None), INVALID), ("adjust", dict(out=None), INVALID), ("adjust", dict(dtype=3), INVALID),
    ("adjust", dict(dtype=1, out_dtype=2), INVALID), ("adjust", dict(steps=0), INVALID), ("adjust", dict(vocab=0), INVALID),
    ("adjust", dict(row_stride=99), INVALID), ("adjust", dict(n_bias=1), INVALID), ("adjust", dict(mask=P, mask_stride=3), INVALID),
    ("adjust", dict(vocab=2000000, row_stride=2000000, out_stride=2000000), CAPACITY), ("adjust", dict(seqs=40000), CAPACITY),
    ("adjust", dict(logits=P, out=P, out_stride=101), INVALID), ("adjust", dict(out=P + 2), INVALID),
])
def test_bad_arguments_are_refused(call, kw, code):
    lib = cache._fns()
    cls = {"attend": cache.AttentionArgs, "scores": cache.ScoreArgs, "append": cache.AppendArgs, "evict": cache.EvictArgs,
           "adjust": cache.AdjustArgs}[call]
    a = rows_args(cls, **(dict(out=P + 4096) if call == "adjust" else {}))
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    c = C.byref(a_cache())
    if call == "adjust":
        got = lib.tms_adjust_logits(C.byref(a), None)
    else:
        got = {"attend": lib.tms_paged_attention, "scores": lib.tms_kv_add_scores, "append": lib.tms_kv_append,
               "evict": lib.tms_kv_evict}[call](c, C.byref(a), None)
    assert got == code


def test_a_workspace_that_is_too_small_is_refused():
    lib = cache._fns()
    c, a = a_cache(max_kv=100000, table_stride=6250), rows_args(cache.AttentionArgs)
    need = lib.tms_paged_attention_workspace(C.byref(c), C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.tms_paged_attention(C.byref(c), C.byref(a), None) == INVALID
    a.workspace, a.workspace_bytes = None, need
    assert lib.tms_paged_attention(C.byref(c), C.byref(a), None) == INVALID


def test_python_calls_refuse_host_tensors_and_wrong_shapes():
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    t, n, s = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for bad in (k, k.float(), k[0], torch.zeros(4, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)):
        with pytest.raises(ValueError):
            tm.paged_attention(q, bad, bad, t, n, s, max_q=1, max_kv=1)
    with pytest.raises(ValueError):
        tm.adjust_logits(torch.zeros(2, 10))
    with pytest.raises(ValueError):
        tm.kv_add_scores(q, torch.zeros(1, 4), k, None, t, n, s, max_q=1, max_kv=1)


def test_ctypes_layouts_match_the_c_header(tmp_path):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no gcc")
    structs = {"tms_cache": cache.CacheArgs, "tms_append_args": cache.AppendArgs, "tms_attention_args": cache.AttentionArgs,
               "tms_score_args": cache.ScoreArgs, "tms_evict_args": cache.EvictArgs, "tms_adjust_args": cache.AdjustArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tmcache_hip.h"', "int main(void) {"]
    for st, cls in structs.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{f} %zu\\n", offsetof({st}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", "/opt/rocm/include",
                    str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout
    got = dict(x.split() for x in out.splitlines())
    for st, cls in structs.items():
        assert int(got[st]) == C.sizeof(cls), st
        for f, _ in cls._fields_:
            assert int(got[f"{st}.{f}"]) == getattr(cls, f).offset, (st, f)
