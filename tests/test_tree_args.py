"""What the tree calls refuse, their structs' layouts and limits, and the rotary
frequencies, without a GPU: every refusal comes before any device work."""
from __future__ import annotations

import ctypes as C
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

import tensormark_amd as tm
from tensormark_amd import cache, tree
from test_cache_args import BAD_CACHE, CAPACITY, INVALID, P, ROOT, a_cache, rows_args


def filled(cls, kw):
    a = cls()
    if cls is tree.RotaryArgs:
        a.x = a.out = a.positions = a.freqs = P
        a.dtype, a.tokens, a.heads, a.head_dim, a.rotary_dim, a.scale = 0, 5, 3, 64, 32, 1.0
        a.x_stride[:], a.out_stride[:] = [192, 64], [192, 64]
    if cls is tree.AppendRotaryArgs:
        a.k_new = a.v_new = a.q = a.out = a.positions = a.freqs = P
        a.q_heads, a.rotary_dim, a.scale = 4, 64, 1.0
        for s in (a.k_new_stride, a.v_new_stride, a.q_stride, a.out_stride):
            s[:] = [256, 64]
    if cls is tree.VerifyTreeArgs:
        a.target = a.draft = a.draft_tokens = a.parents = a.q_start = a.uniforms = a.path = a.kept = a.token = a.workspace = P
        a.target_stride = a.draft_stride = a.vocab = 1000
        a.batch, a.tokens, a.max_q, a.workspace_bytes = 2, 6, 3, 1 << 40
    if cls is tree.CompactArgs:
        a.kept = a.n_kept = P
        a.new_len = P + 4096
        a.kept_stride, a.max_kept = 8, 8
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


def call(cls, kw=None, c=None):
    lib, a, c = tree._fns(), filled(cls, kw or {}), C.byref(a_cache(**{"v": P + (1 << 20), **(c or {})}))
    if cls is tree.RotaryArgs:
        return lib.tms_rotary(C.byref(a), None)
    if cls is tree.AppendRotaryArgs:
        return lib.tms_kv_append_rotary(c, C.byref(a), None)
    if cls is tree.CompactArgs:
        return lib.tms_kv_compact(c, C.byref(a), None)
    need = lib.tms_verify_tree_workspace(C.byref(a))
    got = lib.tms_verify_tree(C.byref(a), None)
    assert need == got or need >= 0
    return got


def attend(c=None, parents=P, **kw):
    lib, c, a = tree._fns(), C.byref(a_cache(**(c or {}))), rows_args(cache.AttentionArgs, **kw)
    need = lib.tms_tree_attention_workspace(c, C.byref(a))
    got = lib.tms_tree_attention(c, C.byref(a), parents, None)
    assert need == got or (need >= 0 and got == INVALID)
    return got


@pytest.mark.parametrize("bad", BAD_CACHE, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
def test_every_call_refuses_a_bad_cache(bad):
    assert call(tree.AppendRotaryArgs, c=bad) == INVALID
    assert call(tree.CompactArgs, c=bad) == INVALID
    assert attend(c=bad) == INVALID


def test_null_structs_are_refused():
    lib, c = tree._fns(), C.byref(a_cache())
    assert lib.tms_rotary(None, None) == INVALID
    assert lib.tms_verify_tree(None, None) == INVALID and lib.tms_verify_tree_workspace(None) == INVALID
    for f in (lib.tms_kv_append_rotary, lib.tms_kv_compact):
        assert f(None, None, None) == INVALID and f(c, None, None) == INVALID
    assert lib.tms_tree_attention(c, None, P, None) == INVALID
    assert lib.tms_tree_attention_workspace(None, None) == INVALID


ROT = [dict(x=None), dict(out=None), dict(x=P + 8), dict(out=P + 4), dict(positions=None), dict(positions=P + 2), dict(freqs=None),
       dict(dtype=3), dict(tokens=-1), dict(heads=-1), dict(head_dim=0), dict(head_dim=60), dict(rotary_dim=0), dict(rotary_dim=31),
       dict(rotary_dim=66), dict(interleaved=2), dict(interleaved=-1), dict(scale=math.inf), dict(scale=math.nan), dict(reserved=1),
       dict(x_stride=(0, 12)), dict(out_stride=(1, -64))]
APP = [dict(k_new=None), dict(v_new=P + 4), dict(q=None), dict(out=None), dict(q=P + 2), dict(freqs=None), dict(freqs=P + 1),
       dict(positions=P + 2), dict(q_heads=-1), dict(rotary_dim=0), dict(rotary_dim=33), dict(rotary_dim=66), dict(interleaved=3),
       dict(scale=math.nan), dict(k_new_stride=(0, 12)), dict(v_new_stride=(1, -8)), dict(q_stride=(0, 4)), dict(out_stride=(1, 7))]
VER = [dict(target=None), dict(target=P + 2), dict(draft=P + 1), dict(target_stride=999), dict(draft_stride=10), dict(dtype=9), dict(vocab=0),
       dict(batch=-1), dict(tokens=-1), dict(max_q=-1), dict(reserved=1), dict(draft_tokens=None), dict(parents=None), dict(q_start=None),
       dict(uniforms=None), dict(uniforms=P + 4), dict(path=None), dict(kept=None), dict(token=None)]
COM = [dict(kept=None), dict(n_kept=None), dict(kept_stride=7), dict(max_kept=-1), dict(reserved=1), dict(dst_tables=P + 64, dst_table_stride=0), dict(dst_tables=P, dst_table_stride=4),
       dict(new_len=P), dict(new_len=P, n_kept=P + 64)]   # (kv_len and kept are at P)


@pytest.mark.parametrize("cls, kw", [(c, kw) for c, many in ((tree.RotaryArgs, ROT), (tree.AppendRotaryArgs, APP), (tree.VerifyTreeArgs, VER),
                                                            (tree.CompactArgs, COM)) for kw in many])
def test_bad_arguments_are_refused(cls, kw):
    assert call(cls, kw) == INVALID


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=P + 2), dict(q_heads=0), dict(q_heads=3), dict(sinks=-1), dict(scale=math.inf),
                                dict(q_stride=(0, 4)), dict(parents=None), dict(parents=P + 2)])
def test_bad_attention_arguments_are_refused(kw):
    assert attend(**kw) == INVALID


def test_limits():
    with open(os.path.join(ROOT, "include", "tmtree_hip.h")) as f:
        most = {k: int(v) for k, v in re.findall(r"#define (TMS_\w+) (\d+)", f.read())}
    n = most["TMS_TREE_MAX_NODES"]
    assert attend(c=dict(tokens=n + 1, max_q=n + 1)) == CAPACITY
    assert call(tree.VerifyTreeArgs, dict(max_q=n + 1)) == CAPACITY
    v = most["TMS_VERIFY_MAX_VOCAB"] + 1
    assert call(tree.VerifyTreeArgs, dict(vocab=v, target_stride=v, draft_stride=v)) == CAPACITY
    assert call(tree.VerifyTreeArgs, dict(batch=most["TMS_VERIFY_MAX_BATCH"] + 1)) == CAPACITY
    assert call(tree.RotaryArgs, dict(heads=most["TMS_ROTARY_MAX_HEADS"] + 1)) == CAPACITY
    assert call(tree.RotaryArgs, dict(head_dim=most["TMS_ROTARY_MAX_HEAD_DIM"] + 8)) == CAPACITY
    assert call(tree.RotaryArgs, dict(tokens=(1 << 28) + 1)) == CAPACITY
    assert call(tree.AppendRotaryArgs, dict(q_heads=most["TMS_ROTARY_MAX_HEADS"])) == CAPACITY
    assert call(tree.AppendRotaryArgs, c=dict(batch=65536, kv_heads=1)) == CAPACITY
    k = most["TMS_COMPACT_MAX_KEPT"] + 1
    assert call(tree.CompactArgs, dict(max_kept=k, kept_stride=k)) == CAPACITY


def test_nothing_to_do_is_no_error():
    assert call(tree.RotaryArgs, dict(tokens=0, x=None, out=None)) == 0
    assert call(tree.RotaryArgs, dict(heads=0)) == 0
    assert call(tree.AppendRotaryArgs, c=dict(tokens=0)) == 0
    assert call(tree.AppendRotaryArgs, c=dict(batch=0)) == 0
    assert call(tree.VerifyTreeArgs, dict(batch=0)) == 0
    assert call(tree.CompactArgs, c=dict(batch=0)) == 0
    assert attend(c=dict(max_q=0)) == 0


def test_a_workspace_that_is_too_small_is_refused():
    lib = tree._fns()
    a = filled(tree.VerifyTreeArgs, dict(vocab=100000, target_stride=100000, draft_stride=100000))
    need = lib.tms_verify_tree_workspace(C.byref(a))
    assert need > 0
    for workspace, n in ((P, need - 1), (None, need), (P + 8, need)):
        a.workspace, a.workspace_bytes = workspace, n
        assert lib.tms_verify_tree(C.byref(a), None) == INVALID
    c, a = a_cache(max_kv=100000, table_stride=6250), rows_args(cache.AttentionArgs)
    need = lib.tms_tree_attention_workspace(C.byref(c), C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = P, need - 1
    assert lib.tms_tree_attention(C.byref(c), C.byref(a), P, None) == INVALID


def test_workspaces_do_not_shrink():
    """With more positions, sequences or nodes a call needs as much workspace or more."""
    lib = tree._fns()

    def need(kv, batch, q):
        c = a_cache(max_kv=kv, table_stride=40000, batch=batch, tokens=q * batch, max_q=q)
        return lib.tms_tree_attention_workspace(C.byref(c), C.byref(rows_args(cache.AttentionArgs)))

    for q in (3, 40, 64, 200):
        for batch in (1, 2, 16, 200, 2000):
            sizes = [need(kv, batch, q) for kv in (1, 100, 512, 1000, 1024, 2000, 3000, 10000, 200000)]
            assert sizes == sorted(sizes) and sizes[0] == 0 and sizes[-1] > 0, (q, batch, sizes)
    for q in (3, 40, 64, 200):
        for kv in (100, 800, 1500, 3000, 50000):
            sizes = [need(kv, batch, q) for batch in (1, 2, 16, 100, 200, 2000)]
            assert sizes == sorted(sizes), (q, kv, sizes)


def test_more_threads_than_a_launch_has():
    def call_(batch):
        c = a_cache(batch=batch, kv_heads=1, tokens=512 * 2, max_q=512)
        return tree._fns().tms_tree_attention_workspace(C.byref(c), C.byref(rows_args(cache.AttentionArgs, q_heads=4096)))

    assert call_(1 << 17) == CAPACITY and call_(1 << 9) == CAPACITY and call_((1 << 9) - 1) >= 0
    assert call(tree.RotaryArgs, dict(tokens=1 << 28, heads=64)) == CAPACITY
    assert call(tree.AppendRotaryArgs, dict(q_heads=65000), dict(tokens=1 << 20, max_q=1 << 20)) == CAPACITY


def test_one_pool_for_keys_and_values_is_refused():
    """Its entries would be moved, or keys and values written, twice at once."""
    assert call(tree.AppendRotaryArgs, c=dict(v=P)) == INVALID
    assert call(tree.CompactArgs, c=dict(v=P)) == INVALID
    assert call(tree.AppendRotaryArgs, c=dict(v=P, tokens=0)) == 0


def test_an_output_that_is_the_input_has_its_strides():
    assert call(tree.RotaryArgs, dict(x_stride=(0, 256))) == INVALID
    assert call(tree.RotaryArgs, dict(out_stride=(1, 128))) == INVALID
    assert call(tree.AppendRotaryArgs, dict(q_stride=(0, 512))) == INVALID


def test_ctypes_layouts_match_the_c_header(tmp_path):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no gcc")
    structs = {"tms_rotary_args": tree.RotaryArgs, "tms_append_rotary_args": tree.AppendRotaryArgs,
               "tms_verify_tree_args": tree.VerifyTreeArgs, "tms_compact_args": tree.CompactArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tmtree_hip.h"', "int main(void) {"]
    for st, cls in structs.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{f} %zu\\n", offsetof({st}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([cc, "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", "/opt/rocm/include",
                    str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())
    for st, cls in structs.items():
        assert int(got[st]) == C.sizeof(cls), st
        for f, _ in cls._fields_:
            assert int(got[f"{st}.{f}"]) == getattr(cls, f).offset, (st, f)


def some(device="cpu"):
    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=device)

    x = dict(k=zeros(4, 2, 16, 64), v=zeros(4, 2, 16, 64), scores=zeros(4, 2, 16, dtype=torch.float32), q=zeros(2, 4, 64),
             kn=zeros(2, 2, 64), vn=zeros(2, 2, 64), lse=zeros(2, 4, dtype=torch.float32), out=zeros(2, 4, 64),
             freqs=zeros(32, dtype=torch.float32), target=zeros(2, 100, dtype=torch.float32) + 1, draft=zeros(2, 100, dtype=torch.float32) + 1,
             u=zeros(2, dtype=torch.float64), x=zeros(2, 3, 64))
    ints = dict(tables=[[0, 1]], kv_len=[20], q_start=[0, 2], parents=[-1, 0], positions=[3, 4], ids=[1, 2], new_len=[0], kept=[[0]],
                n_kept=[1], path=[[0, 0]], n_path=[0], token=[0])
    x.update({n: torch.tensor(v, dtype=torch.int32, device=device) for n, v in ints.items()})
    return x


def calls(x):
    where = (x["tables"], x["kv_len"], x["q_start"])
    return dict(
        rotary=lambda: tm.rotary(x["x"], x["positions"], x["freqs"], out=x["x"]),
        append=lambda: tm.kv_append_rotary(x["q"], x["kn"], x["vn"], x["k"], x["v"], *where, x["positions"], x["freqs"], max_q=2,
                                           scores=x["scores"], out=x["out"]),
        attend=lambda: tm.tree_attention(x["q"], x["k"], x["v"], *where, x["parents"], max_q=2, max_kv=20, out=x["out"], lse=x["lse"]),
        verify=lambda: tm.verify_tree(x["target"], x["ids"], x["parents"], x["q_start"], x["u"], max_q=2, draft=x["draft"], path=x["path"],
                                      kept=x["n_path"], token=x["token"]),
        compact=lambda: tm.kv_compact(x["k"], x["v"], x["tables"], x["kv_len"], x["kept"], x["n_kept"], q_start=x["q_start"],
                                      scores=x["scores"], new_len=x["new_len"]))


TAKES = dict(rotary=("x", "freqs"), append=("q", "kn", "vn", "k", "v", "scores", "out", "freqs"), attend=("q", "k", "v", "out", "lse"),
             verify=("target", "draft", "u"), compact=("k", "v", "scores"))


@pytest.mark.parametrize("call, name", [(c, n) for c, names in TAKES.items() for n in names])
def test_a_tensor_that_requires_a_gradient_is_refused(call, name):
    x = some()
    x[name].requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        calls(x)[call]()
    with torch.no_grad(), pytest.raises(ValueError) as e:   # (a host tensor is refused all the same)
        calls(x)[call]()
    assert "gradient" not in str(e.value)


@pytest.mark.gpu
def test_what_a_call_writes_counts_as_written():
    writes = dict(rotary=("x",), append=("k", "v", "scores", "out"), attend=("out", "lse"), verify=("path", "n_path", "token"),
                  compact=("k", "v", "scores", "new_len"))
    for call, names in writes.items():
        x = some("cuda:0")
        before = {n: t._version for n, t in x.items()}
        calls(x)[call]()
        assert {n for n, t in x.items() if t._version != before[n]} == set(names), call


@pytest.mark.gpu
def test_python_calls_refuse_what_does_not_fit():
    for call, change in [("rotary", dict(positions=torch.zeros(3, dtype=torch.int32, device="cuda:0"))),
                         ("rotary", dict(x=torch.zeros(2, 64, 3, dtype=torch.bfloat16, device="cuda:0").transpose(1, 2))),
                         ("rotary", dict(x=torch.zeros(2, 3, 64, dtype=torch.float64, device="cuda:0"))),
                         ("append", dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda:0"))),
                         ("append", dict(freqs=torch.zeros(32, dtype=torch.float64, device="cuda:0"))),
                         ("append", dict(positions=torch.zeros(2, dtype=torch.int64, device="cuda:0"))),
                         ("append", dict(out=torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda:0")[:, :, ::2])),
                         ("attend", dict(parents=torch.zeros(3, dtype=torch.int32, device="cuda:0"))),
                         ("attend", dict(parents=torch.zeros(2, dtype=torch.int32))),
                         ("verify", dict(draft=torch.zeros(2, 99, device="cuda:0"))),
                         ("verify", dict(u=torch.zeros(2, device="cuda:0"))),
                         ("verify", dict(ids=torch.zeros(3, dtype=torch.int32, device="cuda:0"))),
                         ("verify", dict(path=torch.zeros(1, 3, dtype=torch.int32, device="cuda:0"))),
                         ("verify", dict(target=torch.zeros(2, 100, dtype=torch.float64, device="cuda:0"))),
                         ("compact", dict(kept=torch.zeros(2, 1, dtype=torch.int32, device="cuda:0"))),
                         ("compact", dict(n_kept=torch.zeros(2, dtype=torch.int32, device="cuda:0")))]:
        x = some("cuda:0")
        x.update(change)
        with pytest.raises(ValueError):
            calls(x)[call]()
    x = some("cuda:0")
    x["new_len"] = x["kv_len"]
    with pytest.raises(ValueError):
        calls(x)["compact"]()
    for name in ("n_path", "token"):
        x = some("cuda:0")
        x[name] = x["ids"][:1]
        with pytest.raises(ValueError):
            calls(x)["verify"]()
    x = some("cuda:0")
    x["token"] = x["path"][0, 1:]
    with pytest.raises(ValueError):
        calls(x)["verify"]()
    x = some("cuda:0")
    x["out"] = x["q"] = x["kn"]
    with pytest.raises(ValueError):
        calls(x)["append"]()
    x = some("cuda:0")
    x["freqs"] = torch.zeros(33, device="cuda:0")   # more than the head has
    with pytest.raises(RuntimeError):
        calls(x)["rotary"]()
    with pytest.raises(RuntimeError):
        tm.verify_tree(x["target"], x["ids"], x["parents"], x["q_start"], x["u"], max_q=513)


def test_rotary_frequencies():
    f = tm.rotary_frequencies(64)
    assert f.dtype == torch.float32 and f.shape == (32,)
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert all(abs(a - b) <= 2 ** -24 * b for a, b in zip(f.tolist(), want))   # (rounded once)
    assert torch.equal(tm.rotary_frequencies(64, method="linear", factor=4.0), f / 4)
    g = tm.rotary_frequencies(64, method="base", factor=8.0)
    assert g[0] == 1 and abs(float(g[-1]) * 8 / float(f[-1]) - 1) < 2 ** -22
    h = tm.rotary_frequencies(64, method="bands", factor=8.0, context=4096)
    turns = 4096 * f.double() / (2 * math.pi)
    assert torch.equal(h[turns > 32.1], f[turns > 32.1])
    slow = turns < 0.9
    assert slow.any() and torch.allclose(h[slow], f[slow] / 8, rtol=2 ** -22, atol=0)
    between = (turns > 1.1) & (turns < 31.9)
    assert between.any() and (h[between] < f[between]).all() and (h[between] > f[between] / 8).all()
    assert tm.rotary_frequencies(2, method="base", factor=2.0).tolist() == [1.0]
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=8, method="other"), dict(rotary_dim=8, method="bands", slow=3.0, fast=2.0)):
        with pytest.raises(ValueError):
            tm.rotary_frequencies(**bad)
