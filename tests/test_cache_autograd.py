"""The cache calls and autograd: no call has a backward, so a gradient that would have to
go through one is refused; and what a call writes counts as written."""
from __future__ import annotations

import pytest
import torch

import tensormark_amd as tm


def some(device):
    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=device)

    x = dict(k=zeros(4, 2, 16, 64), v=zeros(4, 2, 16, 64), scores=zeros(4, 2, 16, dtype=torch.float32), q=zeros(1, 4, 64),
             kn=zeros(1, 2, 64), vn=zeros(1, 2, 64), lse=zeros(1, 4, dtype=torch.float32), out=zeros(1, 4, 64),
             logits=zeros(1, 100, dtype=torch.float32), values=zeros(1, 3, dtype=torch.float32))
    ints = dict(tables=[[0, 1]], kv_len=[20], q_start=[0, 1], dst=[[2]], ids=[[1, 2, 3]], new_len=[0])
    x.update({n: torch.tensor(v, dtype=torch.int32, device=device) for n, v in ints.items()})
    x["kept"] = torch.zeros(1, 2, 8, dtype=torch.int32, device=device)
    return x


def calls(x):
    where = (x["tables"], x["kv_len"], x["q_start"])
    both = dict(max_q=1, max_kv=20)
    return dict(
        append=lambda: tm.kv_append(x["kn"], x["vn"], x["k"], x["v"], *where, max_q=1, scores=x["scores"]),
        attend=lambda: tm.paged_attention(x["q"], x["k"], x["v"], *where, **both, out=x["out"], lse=x["lse"]),
        scores=lambda: tm.kv_add_scores(x["q"], x["lse"], x["k"], x["scores"], *where, **both),
        evict=lambda: tm.kv_evict(x["k"], x["v"], x["scores"], x["tables"], x["kv_len"], x["dst"], budget=8, max_kv=20,
                                  new_len=x["new_len"], kept=x["kept"]),
        adjust=lambda: tm.adjust_logits(x["logits"], bias_ids=x["ids"], bias_values=x["values"], out=x["logits"]))


TAKES = dict(append=("kn", "vn", "k", "v", "scores"), attend=("q", "k", "v", "out", "lse"), scores=("q", "lse", "k", "scores"),
             evict=("k", "v", "scores"), adjust=("logits", "values"))


@pytest.mark.parametrize("call, name", [(c, n) for c, names in TAKES.items() for n in names])
def test_a_tensor_that_requires_a_gradient_is_refused(call, name):
    x = some("cpu")
    x[name].requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        calls(x)[call]()
    with torch.no_grad(), pytest.raises(ValueError) as e:   # (a host tensor is refused all the same)
        calls(x)[call]()
    assert "gradient" not in str(e.value)


@pytest.mark.gpu
def test_what_a_call_writes_counts_as_written():
    writes = dict(append=("k", "v", "scores"), attend=("out", "lse"), scores=("scores",), evict=("k", "v", "scores", "new_len", "kept"),
                  adjust=("logits",))
    for call, names in writes.items():
        x = some("cuda:0")
        before = {n: t._version for n, t in x.items()}
        calls(x)[call]()
        assert {n for n, t in x.items() if t._version != before[n]} == set(names), call
    with torch.inference_mode():
        x = some("cuda:0")
    for call in writes:
        calls(x)[call]()
    x = some("cuda:0")
    x["q"].requires_grad_()
    with torch.no_grad():
        out, _ = calls(x)["attend"]()
    assert not out.requires_grad
