"""The paged cache of keys and values, and the logits rules, over the C ABI of
include/tmcache_hip.h: ``kv_append``, ``paged_attention``, ``kv_add_scores``,
``kv_evict`` and ``adjust_logits``.

A pool is a device tensor ``[pages, kv_heads, page_size, head_dim]`` (bf16 or
fp16), of any strides whose last is 1; ``tables`` is int32 ``[batch, entries]``, an
entry outside the pool an unmapped page.  ``kv_len`` (int32 ``[batch]``) counts
a sequence's positions, its new tokens among them; ``q_start`` (int32
``[batch + 1]``) says which rows of the call's tokens are whose.  ``max_q`` and
``max_kv`` are the host's bounds on a sequence's new tokens and positions: the
lengths themselves stay on the device and nothing is synchronised.

The calls run on the current stream (or ``stream``), allocate only what they
return and, for ``paged_attention``, a workspace, with torch's allocator.  They raise
ValueError for tensors that do not fit and RuntimeError for what the library
refuses; there is no fallback.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from .sampler import DTYPE_BF16, DTYPE_F16, DTYPE_F32, ROW_DTYPE, _check, load_library


class CacheArgs(C.Structure):
    """tms_cache."""

    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("scores", C.c_void_p),
        ("k_stride", C.c_int64 * 3), ("v_stride", C.c_int64 * 3),
        ("dtype", C.c_int32), ("pages", C.c_int32), ("kv_heads", C.c_int32),
        ("page_size", C.c_int32), ("head_dim", C.c_int32), ("batch", C.c_int32),
        ("tables", C.c_void_p), ("table_stride", C.c_int64), ("kv_len", C.c_void_p),
        ("q_start", C.c_void_p), ("tokens", C.c_int32), ("max_q", C.c_int32),
        ("max_kv", C.c_int32), ("reserved", C.c_int32),
    ]


class AppendArgs(C.Structure):
    """tms_append_args."""

    _fields_ = [("k_new", C.c_void_p), ("v_new", C.c_void_p),
                ("k_new_stride", C.c_int64 * 2), ("v_new_stride", C.c_int64 * 2)]


class AttentionArgs(C.Structure):
    """tms_attention_args."""

    _fields_ = [
        ("q", C.c_void_p), ("out", C.c_void_p), ("lse", C.c_void_p),
        ("q_stride", C.c_int64 * 2), ("out_stride", C.c_int64 * 2), ("q_heads", C.c_int32),
        ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class ScoreArgs(C.Structure):
    """tms_score_args."""

    _fields_ = [
        ("q", C.c_void_p), ("lse", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64 * 2),
        ("q_heads", C.c_int32), ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float),
    ]


class EvictArgs(C.Structure):
    """tms_evict_args."""

    _fields_ = [
        ("dst_tables", C.c_void_p), ("dst_table_stride", C.c_int64), ("budget", C.c_int32),
        ("sinks", C.c_int32), ("recent", C.c_int32), ("reserved", C.c_int32),
        ("new_len", C.c_void_p), ("kept", C.c_void_p),
    ]


class AdjustArgs(C.Structure):
    """tms_adjust_args."""

    _fields_ = [
        ("logits", C.c_void_p), ("out", C.c_void_p), ("dtype", C.c_int32), ("out_dtype", C.c_int32),
        ("seqs", C.c_int32), ("steps", C.c_int32), ("vocab", C.c_int32), ("n_bias", C.c_int32),
        ("row_stride", C.c_int64), ("out_stride", C.c_int64), ("params", C.c_void_p),
        ("recent", C.c_void_p), ("n_recent", C.c_void_p), ("recent_stride", C.c_int64), ("n_history", C.c_int32), ("reserved", C.c_int32),
        ("drafts", C.c_void_p), ("bias_ids", C.c_void_p), ("bias_values", C.c_void_p),
        ("mask", C.c_void_p), ("mask_stride", C.c_int64),
    ]


_FNS = None


def _fns():
    """The library with this module's calls declared."""
    global _FNS
    if _FNS is None:
        lib = load_library()
        cp, vp = C.POINTER(CacheArgs), C.c_void_p
        lib.tms_kv_append.argtypes = [cp, C.POINTER(AppendArgs), vp]
        lib.tms_paged_attention_workspace.argtypes = [cp, C.POINTER(AttentionArgs)]
        lib.tms_paged_attention_workspace.restype = C.c_int64
        lib.tms_paged_attention.argtypes = [cp, C.POINTER(AttentionArgs), vp]
        lib.tms_kv_add_scores.argtypes = [cp, C.POINTER(ScoreArgs), vp]
        lib.tms_kv_evict.argtypes = [cp, C.POINTER(EvictArgs), vp]
        lib.tms_adjust_logits.argtypes = [C.POINTER(AdjustArgs), vp]
        _FNS = lib
    return _FNS


torch = None   # imported by the first call, like the sampler's


def _ready():
    global torch
    import torch as t

    torch = t


def _stream(stream, device: int):
    """The stream to run on, as an address."""
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream


def _on(stream, t):
    """`stream` as the current one: what a call allocates belongs to it."""
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=t.device))


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t, shape, what, device: int):
    """The address of a contiguous int32 tensor of that shape on the device."""
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{what}: a contiguous int32 tensor {list(shape)} on cuda:{device}, not {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _pool(t, what):
    """A pool's page, head and slot strides; that of a single head or page does not matter."""
    st, shape = t.stride(), t.shape
    if st[3] != 1:
        raise ValueError(f"{what}: the last stride must be 1")
    if shape[0] == 1 or shape[1] == 1:
        return (st[0] if shape[0] > 1 else 0, st[1] if shape[1] > 1 else 0, st[2])
    return st[:3]


# Only addresses, sizes and strides are read here, once each: a decode step is
# short enough for its calls' host time to count.
def _cache(k, v, scores, tables, kv_len, q_start, tokens, max_q, max_kv):
    """The call's tms_cache and its device's index."""
    device, dtype, shape = k.get_device(), k.dtype, k.shape
    if len(shape) != 4 or shape[0] < 1:
        raise ValueError("k_cache: [pages, kv_heads, page_size, head_dim]")
    if dtype == torch.bfloat16:
        code = DTYPE_BF16
    elif dtype == torch.float16:
        code = DTYPE_F16
    else:
        raise ValueError(f"k_cache: bfloat16 or float16, not {dtype}")
    if device < 0:
        raise ValueError("k_cache: a device tensor")
    vp, vs = None, (0, 0, 0)
    if v is not None:
        if v.shape != shape or v.dtype != dtype or v.get_device() != device:
            raise ValueError("v_cache: like k_cache")
        vp, vs = v.data_ptr(), _pool(v, "v_cache")
    sp = None
    if scores is not None:
        if scores.dtype != torch.float32 or scores.shape != shape[:3] or not scores.is_contiguous() or scores.get_device() != device:
            raise ValueError("scores: contiguous float32 [pages, kv_heads, page_size]")
        sp = scores.data_ptr()
    ts = tables.shape
    if tables.dtype != torch.int32 or tables.get_device() != device or len(ts) != 2 or not tables.is_contiguous() or ts[1] < 1:
        raise ValueError("tables: contiguous int32 [batch, entries]")
    batch = ts[0]
    return CacheArgs(k.data_ptr(), vp, sp, _pool(k, "k_cache"), vs, code, *shape, batch, tables.data_ptr(), ts[1],
                     _ints(kv_len, (batch,), "kv_len", device),
                     None if q_start is None else _ints(q_start, (batch + 1,), "q_start", device), tokens, max_q, max_kv, 0), device


def _rows(t, k, what):
    """The token and head strides of [tokens, heads, head_dim] rows of the cache's type; that of a single one does not matter."""
    D, st, shape = k.shape[-1], t.stride(), t.shape
    if len(st) != 3 or t.dtype != k.dtype or t.get_device() != k.get_device() or shape[2] != D or st[2] != 1:
        raise ValueError(f"{what}: [tokens, heads, {D}] of {k.dtype} on {k.device}, last stride 1")
    return (st[0] if shape[0] > 1 else 0, st[1] if shape[1] > 1 else 0)


def _f32_rows(t, rows, what, device: int):
    """The address of a contiguous float32 [tokens, q_heads]."""
    if t.dtype != torch.float32 or t.shape != rows or not t.is_contiguous() or t.get_device() != device:
        raise ValueError(f"{what}: contiguous float32 [tokens, q_heads]")
    return t.data_ptr()


def _reach(n: int) -> int:
    """A window or a number of sinks as the library's 32 bits: none see further."""
    return n if 0 <= n < 2 ** 31 else 0 if n < 0 else 2 ** 31 - 1


def kv_append(k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, scores=None, stream=None) -> None:
    """Write new tokens' keys and values (``[tokens, kv_heads, head_dim]``) to
    their slots, the last positions of each sequence's ``kv_len``; their slots' scores
    become 0.  Tokens without a mapped slot are dropped."""
    if torch is None:
        _ready()
    c, device = _cache(k_cache, v_cache, scores, tables, kv_len, q_start, k_new.shape[0], max_q, 0)
    ks, vs = _rows(k_new, k_cache, "k_new"), _rows(v_new, k_cache, "v_new")
    _want(k_new.shape == v_new.shape and k_new.shape[1] == k_cache.shape[1], "k_new, v_new: one row a key head")
    a = AppendArgs(k_new.data_ptr(), v_new.data_ptr(), ks, vs)
    _check(_fns().tms_kv_append(C.byref(c), C.byref(a), _stream(stream, device)), "tms_kv_append")


def paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                    sinks: int = 0, scale: Optional[float] = None, out=None, lse=None, stream=None):
    """Attention of the new tokens' queries (``[tokens, q_heads, head_dim]``) over
    the cache, causal by position; with ``window`` > 0 a token sees the last ``window``
    positions and the first ``sinks``.  Returns (out, lse): like q, and the float32
    ``[tokens, q_heads]`` log of each row's sum of exponentials (-inf, and
    out 0, where a row sees nothing).  ``scale`` is 1 / sqrt(head_dim) by default."""
    if torch is None:
        _ready()
    if stream is not None:
        with _on(stream, q):
            return paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, max_q=max_q, max_kv=max_kv, window=window,
                                   sinks=sinks, scale=scale, out=out, lse=lse)
    qs = _rows(q, k_cache, "q")
    T, H, D = q.shape
    c, device = _cache(k_cache, v_cache, None, tables, kv_len, q_start, T, max_q, max_kv)
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((T, H), dtype=torch.float32, device=q.device)
    _want(out.shape == q.shape, "out: like q")
    a = AttentionArgs(q.data_ptr(), out.data_ptr(), _f32_rows(lse, (T, H), "lse", device), qs, _rows(out, k_cache, "out"), H,
                      _reach(window), sinks if sinks < 2 ** 31 else 2 ** 31 - 1, 1.0 / math.sqrt(D) if scale is None else scale,
                      None, 0)
    lib = _fns()
    need = lib.tms_paged_attention_workspace(C.byref(c), C.byref(a))
    if need < 0:
        _check(need, "tms_paged_attention")
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _check(lib.tms_paged_attention(C.byref(c), C.byref(a), _stream(None, device)), "tms_paged_attention")
    return out, lse


def kv_add_scores(q, lse, k_cache, scores, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                  sinks: int = 0, scale: Optional[float] = None, out=None, stream=None):
    """Add to every cached key's score the attention weight that the new tokens'
    queries give it, summed over them and the query heads of its key head.
    ``lse``, ``window``, ``sinks`` and ``scale`` are those of the paged_attention call.
    ``out`` (like ``scores``, default ``scores`` itself) is returned; every mapped position
    is written there, nothing else."""
    if torch is None:
        _ready()
    _want(scores is not None, "scores: needed")
    qs, (T, H, D) = _rows(q, k_cache, "q"), q.shape
    c, device = _cache(k_cache, None, scores, tables, kv_len, q_start, T, max_q, max_kv)
    if out is None:
        out = scores
    _want(out.dtype == scores.dtype and out.shape == scores.shape and out.is_contiguous() and out.get_device() == device,
          "out: like scores")
    a = ScoreArgs(q.data_ptr(), _f32_rows(lse, (T, H), "lse", device), out.data_ptr(), qs, H, _reach(window),
                  sinks if sinks < 2 ** 31 else 2 ** 31 - 1, 1.0 / math.sqrt(D) if scale is None else scale)
    _check(_fns().tms_kv_add_scores(C.byref(c), C.byref(a), _stream(stream, device)), "tms_kv_add_scores")
    return out


def kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, *, budget: int, max_kv: int, sinks: int = 0,
             recent: int = 0, new_len=None, kept=None, stream=None):
    """Cut each sequence to ``budget`` positions a head: the first ``sinks``, the
    last ``recent`` and those of the largest scores stay (ties: the lowest position),
    in order, and go with their scores to ``dst_tables``' pages, which must be none of the
    sequences' own.  Returns (new_len, kept): int32 ``[batch]`` and the old positions
    ``[batch, kv_heads, budget]``, -1 past new_len."""
    if torch is None:
        _ready()
    if stream is not None:
        with _on(stream, k_cache):
            return kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, budget=budget, max_kv=max_kv, sinks=sinks,
                            recent=recent, new_len=new_len, kept=kept)
    _want(scores is not None, "scores: needed")
    c, device = _cache(k_cache, v_cache, scores, tables, kv_len, None, 0, 0, max_kv)
    B, H = tables.shape[0], k_cache.shape[1]
    _want(dst_tables.dim() == 2 and dst_tables.shape[0] == B, "dst_tables: int32 [batch, entries]")
    _want(budget >= 1, "budget: at least 1")
    if new_len is None:
        new_len = torch.empty(B, dtype=torch.int32, device=k_cache.device)
    if kept is None:
        kept = torch.empty((B, H, budget), dtype=torch.int32, device=k_cache.device)
    a = EvictArgs(_ints(dst_tables, dst_tables.shape, "dst_tables", device), dst_tables.shape[1], budget, sinks, recent, 0,
                  _ints(new_len, (B,), "new_len", device), _ints(kept, (B, H, budget), "kept", device))
    _check(_fns().tms_kv_evict(C.byref(c), C.byref(a), _stream(None, device)), "tms_kv_evict")
    return new_len, kept


def adjust_logits(logits, params=None, *, recent=None, n_recent=None, drafts=None, steps: int = 1, bias_ids=None,
                  bias_values=None, mask=None, out=None, stream=None):
    """Mask, penalties and biases on rows of logits (``[seqs * steps, vocab]``
    fp32, fp16 or bf16), rounded once into ``out`` (the logits' type or fp32; may be
    ``logits`` itself; by default new and like logits).  Row r is step r % steps of sequence
    r // steps, and its history the sequence's ``recent`` ids (``[seqs, n]``, the first
    n_recent of them) and then its first r % steps ``drafts`` (``[seqs, steps - 1]``), so
    the rows of a speculative verify get what sampling them one by one would.
    ``params`` is a device uint8 tensor of ROW_DTYPE records, one a sequence
    (Sampler.params_tensor); ``bias_ids`` / ``bias_values`` are int32 / float32
    ``[seqs, n]`` (an id outside the vocabulary is left out); ``mask`` is int32 or uint32
    words ``[seqs * steps, ceil(vocab / 32)]``, masked ids become -inf."""
    if torch is None:
        _ready()
    if stream is not None:
        with _on(stream, logits):
            return adjust_logits(logits, params, recent=recent, n_recent=n_recent, drafts=drafts, steps=steps, bias_ids=bias_ids,
                                 bias_values=bias_values, mask=mask, out=out)
    dtype, device = logits.dtype, logits.get_device()
    _want(logits.dim() == 2 and dtype in (torch.float32, torch.float16, torch.bfloat16) and device >= 0 and
          (logits.stride(1) == 1 or logits.shape[1] == 1),
          "logits: device [rows, vocab] of float32, float16 or bfloat16, last stride 1")
    R, V = logits.shape
    _want(steps >= 1 and R % steps == 0, "logits: a multiple of `steps` rows")
    S = R // steps
    a = AdjustArgs()
    a.dtype = a.out_dtype = DTYPE_F32 if dtype == torch.float32 else DTYPE_F16 if dtype == torch.float16 else DTYPE_BF16
    a.seqs, a.steps, a.vocab = S, steps, V
    a.row_stride = a.out_stride = V
    if R > 1:
        a.row_stride = logits.stride(0)
    if params is not None:
        _want(params.dtype == torch.uint8 and params.is_contiguous() and params.numel() == S * ROW_DTYPE.itemsize and
              params.get_device() == device, "params: uint8 ROW_DTYPE records, one a sequence")
        a.params = params.data_ptr()
    if recent is not None:
        _want(recent.dim() == 2 and recent.shape[0] == S and recent.dtype == torch.int32 and recent.get_device() == device and
              (recent.stride(1) == 1 or recent.shape[1] <= 1) and (S <= 1 or recent.stride(0) >= recent.shape[1]),
              "recent: int32 [seqs, n] on the logits' device, rows contiguous")
        a.recent, a.recent_stride, a.n_history = recent.data_ptr(), recent.stride(0) if S > 1 else recent.shape[1], recent.shape[1]
        if n_recent is not None:
            a.n_recent = _ints(n_recent, (S,), "n_recent", device)
    if drafts is not None and steps > 1:
        a.drafts = _ints(drafts, (S, steps - 1), "drafts", device)
    _want((bias_ids is None) == (bias_values is None), "bias_ids and bias_values go together")
    if bias_ids is not None and bias_ids.numel():
        n = bias_ids.shape[-1]
        a.n_bias, a.bias_ids = n, _ints(bias_ids, (S, n), "bias_ids", device)
        _want(bias_values.dtype == torch.float32 and bias_values.shape == (S, n) and bias_values.is_contiguous() and
              bias_values.get_device() == device, "bias_values: contiguous float32, like bias_ids")
        a.bias_values = bias_values.data_ptr()
    if mask is not None:
        _want(mask.dim() == 2 and mask.shape[0] == R and mask.element_size() == 4 and not mask.is_floating_point() and
              (mask.stride(1) == 1 or mask.shape[1] == 1) and mask.get_device() == device and mask.shape[1] >= (V + 31) // 32,
              "mask: 32-bit words [rows, ceil(vocab / 32)]")
        a.mask, a.mask_stride = mask.data_ptr(), mask.stride(0) if R > 1 else mask.shape[1]
    if out is None:
        out = torch.empty((R, V), dtype=dtype, device=logits.device)
    else:
        _want(out.shape == logits.shape and out.dtype in (dtype, torch.float32) and out.get_device() == device and
              (out.stride(1) == 1 or V == 1), "out: like logits, of its type or float32")
        if out.dtype != dtype:
            a.out_dtype = DTYPE_F32
        if R > 1:
            a.out_stride = out.stride(0)
    a.logits, a.out = logits.data_ptr(), out.data_ptr()
    _check(_fns().tms_adjust_logits(C.byref(a), _stream(None, device)), "tms_adjust_logits")
    return out
