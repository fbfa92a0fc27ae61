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
        ("recent", C.c_void_p), ("n_recent", C.c_void_p), ("recent_stride", C.c_int64),
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


def _stream(stream, t) -> C.c_void_p:
    import torch

    return C.c_void_p(stream if stream is not None else torch.cuda.current_stream(t.device).cuda_stream)


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t, shape, what, like):
    """A contiguous int32 tensor of that shape on the pool's device; its address."""
    import torch

    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{what}: a contiguous int32 tensor {list(shape)} on {like.device}, not {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _cache(k, v, scores, tables, kv_len, q_start, tokens, max_q, max_kv) -> CacheArgs:
    import torch

    _want(k.dim() == 4 and k.shape[0] >= 1, "k_cache: [pages, kv_heads, page_size, head_dim]")
    _want(k.dtype in (torch.bfloat16, torch.float16), f"k_cache: bfloat16 or float16, not {k.dtype}")
    _want(k.is_cuda, "k_cache: a device tensor")
    _want(k.stride(3) == 1, "k_cache: the last stride must be 1")
    c = CacheArgs()
    c.k, c.dtype = k.data_ptr(), DTYPE_BF16 if k.dtype == torch.bfloat16 else DTYPE_F16
    c.pages, c.kv_heads, c.page_size, c.head_dim = k.shape
    c.k_stride[0], c.k_stride[1], c.k_stride[2] = k.stride()[:3]
    if v is not None:
        _want(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device and v.stride(3) == 1,
              "v_cache: like k_cache")
        c.v = v.data_ptr()
        c.v_stride[0], c.v_stride[1], c.v_stride[2] = v.stride()[:3]
    if scores is not None:
        _want(scores.dtype == torch.float32 and scores.shape == k.shape[:3] and scores.is_contiguous() and
              scores.device == k.device, "scores: contiguous float32 [pages, kv_heads, page_size]")
        c.scores = scores.data_ptr()
    _want(tables.dim() == 2 and tables.dtype == torch.int32 and tables.device == k.device and
          (tables.stride(1) == 1 or tables.shape[1] <= 1) and tables.shape[1] >= 1, "tables: int32 [batch, entries], rows contiguous")
    c.batch, c.tables = tables.shape[0], tables.data_ptr()
    _want(tables.shape[0] <= 1 or tables.stride(0) == tables.shape[1], "tables: contiguous")
    c.table_stride = tables.shape[1]
    c.kv_len = _ints(kv_len, (c.batch,), "kv_len", k)
    if q_start is not None:
        c.q_start = _ints(q_start, (c.batch + 1,), "q_start", k)
    c.tokens, c.max_q, c.max_kv = tokens, max_q, max_kv
    return c


def _rows(t, k, what):
    """[tokens, heads, head_dim] rows of the cache's type; its token and head strides."""
    _want(t.dim() == 3 and t.dtype == k.dtype and t.device == k.device and t.shape[2] == k.shape[3] and
          (t.stride(2) == 1 or t.shape[2] == 1), f"{what}: [tokens, heads, {k.shape[3]}] of {k.dtype} on {k.device}, last stride 1")
    return t.stride(0), t.stride(1)


def kv_append(k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, scores=None, stream=None) -> None:
    """Write new tokens' keys and values (``[tokens, kv_heads, head_dim]``) to
    their slots, the last positions of each sequence's ``kv_len``; their slots' scores
    become 0.  Tokens without a mapped slot are dropped."""
    c = _cache(k_cache, v_cache, scores, tables, kv_len, q_start, k_new.shape[0], max_q, 0)
    a = AppendArgs()
    a.k_new_stride[0], a.k_new_stride[1] = _rows(k_new, k_cache, "k_new")
    a.v_new_stride[0], a.v_new_stride[1] = _rows(v_new, k_cache, "v_new")
    _want(k_new.shape == v_new.shape and k_new.shape[1] == k_cache.shape[1], "k_new, v_new: one row a key head")
    a.k_new, a.v_new = k_new.data_ptr(), v_new.data_ptr()
    _check(_fns().tms_kv_append(C.byref(c), C.byref(a), _stream(stream, k_cache)), "tms_kv_append")


def paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                    sinks: int = 0, scale: Optional[float] = None, out=None, lse=None, stream=None):
    """Attention of the new tokens' queries (``[tokens, q_heads, head_dim]``) over
    the cache, causal by position; with ``window`` > 0 a token sees the last ``window``
    positions and the first ``sinks``.  Returns (out, lse): like q, and the float32
    ``[tokens, q_heads]`` log of each row's sum of exponentials (-inf, and
    out 0, where a row sees nothing).  ``scale`` is 1 / sqrt(head_dim) by default."""
    import torch

    c = _cache(k_cache, v_cache, None, tables, kv_len, q_start, q.shape[0], max_q, max_kv)
    a = AttentionArgs()
    a.q_stride[0], a.q_stride[1] = _rows(q, k_cache, "q")
    T, H, D = q.shape
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    a.out_stride[0], a.out_stride[1] = _rows(out, k_cache, "out")
    if lse is None:
        lse = torch.empty((T, H), dtype=torch.float32, device=q.device)
    _want(out.shape == q.shape, "out: like q")
    _want(lse.dtype == torch.float32 and lse.shape == (T, H) and lse.is_contiguous() and lse.device == q.device,
          "lse: contiguous float32 [tokens, q_heads]")
    a.q, a.out, a.lse, a.q_heads = q.data_ptr(), out.data_ptr(), lse.data_ptr(), H
    a.window, a.sinks, a.scale = max(window, 0), sinks, 1.0 / math.sqrt(D) if scale is None else scale
    lib = _fns()
    need = lib.tms_paged_attention_workspace(C.byref(c), C.byref(a))
    if need < 0:
        _check(int(need), "tms_paged_attention")
    if need > 0:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        if stream is not None:
            ws.record_stream(torch.cuda.ExternalStream(stream, device=q.device))
    _check(lib.tms_paged_attention(C.byref(c), C.byref(a), _stream(stream, q)), "tms_paged_attention")
    return out, lse


def kv_add_scores(q, lse, k_cache, scores, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                  sinks: int = 0, scale: Optional[float] = None, out=None, stream=None):
    """Add to every cached key's score the attention weight that the new tokens'
    queries give it, summed over them and the query heads of its key head.
    ``lse``, ``window``, ``sinks`` and ``scale`` are those of the paged_attention call.
    ``out`` (like ``scores``, default ``scores`` itself) is returned; every mapped position
    is written there, nothing else."""
    import torch

    _want(scores is not None, "scores: needed")
    c = _cache(k_cache, None, scores, tables, kv_len, q_start, q.shape[0], max_q, max_kv)
    a = ScoreArgs()
    a.q_stride[0], a.q_stride[1] = _rows(q, k_cache, "q")
    _want(lse.dtype == torch.float32 and lse.shape == q.shape[:2] and lse.is_contiguous() and lse.device == q.device,
          "lse: contiguous float32 [tokens, q_heads]")
    if out is None:
        out = scores
    _want(out.dtype == torch.float32 and out.shape == scores.shape and out.is_contiguous() and out.device == q.device,
          "out: like scores")
    a.q, a.lse, a.out, a.q_heads = q.data_ptr(), lse.data_ptr(), out.data_ptr(), q.shape[1]
    a.window, a.sinks, a.scale = max(window, 0), sinks, 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    _check(_fns().tms_kv_add_scores(C.byref(c), C.byref(a), _stream(stream, q)), "tms_kv_add_scores")
    return out


def kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, *, budget: int, max_kv: int, sinks: int = 0,
             recent: int = 0, new_len=None, kept=None, stream=None):
    """Cut each sequence to ``budget`` positions a head: the first ``sinks``, the
    last ``recent`` and those of the largest scores stay (ties: the lowest position),
    in order, and go with their scores to ``dst_tables``' pages, which must be none of the
    sequences' own.  Returns (new_len, kept): int32 ``[batch]`` and the old positions
    ``[batch, kv_heads, budget]``, -1 past new_len."""
    import torch

    _want(scores is not None, "scores: needed")
    c = _cache(k_cache, v_cache, scores, tables, kv_len, None, 0, 0, max_kv)
    _want(dst_tables.dim() == 2 and dst_tables.shape[0] == c.batch, "dst_tables: int32 [batch, entries]")
    a = EvictArgs()
    a.dst_tables = _ints(dst_tables, tuple(dst_tables.shape), "dst_tables", k_cache)
    a.dst_table_stride, a.budget, a.sinks, a.recent = dst_tables.shape[1], budget, sinks, recent
    _want(budget >= 1, "budget: at least 1")
    if new_len is None:
        new_len = torch.empty(c.batch, dtype=torch.int32, device=k_cache.device)
    if kept is None:
        kept = torch.empty((c.batch, c.kv_heads, budget), dtype=torch.int32, device=k_cache.device)
    a.new_len = _ints(new_len, (c.batch,), "new_len", k_cache)
    a.kept = _ints(kept, (c.batch, c.kv_heads, budget), "kept", k_cache)
    _check(_fns().tms_kv_evict(C.byref(c), C.byref(a), _stream(stream, k_cache)), "tms_kv_evict")
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
    import torch

    code = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}
    _want(logits.dim() == 2 and logits.dtype in code and logits.is_cuda and (logits.stride(1) == 1 or logits.shape[1] == 1),
          "logits: device [rows, vocab] of float32, float16 or bfloat16, last stride 1")
    R, V = logits.shape
    _want(steps >= 1 and R % steps == 0, "logits: a multiple of `steps` rows")
    S = R // steps
    if out is None:
        out = torch.empty((R, V), dtype=logits.dtype, device=logits.device)
    _want(out.shape == logits.shape and out.dtype in (logits.dtype, torch.float32) and out.device == logits.device and
          (out.stride(1) == 1 or V == 1), "out: like logits, of its type or float32")
    a = AdjustArgs()
    a.logits, a.out, a.dtype, a.out_dtype = logits.data_ptr(), out.data_ptr(), code[logits.dtype], code[out.dtype]
    a.seqs, a.steps, a.vocab = S, steps, V
    a.row_stride = logits.stride(0) if R > 1 else V
    a.out_stride = out.stride(0) if R > 1 else V
    if params is not None:
        _want(params.dtype == torch.uint8 and params.is_contiguous() and params.numel() == S * ROW_DTYPE.itemsize and
              params.device == logits.device, "params: uint8 ROW_DTYPE records, one a sequence")
        a.params = params.data_ptr()
    if recent is not None:
        _want(recent.dim() == 2 and recent.shape[0] == S, "recent: int32 [seqs, n]")
        _want(recent.dtype == torch.int32 and recent.device == logits.device and (recent.stride(1) == 1 or recent.shape[1] <= 1),
              "recent: int32 rows on the logits' device")
        a.recent, a.recent_stride = recent.data_ptr(), recent.stride(0) if S > 1 else recent.shape[1]
        if n_recent is not None:
            a.n_recent = _ints(n_recent, (S,), "n_recent", logits)
        elif a.recent_stride != recent.shape[1]:
            n_recent = torch.full((S,), recent.shape[1], dtype=torch.int32, device=logits.device)
            a.n_recent = n_recent.data_ptr()
    if drafts is not None and steps > 1:
        a.drafts = _ints(drafts, (S, steps - 1), "drafts", logits)
    _want((bias_ids is None) == (bias_values is None), "bias_ids and bias_values go together")
    if bias_ids is not None and bias_ids.numel():
        n = bias_ids.shape[-1]
        a.n_bias, a.bias_ids = n, _ints(bias_ids, (S, n), "bias_ids", logits)
        _want(bias_values.dtype == torch.float32 and tuple(bias_values.shape) == (S, n) and bias_values.is_contiguous() and
              bias_values.device == logits.device, "bias_values: contiguous float32, like bias_ids")
        a.bias_values = bias_values.data_ptr()
    if mask is not None:
        _want(mask.dim() == 2 and mask.shape[0] == R and mask.element_size() == 4 and not mask.is_floating_point() and
              (mask.stride(1) == 1 or mask.shape[1] == 1) and mask.device == logits.device and mask.shape[1] >= (V + 31) // 32,
              "mask: 32-bit words [rows, ceil(vocab / 32)]")
        a.mask, a.mask_stride = mask.data_ptr(), mask.stride(0) if R > 1 else mask.shape[1]
    _check(_fns().tms_adjust_logits(C.byref(a), _stream(stream, logits)), "tms_adjust_logits")
    return out
