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

The calls run on the tensors' device, on its current stream or on ``stream`` (a
tensor let go before that one has run needs its ``record_stream``), allocate only
what they return and, for ``paged_attention``, a workspace, with torch's allocator.
They raise ValueError for tensors that do not fit and RuntimeError for what the
library refuses; there is no fallback.  None has a backward: where autograd is on, a
tensor that requires a gradient is refused.

The functions here are thin: the checks and the calls are in
csrc/tms_cache_py.cpp, built beside the library.  The ctypes structures are the C
ABI's, for callers without torch.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from .sampler import load_library


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


# The module that checks the tensors, allocates and calls, and torch's current
# stream of a device; loaded by the first call.
_OPS = _RAW_STREAM = None


def _ready():
    global _OPS, _RAW_STREAM
    load_library()   # (says how to build, if it is not)
    import torch

    try:
        from . import _cache_ops
    except ImportError as e:
        raise ImportError(f"the cache calls' module is not built, or not for this torch: run python -m tensormark_amd.build ({e})") from e

    _OPS, _RAW_STREAM = _cache_ops, torch._C._cuda_getCurrentRawStream


def _current(t) -> int:
    """The stream to run on, as an address."""
    return _RAW_STREAM(t.get_device()) if t.is_cuda else 0


def _on(stream, t):
    """`stream` as the current one: what a call allocates belongs to it."""
    import torch

    if not t.is_cuda:
        raise ValueError("a device tensor is needed")
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=t.device))


def kv_append(k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, scores=None, stream=None) -> None:
    """Write new tokens' keys and values (``[tokens, kv_heads, head_dim]``) to
    their slots, the last positions of each sequence's ``kv_len``; their slots' scores
    become 0.  Tokens without a mapped slot are dropped."""
    if _OPS is None:
        _ready()
    _OPS.kv_append(k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, max_q, scores,
                   _current(k_cache) if stream is None else stream)


def paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                    sinks: int = 0, scale: Optional[float] = None, out=None, lse=None, stream=None):
    """Attention of the new tokens' queries (``[tokens, q_heads, head_dim]``) over
    the cache, causal by position; with ``window`` > 0 a token sees the last ``window``
    positions and the first ``sinks``.  Returns (out, lse): like q, and the float32
    ``[tokens, q_heads]`` log of each row's sum of exponentials (-inf, and
    out 0, where a row sees nothing).  ``scale`` is 1 / sqrt(head_dim) by default."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, q):
            return paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, max_q=max_q, max_kv=max_kv, window=window,
                                   sinks=sinks, scale=scale, out=out, lse=lse)
    return _OPS.paged_attention(q, k_cache, v_cache, tables, kv_len, q_start, max_q, max_kv, window, sinks, scale, out, lse,
                                _current(q))


def kv_add_scores(q, lse, k_cache, scores, tables, kv_len, q_start, *, max_q: int, max_kv: int, window: int = 0,
                  sinks: int = 0, scale: Optional[float] = None, out=None, stream=None):
    """Add to every cached key's score the attention weight that the new tokens'
    queries give it, summed over them and the query heads of its key head.
    ``lse``, ``window``, ``sinks`` and ``scale`` are those of the paged_attention call.
    ``out`` (like ``scores``, default ``scores`` itself) is returned; every mapped position
    is written there, nothing else."""
    if _OPS is None:
        _ready()
    return _OPS.kv_add_scores(q, lse, k_cache, scores, tables, kv_len, q_start, max_q, max_kv, window, sinks, scale, out,
                              _current(q) if stream is None else stream)


def kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, *, budget: int, max_kv: int, sinks: int = 0,
             recent: int = 0, new_len=None, kept=None, stream=None):
    """Cut each sequence to ``budget`` positions a head: the first ``sinks``, the
    last ``recent`` and those of the largest scores stay (ties: the lowest position),
    in order, and go with their scores to ``dst_tables``' pages, which must be none of the
    sequences' own.  Positions on unmapped pages are not kept, so a sequence may have fewer
    than ``budget`` left.  Returns (new_len, kept): int32 ``[batch]`` and the old positions
    ``[batch, kv_heads, budget]``, -1 past new_len."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, k_cache):
            return kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, budget=budget, max_kv=max_kv, sinks=sinks,
                            recent=recent, new_len=new_len, kept=kept)
    return _OPS.kv_evict(k_cache, v_cache, scores, tables, kv_len, dst_tables, budget, max_kv, sinks, recent, new_len, kept,
                         _current(k_cache))


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
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, logits):
            return adjust_logits(logits, params, recent=recent, n_recent=n_recent, drafts=drafts, steps=steps, bias_ids=bias_ids,
                                 bias_values=bias_values, mask=mask, out=out)
    return _OPS.adjust_logits(logits, params, recent, n_recent, drafts, steps, bias_ids, bias_values, mask, out, _current(logits))
