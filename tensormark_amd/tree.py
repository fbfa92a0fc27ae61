"""Speculative decoding with trees of drafts over the paged cache, over the C ABI of
include/tmtree_hip.h: ``rotary_frequencies``, ``rotary``, ``kv_append_rotary``,
``tree_attention``, ``verify_tree`` and ``kv_compact``.

Pools, ``tables``, ``kv_len``, ``q_start``, ``max_q`` and ``max_kv`` are those of
tensormark_amd.cache.  A sequence's new tokens are its tree: node i is token
``q_start[b] + i``, cached at position ``kv_len - n + i`` of n nodes, and ``parents[t]``
(int32 ``[tokens]``) is the parent's i, below the node's own, or -1.  Node 0 is the last settled
token, the others are drafts.

The calls keep the cache calls' rules: they run on the tensors' device, on its current stream or
on ``stream`` (a tensor let go before that one has run needs its ``record_stream``), allocate
only what they return and a workspace, raise ValueError for tensors that do not fit and
RuntimeError for what the library refuses, have no derivative (tensors that require a gradient or
have a forward-mode tangent are refused) and no fallback.

The functions are thin: the checks and the calls are in csrc/tms_tree_py.cpp, built beside the
library.  The ctypes structures are the C ABI's, for callers without torch.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

from .cache import AttentionArgs, CacheArgs, _on
from .sampler import load_library


class RotaryArgs(C.Structure):
    """tms_rotary_args."""

    _fields_ = [
        ("x", C.c_void_p), ("out", C.c_void_p), ("x_stride", C.c_int64 * 2), ("out_stride", C.c_int64 * 2),
        ("positions", C.c_void_p), ("freqs", C.c_void_p), ("dtype", C.c_int32), ("tokens", C.c_int32), ("heads", C.c_int32),
        ("head_dim", C.c_int32), ("rotary_dim", C.c_int32), ("interleaved", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32),
    ]


class AppendRotaryArgs(C.Structure):
    """tms_append_rotary_args."""

    _fields_ = [
        ("k_new", C.c_void_p), ("v_new", C.c_void_p), ("k_new_stride", C.c_int64 * 2), ("v_new_stride", C.c_int64 * 2),
        ("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_int64 * 2), ("out_stride", C.c_int64 * 2),
        ("positions", C.c_void_p), ("freqs", C.c_void_p), ("q_heads", C.c_int32), ("rotary_dim", C.c_int32),
        ("interleaved", C.c_int32), ("scale", C.c_float),
    ]


class VerifyTreeArgs(C.Structure):
    """tms_verify_tree_args."""

    _fields_ = [
        ("target", C.c_void_p), ("draft", C.c_void_p), ("target_stride", C.c_int64), ("draft_stride", C.c_int64),
        ("dtype", C.c_int32), ("vocab", C.c_int32), ("batch", C.c_int32), ("tokens", C.c_int32), ("max_q", C.c_int32),
        ("reserved", C.c_int32), ("draft_tokens", C.c_void_p), ("parents", C.c_void_p), ("q_start", C.c_void_p),
        ("uniforms", C.c_void_p), ("path", C.c_void_p), ("kept", C.c_void_p), ("token", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class CompactArgs(C.Structure):
    """tms_compact_args."""

    _fields_ = [
        ("kept", C.c_void_p), ("kept_stride", C.c_int64), ("n_kept", C.c_void_p), ("dst_tables", C.c_void_p),
        ("dst_table_stride", C.c_int64), ("new_len", C.c_void_p), ("max_kept", C.c_int32), ("reserved", C.c_int32),
    ]


_FNS = None


def _fns():
    """The library with this module's calls declared."""
    global _FNS
    if _FNS is None:
        lib = load_library()
        cp, vp = C.POINTER(CacheArgs), C.c_void_p
        lib.tms_rotary.argtypes = [C.POINTER(RotaryArgs), vp]
        lib.tms_kv_append_rotary.argtypes = [cp, C.POINTER(AppendRotaryArgs), vp]
        lib.tms_tree_attention_workspace.argtypes = [cp, C.POINTER(AttentionArgs)]
        lib.tms_tree_attention_workspace.restype = C.c_int64
        lib.tms_tree_attention.argtypes = [cp, C.POINTER(AttentionArgs), vp, vp]
        lib.tms_verify_tree_workspace.argtypes = [C.POINTER(VerifyTreeArgs)]
        lib.tms_verify_tree_workspace.restype = C.c_int64
        lib.tms_verify_tree.argtypes = [C.POINTER(VerifyTreeArgs), vp]
        lib.tms_kv_compact.argtypes = [cp, C.POINTER(CompactArgs), vp]
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
        from . import _tree_ops
    except ImportError as e:
        raise ImportError(f"the tree calls' module is not built, or not for this torch: run python -m tensormark_amd.build ({e})") from e

    _OPS, _RAW_STREAM = _tree_ops, torch._C._cuda_getCurrentRawStream


def _current(t) -> int:
    """The stream to run on, as an address."""
    return _RAW_STREAM(t.get_device()) if t.is_cuda else 0


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, method: str = "none", factor: float = 1.0, context: int = 4096,
                       slow: float = 1.0, fast: float = 32.0, device=None):
    """The angles a position, float32 ``[rotary_dim / 2]``: ``base ** (-2 i / rotary_dim)``, and for
    contexts ``factor`` times the trained ``context``

    - "linear": all divided by ``factor``;
    - "base": the base raised so that the slowest is divided by ``factor`` and the fastest stays;
    - "bands": those with fewer than ``slow`` turns in the trained context divided, those with more
      than ``fast`` as they are, between them a share of both, linear in the turns.
    """
    import torch

    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim: even, 2 at least")
    if not (base > 0 and math.isfinite(base)) or not (factor >= 1 and math.isfinite(factor)):
        raise ValueError("base: above 0; factor: 1 at least")
    if method not in ("none", "linear", "base", "bands"):
        raise ValueError("method: none, linear, base or bands")
    if method == "bands" and not (0 <= slow < fast and context >= 1):
        raise ValueError("slow and fast: numbers of turns, the first the smaller; context: 1 at least")
    if method == "base" and rotary_dim > 2:
        base *= factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if method == "linear":
        f = f / factor
    elif method == "bands":
        keep = ((context * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(torch.float32).to(device)


def rotary(x, positions, freqs, *, interleaved: bool = False, scale: float = 1.0, out=None, stream=None):
    """Turn the first 2 len(freqs) values of each head (``[tokens, heads, head_dim]`` fp32, fp16 or
    bf16) by its token's position (int32 ``[tokens]``, any numbers): pairs (x, y) of values i and
    i + len(freqs), or 2 i and 2 i + 1 with ``interleaved``, become (x cos a - y sin a, y cos a +
    x sin a) * scale, with a = position * freqs[i]; the other values are copied.  ``out`` may be
    ``x`` itself.  Negative positions turn back (with 1 / ``scale``)."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, x):
            return rotary(x, positions, freqs, interleaved=interleaved, scale=scale, out=out)
    return _OPS.rotary(x, positions, freqs, interleaved, scale, out, _current(x))


def kv_append_rotary(q, k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, positions, freqs, *, max_q: int,
                     interleaved: bool = False, scale: float = 1.0, scores=None, out=None, stream=None):
    """kv_append with the keys turned as by ``rotary`` on their way into the cache, and the same
    tokens' queries (``[tokens, q_heads, head_dim]``, or None) turned into ``out``, which is
    returned and may be ``q`` itself.  ``positions`` None are those in the cache; a tree's are its
    first node's plus the nodes' depths.  Rows of q that are no new token's are left out."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, k_cache):
            return kv_append_rotary(q, k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, positions, freqs, max_q=max_q,
                                    interleaved=interleaved, scale=scale, scores=scores, out=out)
    return _OPS.kv_append_rotary(q, k_new, v_new, k_cache, v_cache, tables, kv_len, q_start, positions, freqs, max_q, interleaved,
                                 scale, scores, out, _current(k_cache))


def tree_attention(q, k_cache, v_cache, tables, kv_len, q_start, parents, *, max_q: int, max_kv: int, window: int = 0,
                   sinks: int = 0, scale: Optional[float] = None, out=None, lse=None, stream=None):
    """paged_attention for trees: a node sees the positions before its tree, its ancestors
    and itself; with ``window`` > 0 those of them among the last ``window`` positions of its own
    line and the first ``sinks``.  Trees have up to 512 nodes."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, q):
            return tree_attention(q, k_cache, v_cache, tables, kv_len, q_start, parents, max_q=max_q, max_kv=max_kv, window=window,
                                  sinks=sinks, scale=scale, out=out, lse=lse)
    return _OPS.tree_attention(q, k_cache, v_cache, tables, kv_len, q_start, parents, max_q, max_kv, window, sinks, scale, out, lse,
                               _current(q))


def verify_tree(target, tokens, parents, q_start, uniforms, *, max_q: int, draft=None, path=None, kept=None, token=None, stream=None):
    """Verify drafted trees against the target's probabilities (``[tokens, vocab]`` fp32, fp16 or bf16: row t
    holds those of what follows token t).  From node 0 on, each node's children are tried in order
    against ``uniforms`` (float64 ``[tokens]`` in [0, 1)): accepted with the target's probability
    over the draft's, else the rest of the target over what the draft's share leaves is tried
    further; the step's token is drawn from what is left at the last node with node 0's number.
    So tokens are distributed as the target's, as far as rows sum to 1.
    ``draft`` holds the rows that each node's children were drawn from, independently; without it the drafts are
    given, by whatever rule.  Returns (path, kept, token): the nodes of the walk, node 0 first
    (int32 ``[batch, max_q]``, -1 past them), how many they are, and the token that follows."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, target):
            return verify_tree(target, tokens, parents, q_start, uniforms, max_q=max_q, draft=draft, path=path, kept=kept, token=token)
    return _OPS.verify_tree(target, tokens, parents, q_start, uniforms, max_q, draft, path, kept, token, _current(target))


def kv_compact(k_cache, v_cache, tables, kv_len, kept, n_kept, *, q_start=None, dst_tables=None, scores=None, new_len=None, stream=None):
    """Keep chosen entries of each sequence: entry base + kept[b, i] (int32 ``[batch, n]``, the first
    n_kept[b] of them) goes, with its score, to position base + i; base is the first new token's position with
    ``q_start`` (``kept`` and ``n_kept`` are then a verify_tree's path and kept), else 0.  In place, with
    kept[b, i] >= i, as if all were read first; with ``dst_tables`` to that table's pages, which must be none that
    the call reads.  Returns the new lengths, int32 ``[batch]``; ``new_len`` is none of the inputs."""
    if _OPS is None:
        _ready()
    if stream is not None:
        with _on(stream, k_cache):
            return kv_compact(k_cache, v_cache, tables, kv_len, kept, n_kept, q_start=q_start, dst_tables=dst_tables, scores=scores,
                              new_len=new_len)
    return _OPS.kv_compact(k_cache, v_cache, tables, kv_len, kept, n_kept, q_start, dst_tables, scores, new_len, _current(k_cache))
