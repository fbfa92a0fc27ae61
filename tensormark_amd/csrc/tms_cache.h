// tms_cache.h -- the paged cache as the kernels see it, and the host checks
// of a tms_cache that its entry points share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tmcache_hip.h"

namespace tms {

constexpr int kMaxLen = 1 << 29;   // positions of a sequence, and a window: sums of three fit 32 bits

struct CacheView {
    char* k;
    char* v;
    float* scores;
    int64_t kp, kh, ks;   // bytes between pages, heads, slots
    int64_t vp, vh, vs;
    const int32_t* tables;
    int64_t tstride;
    const int32_t* kv_len;
    const int32_t* q_start;
    int pages, kv_heads, head_dim, batch, tokens, max_q;
    int shift, smask;     // log2 and mask of the page size
};

// A sequence of the call: its new tokens [q0, q0 + n) stand at positions
// p0.. of the cache, whose mapped positions are below `len`.  Lengths and
// offsets are device data: what does not fit the tensors is cut here, so no
// value of theirs leads a kernel out of range.
struct SeqView {
    int q0, n, p0, len;
};

__device__ __forceinline__ SeqView seq_view(const CacheView& c, int b) {
    SeqView s;
    const int64_t cap = c.tstride << c.shift;
    const int L = min(max(c.kv_len[b], 0), kMaxLen);
    s.len = (int)(cap < L ? cap : L);
    const int a = c.q_start[b], e = c.q_start[b + 1];
    s.q0 = min(max(a, 0), c.tokens);
    const int q1 = min(max(e, s.q0), c.tokens);
    s.n = min(q1 - s.q0, c.max_q);
    s.p0 = L - (q1 - s.q0);
    return s;
}

// Page of position j of the table row, -1 where j does not exist or the
// entry names no page.
__device__ __forceinline__ int page_of(const CacheView& c, const int32_t* row, int j, int len) {
    if ((unsigned)j >= (unsigned)len) return -1;
    const int p = row[j >> c.shift];
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// TMS_OK, or what the entry points answer for this cache.
inline int check_cache(const tms_cache* c, bool need_v, bool need_q) {
    if (!c || c->reserved != 0) return TMS_ERR_INVALID_ARG;
    if (c->dtype != TMS_DTYPE_F16 && c->dtype != TMS_DTYPE_BF16) return TMS_ERR_INVALID_ARG;
    if (!c->k || !aligned16(c->k) || (need_v && (!c->v || !aligned16(c->v)))) return TMS_ERR_INVALID_ARG;
    if ((uintptr_t)c->scores & 15) return TMS_ERR_INVALID_ARG;
    if (c->pages < 1 || c->kv_heads < 1 || c->batch < 0 || c->tokens < 0 || c->max_q < 0 || c->max_kv < 0)
        return TMS_ERR_INVALID_ARG;
    if (c->page_size < TMS_CACHE_MIN_PAGE || c->page_size > TMS_CACHE_MAX_PAGE || (c->page_size & (c->page_size - 1)))
        return TMS_ERR_INVALID_ARG;
    if (c->head_dim < 8 || c->head_dim > TMS_CACHE_MAX_HEAD_DIM || c->head_dim % 8) return TMS_ERR_INVALID_ARG;
    for (int i = 0; i < 3; ++i) {
        if (c->k_stride[i] < 0 || c->k_stride[i] % 8) return TMS_ERR_INVALID_ARG;
        if (need_v && (c->v_stride[i] < 0 || c->v_stride[i] % 8)) return TMS_ERR_INVALID_ARG;
    }
    if (c->batch > 0 && (!c->tables || c->table_stride < 1 || !c->kv_len || (need_q && !c->q_start)))
        return TMS_ERR_INVALID_ARG;
    if ((int64_t)c->batch * c->kv_heads > TMS_CACHE_MAX_PAIRS || c->tokens > TMS_CACHE_MAX_TOKENS) return TMS_ERR_CAPACITY;
    return TMS_OK;
}

inline CacheView view_of(const tms_cache* c) {
    CacheView w;
    w.k = (char*)c->k;
    w.v = (char*)c->v;
    w.scores = c->scores;
    w.kp = 2 * c->k_stride[0];
    w.kh = 2 * c->k_stride[1];
    w.ks = 2 * c->k_stride[2];
    w.vp = 2 * c->v_stride[0];
    w.vh = 2 * c->v_stride[1];
    w.vs = 2 * c->v_stride[2];
    w.tables = c->tables;
    w.tstride = c->table_stride;
    w.kv_len = c->kv_len;
    w.q_start = c->q_start;
    w.pages = c->pages;
    w.kv_heads = c->kv_heads;
    w.head_dim = c->head_dim;
    w.batch = c->batch;
    w.tokens = c->tokens;
    w.max_q = c->max_q;
    w.shift = __builtin_ctz((unsigned)c->page_size);
    w.smask = c->page_size - 1;
    return w;
}

}  // namespace tms
