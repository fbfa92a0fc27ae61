// tms_compact.hip -- chosen entries of each sequence of the paged cache moved to the
// front (tms_kv_compact): the accepted path of a tree of drafts, a session cut to its first
// and last positions, a copy on other pages.
//
// Bound by memory, and by latency (list, page, data, one after another) for a tree's path.
#include <algorithm>

#include "tms_cache.h"
#include "../../include/tmtree_hip.h"

namespace tms {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CompactParams {
    CacheView c;
    const int32_t* kept;
    int64_t kstride;
    const int32_t* n_kept;
    const int32_t* dst;      // null: in place
    int64_t dstride;
    int32_t* new_len;
    int max_kept;
    int hv;                  // 16-byte pieces of a head's row
    int columns, width;      // of a key's or value's row; pieces of a column
    bool apart;              // in place: keys and values by different workgroups
};

// The entries of a sequence from `base` on, `n` of them (32 bits hold every sum below:
// lengths are at most 2^29, a span of q_start too).
struct CompactSeq {
    int base, n, len;
};

__device__ __forceinline__ CompactSeq compact_seq(const CompactParams& a, int b) {
    CompactSeq s;
    const int64_t cap = a.c.tstride << a.c.shift;
    const int L = min(max(a.c.kv_len[b], 0), kMaxLen);
    s.len = (int)(cap < L ? cap : L);
    int64_t span = L;
    if (a.c.q_start) span = min(max((int64_t)a.c.q_start[b + 1] - a.c.q_start[b], (int64_t)0), (int64_t)kMaxLen);
    s.base = L - (int)span;
    s.n = min(max(a.n_kept[b], 0), a.max_kept);
    if (!a.dst) s.n = min(s.n, (int)span);
    return s;
}

// Page and slot of entry i of the list, -1 where it is not moved.
__device__ __forceinline__ void compact_from(const CompactParams& a, const CompactSeq& s, const int32_t* row, int i, int kept, int& page, int& slot) {
    const int j = s.base + kept;
    page = (unsigned)kept < (unsigned)kMaxLen && (a.dst || kept > i) ? page_of(a.c, row, j, s.len) : -1;   // (kept == i stays)
    slot = j & a.c.smask;
}

__device__ __forceinline__ void compact_to(const CompactParams& a, const int32_t* row, int64_t stride, int j, int& page, int& slot) {
    const bool in = j >= 0 && (j >> a.c.shift) < stride;
    const int p = row[in ? j >> a.c.shift : 0];
    page = in && (unsigned)p < (unsigned)a.c.pages ? p : -1;
    slot = j & a.c.smask;
}

// To other pages: a thread moves 16 bytes of a key and of a value of two entries, all on the way
// together.  Stores past the caches: what is copied is read next after much else (8 sequences of 500 to
// 4001, 8 heads of 128, 149 MB: 31 us, 4.8 TB/s; 36.7 with ordinary stores, 39.8 with four entries).
__global__ __launch_bounds__(256) void compact_copy_kernel(CompactParams a) {
    constexpr int UN = 2;
    const int b = blockIdx.x / a.c.kv_heads, h = blockIdx.x - b * a.c.kv_heads;
    const CompactSeq s = compact_seq(a, b);
    if (a.new_len && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.new_len[b] = max(s.base + s.n, 0);
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const int32_t* dst = a.dst + (int64_t)b * a.dstride;
    const int32_t* kept = a.kept + (int64_t)b * a.kstride;
    char* const kh = a.c.k + h * a.c.kh;
    char* const vh = a.c.v + h * a.c.vh;
    float* const scores = a.c.scores ? a.c.scores + ((int64_t)h << a.c.shift) : nullptr;
    const int64_t all = (int64_t)s.n * a.hv, sp = (int64_t)a.c.kv_heads << a.c.shift;
    for (int64_t x0 = (int64_t)blockIdx.y * 256 * UN; x0 < all; x0 += (int64_t)gridDim.y * 256 * UN) {
        int from[UN], to[UN], s0[UN], s1[UN], d[UN];
        u32x4 kx[UN], vx[UN];
        float sc[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int64_t x = x0 + u * 256 + threadIdx.x, in = min(x, all - 1);
            const int i = (int)(in / a.hv);
            d[u] = (int)(in - (int64_t)i * a.hv);
            compact_from(a, s, row, i, kept[i], from[u], s0[u]);
            compact_to(a, dst, a.dstride, s.base + i, to[u], s1[u]);
            if (x >= all || to[u] < 0) from[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (from[u] >= 0) {
                kx[u] = *(const u32x4*)(kh + from[u] * a.c.kp + s0[u] * a.c.ks + 16 * d[u]);
                vx[u] = *(const u32x4*)(vh + from[u] * a.c.vp + s0[u] * a.c.vs + 16 * d[u]);
                if (d[u] == 0 && scores) sc[u] = scores[from[u] * sp + s0[u]];
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (from[u] >= 0) {
                __builtin_nontemporal_store(kx[u], (u32x4*)(kh + to[u] * a.c.kp + s1[u] * a.c.ks + 16 * d[u]));
                __builtin_nontemporal_store(vx[u], (u32x4*)(vh + to[u] * a.c.vp + s1[u] * a.c.vs + 16 * d[u]));
                if (d[u] == 0 && scores) scores[to[u] * sp + s1[u]] = sc[u];
            }
    }
}

// In place: entry i's place is some earlier entry's source or nobody's, never a later one's
// (those have kept > i), so a list may be gone through from its start: a step's entries are
// read, and once all of the workgroup's are in, written.  Only a step's own entries can meet;
// rows are independent by head and by 16 bytes, so long lists are spread over
// workgroups by those: key or value, 128 bytes (16 sequences of 4600 to 8192 to 2200 entries, 8 heads of 128,
// 291 MB: 65 us, 4.5 TB/s; 70 with ordinary loads and stores, 76 with whole rows of 256 bytes, 80 with
// twice the entries a step, which leaves one workgroup a CU).
template <int NT, int UN, bool LONG>
__global__ __launch_bounds__(NT) void compact_place_kernel(CompactParams a) {
    const int b = blockIdx.x / a.c.kv_heads, h = blockIdx.x - b * a.c.kv_heads;
    const CompactSeq s = compact_seq(a, b);
    const int t = threadIdx.x;
    const int part = blockIdx.y, column = part % a.columns;
    if (a.new_len && h == 0 && part == 0 && t == 0) a.new_len[b] = max(s.base + s.n, 0);
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const int32_t* kept = a.kept + (int64_t)b * a.kstride;
    // The thread's piece: of a key or a value, and which of a step's entries.
    const int wide = min(a.width, a.hv - column * a.width), pieces = a.apart ? wide : 2 * wide;
    const int entries = NT / pieces, e0 = t / pieces, p = t - e0 * pieces;
    const bool value = a.apart ? part >= a.columns : p >= wide;
    const int d = column * a.width + (p >= wide ? p - wide : p);
    const bool score = a.c.scores && !value && d == 0;
    char* const pool = (value ? a.c.v + h * a.c.vh : a.c.k + h * a.c.kh) + 16 * d;
    const int64_t pstride = value ? a.c.vp : a.c.kp, sstride = value ? a.c.vs : a.c.ks;
    // A step's entries, read while the step before is written: that one lies below all of them.
    struct Step {
        u32x4 x[UN];
        float sc[UN];
        int from[UN], to[UN], s0[UN], s1[UN];
    };
    auto read = [&](int i0, Step& p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int i = i0 + u * entries + e0, at = min(i, s.n - 1);
            compact_from(a, s, row, at, kept[at], p.from[u], p.s0[u]);
            compact_to(a, row, a.c.tstride, s.base + at, p.to[u], p.s1[u]);
            if (e0 >= entries || i >= s.n || p.to[u] < 0) p.from[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            p.x[u] = (u32x4){0, 0, 0, 0};
            p.sc[u] = 0.f;
            if (p.from[u] >= 0) {
                const u32x4* at = (const u32x4*)(pool + p.from[u] * pstride + p.s0[u] * sstride);
                p.x[u] = LONG ? __builtin_nontemporal_load(at) : *at;
                if (score) p.sc[u] = a.c.scores[(((int64_t)p.from[u] * a.c.kv_heads + h) << a.c.shift) + p.s0[u]];
            }
        }
    };
    auto write = [&](const Step& p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (p.from[u] >= 0) {
                u32x4* at = (u32x4*)(pool + p.to[u] * pstride + p.s1[u] * sstride);
                if (LONG) __builtin_nontemporal_store(p.x[u], at);
                else *at = p.x[u];
                if (score) a.c.scores[(((int64_t)p.to[u] * a.c.kv_heads + h) << a.c.shift) + p.s1[u]] = p.sc[u];
            }
    };
    // All of a step is in registers, in every wave, before any of it is written.
    auto all_in = [&](const Step& p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < UN; ++u) asm volatile("" ::"v"(p.x[u]), "v"(p.sc[u]) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    const int step = entries * UN;
    if (s.n <= 0) return;
    Step now, next;
    read(0, now);
    for (int i0 = 0;;) {
        all_in(now);
        i0 += step;
        if (i0 < s.n) read(i0, next);
        write(now);
        if (i0 >= s.n) return;
        now = next;
    }
}

}  // namespace tms

extern "C" int tms_kv_compact(const tms_cache* cache, const tms_compact_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_cache(cache, true, false);
    if (rc != TMS_OK) return rc;
    if (!args || args->reserved != 0 || args->max_kept < 0) return TMS_ERR_INVALID_ARG;
    if (args->max_kept > TMS_COMPACT_MAX_KEPT) return TMS_ERR_CAPACITY;
    if (cache->batch == 0) return TMS_OK;
    if (!args->n_kept || (args->max_kept > 0 && !args->kept) || args->kept_stride < args->max_kept) return TMS_ERR_INVALID_ARG;
    if (args->dst_tables && (args->dst_table_stride < 1 || args->dst_tables == cache->tables)) return TMS_ERR_INVALID_ARG;
    if (args->new_len && (args->new_len == cache->kv_len || args->new_len == args->n_kept || args->new_len == args->kept))
        return TMS_ERR_INVALID_ARG;
    if (cache->k == cache->v) return TMS_ERR_INVALID_ARG;
    CompactParams a{};
    a.c = view_of(cache);
    a.kept = args->kept;
    a.kstride = args->kept_stride;
    a.n_kept = args->n_kept;
    a.dst = args->dst_tables;
    a.dstride = args->dst_table_stride;
    a.new_len = args->new_len;
    a.max_kept = args->max_kept;
    a.hv = cache->head_dim / 8;
    const int pairs = cache->batch * cache->kv_heads;
    if (a.dst) {
        const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(((int64_t)a.max_kept * a.hv + 511) / 512, 65535));
        hipLaunchKernelGGL(compact_copy_kernel, dim3(pairs, (unsigned)blocks), dim3(256), 0, stream, a);
    } else if (a.max_kept <= 64) {
        a.columns = 1;
        a.width = a.hv;
        a.apart = false;
        hipLaunchKernelGGL((compact_place_kernel<256, 1, false>), dim3(pairs, 1), dim3(256), 0, stream, a);
    } else {
        a.width = std::min(a.hv, 8);
        a.columns = (a.hv + a.width - 1) / a.width;
        a.apart = true;
        hipLaunchKernelGGL((compact_place_kernel<1024, 2, true>), dim3(pairs, 2 * a.columns), dim3(1024), 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
