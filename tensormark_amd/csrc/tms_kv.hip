// tms_kv.hip -- the paged cache's own moves: new tokens written to their slots
// (tms_kv_append), and a cache cut down to the entries of the largest
// accumulated attention weight (tms_kv_evict).
#include <algorithm>

#include "tms_cache.h"
#include "tms_device.h"

namespace tms {

struct AppendParams {
    CacheView c;
    const char* k;
    const char* v;
    int64_t kt, kh, vt, vh;   // bytes between tokens, heads
    int hv, tv;               // 16-byte pieces of a head's row and of a token's
};

// A thread moves 16 bytes of a key and of a value.  Bound by latency for a
// decode step (length, table entry and data one after another), by memory for
// a prompt.
__global__ __launch_bounds__(256) void append_kernel(AppendParams a) {
    const int b = blockIdx.y;
    const SeqView sq = seq_view(a.c, b);
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const int64_t all = (int64_t)sq.n * a.tv;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < all; x += (int64_t)gridDim.x * 256) {
        const int i = (int)(x / a.tv), w = (int)(x - (int64_t)i * a.tv), h = w / a.hv, d = w - h * a.hv;
        const int64_t tok = sq.q0 + i;
        const uint4 kx = *(const uint4*)(a.k + tok * a.kt + h * a.kh + 16 * d);
        const uint4 vx = *(const uint4*)(a.v + tok * a.vt + h * a.vh + 16 * d);
        const int j = sq.p0 + i, page = page_of(a.c, row, j, sq.len);
        if (page < 0) continue;
        const int slot = j & a.c.smask;
        *(uint4*)(a.c.k + (int64_t)page * a.c.kp + h * a.c.kh + (int64_t)slot * a.c.ks + 16 * d) = kx;
        *(uint4*)(a.c.v + (int64_t)page * a.c.vp + h * a.c.vh + (int64_t)slot * a.c.vs + 16 * d) = vx;
        if (d == 0 && a.c.scores) a.c.scores[(((int64_t)page * a.c.kv_heads + h) << a.c.shift) + slot] = 0.f;
    }
}

struct EvictParams {
    CacheView c;
    const int32_t* dst;
    int64_t dstride;
    int budget, sinks, recent, max_kv;
    int32_t* new_len;
    int32_t* kept;
};

__device__ __forceinline__ int evict_len(const EvictParams& a, int b) {
    const int64_t cap = a.c.tstride << a.c.shift;
    const int L = min(max(a.c.kv_len[b], 0), a.max_kv);
    return (int)(cap < L ? cap : L);
}

// One workgroup a sequence and head: the key of the last entry kept, by a
// radix select over the scores' order keys, 8 bits a pass; then the entries
// above it and the first of those tied with it, in order, at
// sinks + above + min(tied, those that still fit).  The sinks and the last are
// kept without a look.  Where some of a sequence's positions have no page, nothing
// of it is known beforehand: all positions are gone through, those without a page below
// every key and never among the kept, the sinks and the last above every one.
//
// Entry j is thread j % 1024's.  Its keys of kBlocks blocks stay in registers,
// so that a head of up to 16384 entries reads its scores once, four blocks' loads in
// flight together (16 sequences of 1500 to 8192, 8 heads: 15 us; 29 with the scores
// read in each pass); a longer one reads them again for each pass and stretch.
constexpr int kBlocks = 16, kStretch = kBlocks * 1024;

__global__ __launch_bounds__(1024) void evict_select_kernel(EvictParams a) {
    __shared__ uint32_t hist[16][256];
    __shared__ uint32_t part[kBlocks * 16][2];   // above and tied before a block's wave
    __shared__ uint32_t total[256], pick[2], gone;
    const int b = blockIdx.x / a.c.kv_heads, h = blockIdx.x - b * a.c.kv_heads;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int L = evict_len(a, b);
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
    int lo = a.sinks, hi = L - a.recent, want = a.budget - a.sinks - a.recent;

    // A score's order key: larger is kept longer.  No number's is 0, 1 or ~0.
    uint32_t key[kBlocks];
    int page[kBlocks];
    float score[kBlocks];
    auto fetch = [&](int base) __attribute__((always_inline)) {   // four blocks' loads without a branch between them
        auto entry_of = [&](int k) { return min(base + k * 1024 + t, hi - 1); };
#pragma unroll
        for (int g = 0; g < kBlocks; g += 4)
            if (g == 0 || base + g * 1024 < hi)
#pragma unroll
                for (int k = g; k < g + 4; ++k) page[k] = row[entry_of(k) >> a.c.shift];
#pragma unroll
        for (int g = 0; g < kBlocks; g += 4)
            if (g == 0 || base + g * 1024 < hi)
#pragma unroll
                for (int k = g; k < g + 4; ++k) {
                    const int at = (unsigned)page[k] < (unsigned)a.c.pages ? page[k] : 0;
                    score[k] = a.c.scores[(((int64_t)at * a.c.kv_heads + h) << a.c.shift) + (entry_of(k) & a.c.smask)];
                }
    };
    bool holes = false;   // some positions have no page
    auto keys = [&](int base) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kBlocks; ++k)
            if (base + k * 1024 < hi) {
                key[k] = score[k] == score[k] ? okey(score[k]) : 1u;
                if (holes) {
                    const int j = base + k * 1024 + t;
                    if (j < a.sinks || j >= L - a.recent) key[k] = ~0u;
                    if ((unsigned)page[k] >= (unsigned)a.c.pages) key[k] = 0u;
                }
            }
    };
    auto load = [&](int base) __attribute__((always_inline)) {
        fetch(base);
        keys(base);
    };
    // How many positions have no page, counted while the scores are on the way.
    const int entries = (L + a.c.smask) >> a.c.shift, entry = row[min(t, max(entries - 1, 0))];
    const bool held = L > a.budget && hi - lo <= kStretch;
    if (held) fetch(lo);
    int none = t < entries && (unsigned)entry >= (unsigned)a.c.pages ? min(L - (t << a.c.shift), a.c.smask + 1) : 0;
    for (int e = t + 1024; e < entries; e += 1024)
        if ((unsigned)row[e] >= (unsigned)a.c.pages) none += min(L - (e << a.c.shift), a.c.smask + 1);
    if (t == 0) gone = 0;
    lds_sync();
    if (none) atomicAdd(&gone, (uint32_t)none);
    lds_sync();
    const int there = L - (int)gone;
    for (int64_t i = min(there, a.budget) + t; i < a.budget; i += 1024) kept[i] = -1;   // (a budget may be any: 32 bits would wrap)
    holes = there < L;
    if (holes) {
        lo = 0;
        hi = L;
        want = min(there, a.budget);
        if (want == 0) return;
        if (hi <= kStretch) load(0);
    } else {
        if (L <= a.budget) {
            for (int i = t; i < L; i += 1024) kept[i] = i;
            return;
        }
        for (int i = t; i < lo; i += 1024) kept[i] = i;
        for (int i = t; i < a.recent; i += 1024) kept[a.budget - a.recent + i] = hi + i;
        if (want == 0) return;
        if (held) keys(lo);
    }

    // Each wave counts into bins of its own, and each finds the digit from the
    // sums by itself: two barriers a pass.  Where a digit's entries are all kept,
    // the digits below need no look.
    uint32_t prefix = 0, fixed = 0;
    uint32_t left = (uint32_t)want;   // of the entries that share the prefix
    for (int i = lane; i < 256; i += 64) hist[wave][i] = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int base = lo; base < hi; base += kStretch) {
            if (hi - lo > kStretch) load(base);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                if (base + k * 1024 >= hi) break;
                if (base + k * 1024 + t < hi && (key[k] & fixed) == prefix) atomicAdd(&hist[wave][key[k] >> shift & 255], 1u);
            }
        }
        lds_sync();
        if (t < 256) {
            uint32_t n = 0;
#pragma unroll
            for (int w = 0; w < 16; ++w) n += hist[w][t];
            total[t] = n;
        }
        lds_sync();
        for (int i = lane; i < 256; i += 64) hist[wave][i] = 0;
        uint32_t n[4], mine = 0;   // the highest digit with `left` entries at or above it
        for (int i = 0; i < 4; ++i) mine += n[i] = total[255 - (4 * lane + i)];
        uint32_t upto = mine;
        for (int x = 1; x < 64; x <<= 1) {
            const uint32_t y = __shfl_up(upto, x);
            if (lane >= x) upto += y;
        }
        uint32_t above = upto - mine, digit = 0, rest = 0, alike = 0;
        bool found = false;
        for (int i = 0; i < 4; ++i) {
            if (above < left && above + n[i] >= left) {
                found = true;
                digit = 255 - (4 * lane + i);
                rest = left - above;
                alike = n[i];
            }
            above += n[i];
        }
        const int from = __ffsll((unsigned long long)__ballot(found)) - 1;
        prefix |= (uint32_t)__builtin_amdgcn_readlane(digit, from) << shift;
        fixed |= 255u << shift;
        left = __builtin_amdgcn_readlane(rest, from);
        if ((uint32_t)__builtin_amdgcn_readlane(alike, from) == left) break;
    }

    uint32_t above0 = 0, tied0 = 0;   // before the stretch
    const uint64_t before = (1ull << lane) - 1;
    for (int base = lo; base < hi; base += kStretch) {
        if (hi - lo > kStretch) load(base);
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            uint64_t up = 0, eq = 0;
            if (base + k * 1024 < hi) {
                const bool in = base + k * 1024 + t < hi;
                up = __ballot(in && (key[k] & fixed) > prefix);
                eq = __ballot(in && (key[k] & fixed) == prefix);
            }
            if (lane == 0) {
                part[k * 16 + wave][0] = __popcll(up);
                part[k * 16 + wave][1] = __popcll(eq);
            }
        }
        lds_sync();
        if (t < 64) {
            uint32_t n[4][2], sum[2] = {0, 0};
            for (int i = 0; i < 4; ++i)
                for (int c = 0; c < 2; ++c) sum[c] += n[i][c] = part[4 * t + i][c];
            for (int c = 0; c < 2; ++c) {
                uint32_t upto = sum[c];
                for (int x = 1; x < 64; x <<= 1) {
                    const uint32_t y = __shfl_up(upto, x);
                    if (lane >= x) upto += y;
                }
                if (t == 63) pick[c] = upto;
                upto -= sum[c];
                for (int i = 0; i < 4; ++i) {
                    part[4 * t + i][c] = upto;
                    upto += n[i][c];
                }
            }
        }
        lds_sync();
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            if (base + k * 1024 >= hi) break;
            const int j = base + k * 1024 + t;
            const bool in = j < hi, over = (key[k] & fixed) > prefix, tie = (key[k] & fixed) == prefix;
            const uint64_t up = __ballot(in && over), eq = __ballot(in && tie);
            const uint32_t sa = above0 + part[k * 16 + wave][0] + __popcll(up & before);
            const uint32_t st = tied0 + part[k * 16 + wave][1] + __popcll(eq & before);
            if (in && (over || (tie && st < left))) kept[lo + sa + min(st, left)] = j;
        }
        above0 += pick[0];
        tied0 += pick[1];
        lds_sync();
    }
}

// 16 bytes of a kept entry's key and value a thread, from its old slot to its
// new one; the first piece's thread moves the score too.  new_len may be the
// array kv_len: a length read here is the old or the new one, and neither is below
// the number of entries; which there are, and where they lie, is in `kept`.
__global__ __launch_bounds__(256) void evict_copy_kernel(EvictParams a, int hv) {
    const int b = blockIdx.x / a.c.kv_heads, h = blockIdx.x - b * a.c.kv_heads;
    const int n = min(evict_len(a, b), a.budget);
    const int end = (int)min(a.c.tstride << a.c.shift, (int64_t)kMaxLen);
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const int32_t* dst = a.dst + (int64_t)b * a.dstride;
    const int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
    const int last = n > 0 ? kept[n - 1] : 0;
    const int64_t all = (int64_t)n * hv;
    for (int64_t x = (int64_t)blockIdx.y * 256 + threadIdx.x; x < all; x += (int64_t)gridDim.y * 256) {
        const int i = (int)(x / hv), d = (int)(x - (int64_t)i * hv);
        const int j = kept[i], from = page_of(a.c, row, j, end), to = dst[i >> a.c.shift];
        if (from < 0 || (unsigned)to >= (unsigned)a.c.pages) continue;
        const int64_t s0 = j & a.c.smask, s1 = i & a.c.smask;
        const uint4 kx = *(const uint4*)(a.c.k + from * a.c.kp + h * a.c.kh + s0 * a.c.ks + 16 * d);
        const uint4 vx = *(const uint4*)(a.c.v + from * a.c.vp + h * a.c.vh + s0 * a.c.vs + 16 * d);
        *(uint4*)(a.c.k + to * a.c.kp + h * a.c.kh + s1 * a.c.ks + 16 * d) = kx;
        *(uint4*)(a.c.v + to * a.c.vp + h * a.c.vh + s1 * a.c.vs + 16 * d) = vx;
        if (d == 0)
            a.c.scores[(((int64_t)to * a.c.kv_heads + h) << a.c.shift) + s1] =
                a.c.scores[(((int64_t)from * a.c.kv_heads + h) << a.c.shift) + s0];
    }
    if (h == 0 && blockIdx.y == 0 && threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int from = n, upto = n;   // the number of entries, at least and at most
        if (last < 0) {
            from = 0;
            upto = n - 1;
        }
        while (from < upto) {
            const int step = (upto - from + 63) / 64, i = from + lane * step;
            const int k = __popcll(__ballot(i < upto && kept[i] >= 0));
            upto = k == 0 ? from : min(upto, from + k * step);
            from = k == 0 ? from : from + (k - 1) * step + 1;
        }
        if (lane == 0) a.new_len[b] = from;
    }
}

}  // namespace tms

extern "C" int tms_kv_append(const tms_cache* cache, const tms_append_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_cache(cache, true, true);
    if (rc != TMS_OK) return rc;
    if (!args) return TMS_ERR_INVALID_ARG;
    for (int i = 0; i < 2; ++i)
        if (args->k_new_stride[i] < 0 || args->k_new_stride[i] % 8 || args->v_new_stride[i] < 0 || args->v_new_stride[i] % 8)
            return TMS_ERR_INVALID_ARG;
    if (cache->batch > TMS_APPEND_MAX_BATCH) return TMS_ERR_CAPACITY;
    if (cache->batch == 0 || cache->tokens == 0 || cache->max_q == 0) return TMS_OK;
    if (!args->k_new || !args->v_new || !aligned16(args->k_new) || !aligned16(args->v_new)) return TMS_ERR_INVALID_ARG;
    AppendParams a;
    a.c = view_of(cache);
    a.k = (const char*)args->k_new;
    a.v = (const char*)args->v_new;
    a.kt = 2 * args->k_new_stride[0];
    a.kh = 2 * args->k_new_stride[1];
    a.vt = 2 * args->v_new_stride[0];
    a.vh = 2 * args->v_new_stride[1];
    a.hv = cache->head_dim / 8;
    a.tv = a.hv * cache->kv_heads;
    const int64_t blocks = ((int64_t)std::min(cache->max_q, cache->tokens) * a.tv + 255) / 256;
    hipLaunchKernelGGL(append_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20), cache->batch), dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}

extern "C" int tms_kv_evict(const tms_cache* cache, const tms_evict_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_cache(cache, true, false);
    if (rc != TMS_OK) return rc;
    if (!args || args->reserved != 0 || args->budget < 1 || args->sinks < 0 || args->recent < 0 ||
        (int64_t)args->sinks + args->recent > args->budget)
        return TMS_ERR_INVALID_ARG;
    if (cache->max_kv > TMS_EVICT_MAX_KV) return TMS_ERR_CAPACITY;
    if (cache->batch == 0) return TMS_OK;
    const int most = std::min(args->budget, cache->max_kv);
    if (!cache->scores || !args->dst_tables || !args->new_len || !args->kept || args->dst_table_stride < 1 ||
        args->dst_table_stride < (most + cache->page_size - 1) / cache->page_size)
        return TMS_ERR_INVALID_ARG;
    EvictParams a;
    a.c = view_of(cache);
    a.dst = args->dst_tables;
    a.dstride = args->dst_table_stride;
    a.budget = args->budget;
    a.sinks = args->sinks;
    a.recent = args->recent;
    a.max_kv = cache->max_kv;
    a.new_len = args->new_len;
    a.kept = args->kept;
    const int pairs = cache->batch * cache->kv_heads, hv = cache->head_dim / 8;
    hipLaunchKernelGGL(evict_select_kernel, dim3(pairs), dim3(1024), 0, stream, a);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(((int64_t)most * hv + 255) / 256, 65535));
    hipLaunchKernelGGL(evict_copy_kernel, dim3(pairs, (unsigned)blocks), dim3(256), 0, stream, a, hv);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
