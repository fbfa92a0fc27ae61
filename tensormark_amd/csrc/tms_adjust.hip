// tms_adjust.hip -- the logits rules as an operator of their own
// (tms_adjust_logits): mask, penalties and biases on rows that are sampled
// elsewhere or go to the speculative verify.
//
// Bound by memory: a row is read once and written once.  Of its ids only those
// of the history and of the bias list change otherwise than by the mask, some
// hundreds among 100,000 and more.  A workgroup takes kAdjChunk ids of a row
// at a time: while their logits are on the way it puts those ids into a list
// and a bitmap in LDS, their counts and biases into words of their own (read
// for ids of the list alone, so nothing is cleared but the bitmap), and works
// each id out in a thread; the vectors then only take the results.  (Worked out
// where the vector lies, a wave went through its ids one after another: 288
// rows of 128256 bf16 in 72 us.)
#include <algorithm>

#include "tms_device.h"
#include "../../include/tmcache_hip.h"
#include "tms_sample_common.h"

namespace tms {

constexpr uint32_t kBiasHeld = 512;
// Ids at a time: 8 KiB each of counts and biases, seven workgroups a CU (288 rows
// of 128256 bf16, other ones each time: 46 us; 63 with 4096 and three workgroups).
constexpr int kAdjChunk = 2048;

struct AdjustParams {
    const char* x;
    char* y;
    int steps, vocab, n_bias;
    int subs;         // chunks a workgroup
    int64_t xs, ys;   // elements between rows
    const tms_row_params* params;
    const int32_t* recent;
    const int32_t* n_recent;
    int64_t rstride;
    int history;
    const int32_t* drafts;
    const int32_t* bias_ids;
    const float* bias_values;
    const uint32_t* mask;
    int64_t mstride;
};

template <typename T> struct Widen;
template <> struct Widen<float> {
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Widen<_Float16> {
    static __device__ __forceinline__ float up(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <> struct Widen<__bf16> {
    static __device__ __forceinline__ float up(__bf16 x) { return (float)x; }
    static __device__ __forceinline__ __bf16 down(float x) { return (__bf16)x; }
};

// Rows may begin at any element: vectors are moved without an alignment of
// their own (the memory system takes them at any address).
template <typename T> struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A workgroup takes `subs` chunks of a row one after another, the next one's
// logits on the way meanwhile, and keeps the first kHist ids of the history and
// the first kBias biases of a thread in registers.
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void adjust_kernel(AdjustParams a) {
    constexpr int VEC = Vec16<TI>::N, NV = kAdjChunk / (256 * VEC), kHist = 4, kBias = 2;
    typedef typename Vec16<TI>::type In;
    typedef TO Out __attribute__((ext_vector_type(VEC), aligned(sizeof(TO))));
    __shared__ uint32_t touched[2][kAdjChunk / 32];
    __shared__ uint32_t cnt[kAdjChunk];    // an id's count, then its result
    __shared__ uint32_t bias[kAdjChunk];   // the bias list's first entry for the id
    __shared__ float value[kBiasHeld];     // the first entries' values
    __shared__ uint16_t list[kAdjChunk];   // the ids that the chunk has
    __shared__ uint32_t listed[2];
    __shared__ int twice;
    const float low = -__builtin_huge_valf();
    const int t = threadIdx.x;
    const int r = blockIdx.y, seq = r / a.steps, step = r - seq * a.steps;
    const TI* row_in = (const TI*)a.x + (int64_t)r * a.xs;
    TO* row_out = (TO*)a.y + (int64_t)r * a.ys;
    const uint32_t* mrow = a.mask ? a.mask + (int64_t)r * a.mstride : nullptr;
    In v[NV];
    uint32_t word[NV];
    auto load = [&](int c0) __attribute__((always_inline)) {   // a whole chunk
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = *(const In*)(row_in + c0 + (k * 256 + t) * VEC);
        if (mrow) {
#pragma unroll
            for (int k = 0; k < NV; ++k) word[k] = mrow[(c0 + (k * 256 + t) * VEC) >> 5];
        }
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) word[k] = ~0u;
    const int first = blockIdx.x * a.subs * kAdjChunk, last = min(first + a.subs * kAdjChunk, a.vocab);
    if (first + kAdjChunk <= a.vocab) load(first);

    Pen pn;
    pn.on = pn.rep_on = pn.fp_on = false;
    pn.rep = pn.freq = pn.pres = 0.f;
    int from = 0, have = 0, total = 0;   // the window: [from, total) of the row's history
    if (a.params) {
        const tms_row_params& P = a.params[seq];
        pn.rep_on = !(P.repeat_penalty <= 1.0f);
        pn.fp_on = P.frequency_penalty != 0.f || P.presence_penalty != 0.f;
        pn.rep = P.repeat_penalty;
        pn.freq = P.frequency_penalty;
        pn.pres = P.presence_penalty;
        if (a.recent) have = min(max(a.n_recent ? a.n_recent[seq] : a.history, 0), a.history);
        total = have + (a.drafts ? step : 0);
        pn.on = total > 0 && P.repeat_last_n > 0 && (pn.rep_on || pn.fp_on);
        from = total > P.repeat_last_n ? total - P.repeat_last_n : 0;
    }
    if (!pn.on) from = total;
    const int32_t* recent = a.recent + (int64_t)seq * a.rstride;
    const int32_t* drafts = a.drafts + (int64_t)seq * (a.steps - 1);
    const int32_t* bid = a.bias_ids + (int64_t)seq * a.n_bias;
    const float* bval = a.bias_values + (int64_t)seq * a.n_bias;
    auto hist = [&](int i) { return *(i < have ? recent + i : drafts + (i - have)); };
    int hid[kHist], bidr[kBias];   // -1: none (no id of a chunk)
#pragma unroll
    for (int k = 0; k < kBias; ++k) {
        const int i = k * 256 + t;
        bidr[k] = -1;
        if (i < a.n_bias) {
            bidr[k] = bid[i];
            if (i < (int)kBiasHeld) value[i] = bval[i];
        }
    }
#pragma unroll
    for (int k = 0; k < kHist; ++k) {
        const int i = from + k * 256 + t;
        hid[k] = -1;
        if (i < total) hid[k] = hist(i);
    }
    // f(id, entry) of every id of the window (entry -1) and of the bias list.
    auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kHist; ++k) f(hid[k], -1);
        for (int i = from + kHist * 256 + t; i < total; i += 256) f(hist(i), -1);
#pragma unroll
        for (int k = 0; k < kBias; ++k) f(bidr[k], k * 256 + t);
        for (int i = kBias * 256 + t; i < a.n_bias; i += 256) f(bid[i], i);
    };

    for (int i = t; i < 2 * kAdjChunk / 32; i += 256) (&touched[0][0])[i] = 0;
    if (t == 0) twice = listed[0] = listed[1] = 0;
    int which = 0;
    for (int c0 = first; c0 < last; c0 += kAdjChunk, which ^= 1) {
        const int n = min(kAdjChunk, a.vocab - c0);
        uint32_t* const set = touched[which];
        lds_sync();
        each([&](int id, int) {
            const uint32_t at = (uint32_t)id - (uint32_t)c0;
            if (at < (uint32_t)n) {
                cnt[at] = 0;
                bias[at] = ~0u;
                const uint32_t bit = 1u << (at & 31);
                if (!(atomicOr(&set[at >> 5], bit) & bit)) list[atomicAdd(&listed[which], 1u)] = (uint16_t)at;
            }
        });
        lds_sync();
        // A thread has an id to work out; its logit is on the way during the counts.
        const int ids = (int)listed[which];
        TI x = (TI)0.f;
        if (t < ids) x = row_in[c0 + list[t]];
        each([&](int id, int entry) {
            const uint32_t at = (uint32_t)id - (uint32_t)c0;
            if (at >= (uint32_t)n) return;
            if (entry < 0) atomicAdd(&cnt[at], 1u);
            else if (atomicMin(&bias[at], (uint32_t)entry) != ~0u) twice = 1;   // (most lists name an id once)
        });
        if (t < kAdjChunk / 32) touched[which ^ 1][t] = 0;
        if (t == 0) listed[which ^ 1] = 0;
        lds_sync();
        for (int l = t; l < ids; l += 256) {
            const int id = list[l];
            if (l != t) x = row_in[c0 + id];
            float f = Widen<TI>::up(x);
            const uint32_t c = cnt[id];
            if (c) f = apply_pen<true>(f, c, pn);
            const uint32_t head = bias[id];
            if (head != ~0u) {
                float sum = head < kBiasHeld ? value[head] : bval[head];
                if (twice)
                    for (int i = (int)head + 1; i < a.n_bias; ++i)
                        if (bid[i] - c0 == id) sum += bval[i];
                f += sum;
            }
            cnt[id] = __float_as_uint(f);
        }
        lds_sync();
        if (n < kAdjChunk) {   // the row's last, element by element
            for (int i = t; i < n; i += 256) {
                float f = set[i >> 5] >> (i & 31) & 1 ? __uint_as_float(cnt[i]) : Widen<TI>::up(row_in[c0 + i]);
                if (mrow && !(mrow[(c0 + i) >> 5] >> (i & 31) & 1)) f = low;
                row_out[c0 + i] = Widen<TO>::down(f);
            }
            break;
        }
        In now[NV];
        uint32_t allow[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            now[k] = v[k];
            allow[k] = word[k] >> ((k * 256 + t) * VEC & 31);
        }
        if (c0 + 2 * kAdjChunk <= a.vocab && c0 + kAdjChunk < last) load(c0 + kAdjChunk);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int i = (k * 256 + t) * VEC;
            const uint32_t hit = set[i >> 5] >> (i & 31) & ((1u << VEC) - 1) & allow[k];
            Out o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = Widen<TO>::down(allow[k] >> e & 1 ? Widen<TI>::up(now[k][e]) : low);
            if (hit) {
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (hit >> e & 1) o[e] = Widen<TO>::down(__uint_as_float(cnt[i + e]));
            }
            *(Out*)(row_out + c0 + i) = o;
        }
    }
}

}  // namespace tms

extern "C" int tms_adjust_logits(const tms_adjust_args* args, hipStream_t stream) {
    using namespace tms;
    if (!args) return TMS_ERR_INVALID_ARG;
    const tms_adjust_args& p = *args;
    if (p.dtype < TMS_DTYPE_F32 || p.dtype > TMS_DTYPE_BF16 || (p.out_dtype != p.dtype && p.out_dtype != TMS_DTYPE_F32))
        return TMS_ERR_INVALID_ARG;
    if (p.seqs < 0 || p.steps < 1 || p.vocab < 1 || p.n_bias < 0 || p.row_stride < p.vocab || p.out_stride < p.vocab ||
        p.n_history < 0 || p.recent_stride < p.n_history || p.reserved != 0)
        return TMS_ERR_INVALID_ARG;
    const int64_t rows = (int64_t)p.seqs * p.steps;
    if (p.vocab > 1048576 || p.n_bias > 65535 || rows > 65535 || p.n_history > (1 << 28)) return TMS_ERR_CAPACITY;
    if (rows == 0) return TMS_OK;
    if (!p.logits || !p.out || (p.n_bias && (!p.bias_ids || !p.bias_values)) ||
        (p.mask && p.mask_stride < (p.vocab + 31) / 32))
        return TMS_ERR_INVALID_ARG;
    if (p.out == p.logits && (p.out_dtype != p.dtype || p.out_stride != p.row_stride)) return TMS_ERR_INVALID_ARG;
    const int esz = p.dtype == TMS_DTYPE_F32 ? 4 : 2, osz = p.out_dtype == TMS_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)p.logits % esz || (uintptr_t)p.out % osz) return TMS_ERR_INVALID_ARG;
    AdjustParams a;
    a.x = (const char*)p.logits;
    a.y = (char*)p.out;
    a.steps = p.steps;
    a.vocab = p.vocab;
    a.n_bias = p.n_bias;
    a.xs = p.row_stride;
    a.ys = p.out_stride;
    a.params = p.params;
    a.recent = p.recent;
    a.n_recent = p.n_recent;
    a.rstride = p.recent_stride;
    a.history = p.n_history;
    a.drafts = p.drafts;
    a.bias_ids = p.bias_ids;
    a.bias_values = p.bias_values;
    a.mask = p.mask;
    a.mstride = p.mask_stride;
    // Chunks a workgroup: as many as leave some two rounds of the 1792 workgroups
    // that the card holds (288 rows of 128256 bf16, other ones each time: 46 us with 4096
    // workgroups, 50 with 1024, 54 with 8192, 58 with one a chunk).
    const int chunks = (p.vocab + kAdjChunk - 1) / kAdjChunk;
    a.subs = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, rows * chunks / 4096));
    const dim3 grid((chunks + a.subs - 1) / a.subs, (unsigned)rows);
    const bool wide = p.out_dtype == TMS_DTYPE_F32;
    if (p.dtype == TMS_DTYPE_F32) hipLaunchKernelGGL((adjust_kernel<float, float>), grid, dim3(256), 0, stream, a);
    else if (p.dtype == TMS_DTYPE_F16 && wide) hipLaunchKernelGGL((adjust_kernel<_Float16, float>), grid, dim3(256), 0, stream, a);
    else if (p.dtype == TMS_DTYPE_F16) hipLaunchKernelGGL((adjust_kernel<_Float16, _Float16>), grid, dim3(256), 0, stream, a);
    else if (wide) hipLaunchKernelGGL((adjust_kernel<__bf16, float>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((adjust_kernel<__bf16, __bf16>), grid, dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
