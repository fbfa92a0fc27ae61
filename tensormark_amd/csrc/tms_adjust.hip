// tms_adjust.hip -- the logits rules as an operator of their own
// (tms_adjust_logits): mask, penalties and biases on rows that are sampled
// elsewhere or go to the speculative verify.
//
// Bound by memory: a row is read once and written once.  Of its ids only those
// of the history and of the bias list change otherwise than by the mask, some
// hundreds among 100,000 and more.  A workgroup takes kChunk ids of a row, and
// while its logits are on the way puts those ids' counts and biases into LDS,
// one word each per id of the chunk; a bitmap says which words were set (the
// others are never read, so nothing is cleared but the bitmap).
#include <algorithm>

#include "tms_device.h"
#include "../../include/tmcache_hip.h"
#include "tms_sample_common.h"

namespace tms {

constexpr uint32_t kBiasHeld = 512;
constexpr int kAdjChunk = 4096;   // ids a workgroup: 16 KiB each of counts and biases, four workgroups a CU

struct AdjustParams {
    const char* x;
    char* y;
    int steps, vocab, n_bias;
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
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void adjust_kernel(AdjustParams a) {
    constexpr int VEC = 16 / sizeof(TI), NV = kAdjChunk / (256 * VEC);
    struct In { TI x[VEC]; };
    struct Out { TO x[VEC]; };
    __shared__ uint32_t touched[kAdjChunk / 32];
    __shared__ uint32_t cnt[kAdjChunk];
    __shared__ uint32_t bias[kAdjChunk];   // the list's first entry for the id
    __shared__ float value[kBiasHeld];     // the first entries' values
    __shared__ int twice;
    const int t = threadIdx.x;
    const int r = blockIdx.y, seq = r / a.steps, step = r - seq * a.steps;
    const int c0 = blockIdx.x * kAdjChunk, n = min(kAdjChunk, a.vocab - c0);
    const TI* x = (const TI*)a.x + (int64_t)r * a.xs + c0;
    TO* y = (TO*)a.y + (int64_t)r * a.ys + c0;
    In v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = (k * 256 + t) * VEC;
        if (i + VEC <= n) __builtin_memcpy(&v[k], x + i, sizeof(In));
        else
            for (int e = 0; e < VEC; ++e) v[k].x[e] = i + e < n ? x[i + e] : (TI)0.f;
    }

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
    auto hist = [&](int i) { return (i < have ? recent[i] : drafts[i - have]) - c0; };

    if (t < kAdjChunk / 32) touched[t] = 0;
    if (t == 0) twice = 0;
    __syncthreads();
    for (int i = from + t; i < total; i += 256) {
        const int id = hist(i);
        if ((unsigned)id < (unsigned)n) {
            cnt[id] = 0;
            bias[id] = ~0u;
            atomicOr(&touched[id >> 5], 1u << (id & 31));
        }
    }
    for (int i = t; i < a.n_bias; i += 256) {
        const int id = bid[i] - c0;
        if (i < (int)kBiasHeld) value[i] = bval[i];
        if ((unsigned)id < (unsigned)n) {
            cnt[id] = 0;
            bias[id] = ~0u;
            atomicOr(&touched[id >> 5], 1u << (id & 31));
        }
    }
    __syncthreads();
    for (int i = from + t; i < total; i += 256) {
        const int id = hist(i);
        if ((unsigned)id < (unsigned)n) atomicAdd(&cnt[id], 1u);
    }
    for (int i = t; i < a.n_bias; i += 256) {
        const int id = bid[i] - c0;
        if ((unsigned)id < (unsigned)n) atomicMin(&bias[id], (uint32_t)i);
    }
    __syncthreads();
    for (int i = t; i < a.n_bias; i += 256) {
        const int id = bid[i] - c0;
        if ((unsigned)id < (unsigned)n && bias[id] != (uint32_t)i) twice = 1;
    }
    __syncthreads();
    const bool again = twice != 0;

#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int i = (k * 256 + t) * VEC;
        if (i >= n) break;
        const uint32_t hit = touched[i >> 5] >> (i & 31) & ((1u << VEC) - 1);
        const uint32_t allow = a.mask ? a.mask[(int64_t)r * a.mstride + ((c0 + i) >> 5)] >> ((c0 + i) & 31) : ~0u;
        Out o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float f = Widen<TI>::up(v[k].x[e]);
            if (hit >> e & 1) {
                const uint32_t c = cnt[i + e];
                if (c) f = apply_pen<true>(f, c, pn);
                const uint32_t first = bias[i + e];
                if (first != ~0u) {
                    float sum = first < kBiasHeld ? value[first] : bval[first];
                    if (again)   // (most lists name an id once)
                        for (int l = (int)first + 1; l < a.n_bias; ++l)
                            if (bid[l] - c0 == i + e) sum += bval[l];
                    f += sum;
                }
            }
            o.x[e] = Widen<TO>::down(allow >> e & 1 ? f : -__builtin_huge_valf());
        }
        if (i + VEC <= n) __builtin_memcpy(y + i, &o, sizeof(Out));
        else
            for (int e = 0; e < VEC; ++e)
                if (i + e < n) y[i + e] = o.x[e];
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
    const dim3 grid((p.vocab + kAdjChunk - 1) / kAdjChunk, (unsigned)rows);
    const bool wide = p.out_dtype == TMS_DTYPE_F32;
    if (p.dtype == TMS_DTYPE_F32) hipLaunchKernelGGL((adjust_kernel<float, float>), grid, dim3(256), 0, stream, a);
    else if (p.dtype == TMS_DTYPE_F16 && wide) hipLaunchKernelGGL((adjust_kernel<_Float16, float>), grid, dim3(256), 0, stream, a);
    else if (p.dtype == TMS_DTYPE_F16) hipLaunchKernelGGL((adjust_kernel<_Float16, _Float16>), grid, dim3(256), 0, stream, a);
    else if (wide) hipLaunchKernelGGL((adjust_kernel<__bf16, float>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((adjust_kernel<__bf16, __bf16>), grid, dim3(256), 0, stream, a);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
