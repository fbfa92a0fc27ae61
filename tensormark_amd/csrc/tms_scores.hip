// tms_scores.hip -- the attention weight that new tokens give to each cached
// key (tms_kv_add_scores): score[j] += sum over rows of 2^(s_j - lse), with
// s and lse to base 2.  One matrix product, S^T = K Q^T, and no exchange
// between workgroups: a wave keeps its keys in registers and passes over the
// rows that see them, so a key's sum is one lane group's, in row order.
#include <algorithm>
#include <cmath>

#include "tms_attn.h"

namespace tms {

// Each of the four waves takes 16 * KT keys of one key head; a lane holds one
// row's scores (row = lane % 16) of 4 * KT keys and sums weights over the
// rows' tiles; the 16 rows' sums are joined once at the end.
template <typename T, int KS, int KT>
__global__ __launch_bounds__(256) void score_kernel(AttnParams a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n16 = lane & 15, g4 = lane >> 4;
    const int pair = blockIdx.x, b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    const SeqView sq = seq_view(a.c, b);
    const int t0 = (blockIdx.y * 4 + wave) * (16 * KT);
    if (t0 >= sq.len) return;
    const int G = a.group, rows = sq.n * G, D = a.c.head_dim;
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const char* kbase = a.c.k + (int64_t)h * a.c.kh;

    u32x4 kr[KT][KS];
    int vp[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int j = t0 + 16 * kt + n16;
        const int page = page_of(a.c, row, j, sq.len);
        vp[kt] = page_of(a.c, row, t0 + 16 * kt + 4 * g4, sq.len);
        const char* src = kbase + (page < 0 ? 0 : (int64_t)page * a.c.kp + (int64_t)(j & a.c.smask) * a.c.ks);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 32 + g4 * 8;
            kr[kt][s] = d < D ? *(const u32x4*)(src + 2 * d) : (u32x4){0, 0, 0, 0};
        }
    }
    f32x4 sum[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) sum[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // Rows that see a key of the wave's: from the first at or past its first
    // key to the last whose window still reaches its last key.
    const int t1 = min(t0 + 16 * KT, sq.len) - 1;
    int first = min(max(t0 - sq.p0, 0), sq.n), last = sq.n - 1;
    if (a.window > 0 && t0 >= a.sinks) last = min(last, t1 - sq.p0 + a.window - 1);
    for (int r = first * G / 16 * 16; r <= last * G + G - 1; r += 16) {
        const int rr = r + n16;
        const bool in = rr < rows;
        const int tok = in ? rr / G : 0, hd = in ? rr - tok * G : 0;
        const int pos = in ? sq.p0 + tok : -1;
        const char* src = a.q + (int64_t)(sq.q0 + tok) * a.qt + (int64_t)(h * G + hd) * a.qh;
        float lse = in ? a.lse[(int64_t)(sq.q0 + tok) * a.q_heads + h * G + hd] * kLog2e : 0.f;
        if (lse == -__builtin_huge_valf()) lse = -lse;   // the row saw nothing: no weight
        u32x4 qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 32 + g4 * 8;
            qf[s] = in && d < D ? (*(const u32x4*)(src + 2 * d) & a.qand) ^ a.qxor : (u32x4){0, 0, 0, 0};
        }
        const int pfirst = sq.p0 + r / G, plast = sq.p0 + (r + 15) / G;
        const bool edge = r + 15 >= rows || t0 + 16 * KT - 1 > pfirst ||
                          (a.window > 0 && t0 <= plast - a.window && t0 + 16 * KT > a.sinks);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            f32x4 s = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = T::mfma16(kr[kt][ks], qf[ks], s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = fmaf(s[i], a.scale, -lse);
                if (edge && !sees(t0 + 16 * kt + 4 * g4 + i, pos, a.window, a.sinks)) x = -__builtin_huge_valf();
                sum[kt][i] += __builtin_amdgcn_exp2f(x);
            }
        }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum[kt][i] += __shfl_xor(sum[kt][i], x);
        const int j = t0 + 16 * kt + 4 * g4;
        if (n16 < 4 && vp[kt] >= 0 && j + n16 < sq.len) {
            const int64_t at = (((int64_t)vp[kt] * a.c.kv_heads + h) << a.c.shift) + ((j + n16) & a.c.smask);
            const float add = n16 == 0 ? sum[kt][0] : n16 == 1 ? sum[kt][1] : n16 == 2 ? sum[kt][2] : sum[kt][3];
            a.score_out[at] = a.c.scores[at] + add;
        }
    }
}

template <typename T, int KS>
static void launch_scores(const AttnParams& a, int max_kv, int max_q, hipStream_t stream) {
    const int pairs = a.c.batch * a.c.kv_heads;
    if (max_q * a.group > 64) {
        constexpr int KT = KS > 4 ? 2 : 4;
        hipLaunchKernelGGL((score_kernel<T, KS, KT>), dim3(pairs, (max_kv + 64 * KT - 1) / (64 * KT)), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((score_kernel<T, KS, 2>), dim3(pairs, (max_kv + 127) / 128), dim3(256), 0, stream, a);
    }
}

template <typename T>
static void launch_scores(const AttnParams& a, int max_kv, int max_q, hipStream_t stream) {
    const int D = a.c.head_dim;
    if (D <= 64) launch_scores<T, 2>(a, max_kv, max_q, stream);
    else if (D <= 96) launch_scores<T, 3>(a, max_kv, max_q, stream);
    else if (D <= 128) launch_scores<T, 4>(a, max_kv, max_q, stream);
    else launch_scores<T, 8>(a, max_kv, max_q, stream);
}

}  // namespace tms

extern "C" int tms_kv_add_scores(const tms_cache* cache, const tms_score_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_cache(cache, false, true);
    if (rc != TMS_OK) return rc;
    if (!args || !cache->scores || args->q_heads < 1 || args->q_heads % cache->kv_heads || args->sinks < 0 ||
        !std::isfinite(args->scale) || args->q_stride[0] < 0 || args->q_stride[0] % 8 || args->q_stride[1] < 0 ||
        args->q_stride[1] % 8 || ((uintptr_t)args->out & 15) || ((uintptr_t)args->lse & 3))
        return TMS_ERR_INVALID_ARG;
    if (cache->max_kv > 4 * 1024 * 1024 || (int64_t)cache->max_q * (args->q_heads / cache->kv_heads) > (1 << 24))
        return TMS_ERR_CAPACITY;
    if (cache->tokens > 0 && (!args->q || !args->lse || !aligned16(args->q))) return TMS_ERR_INVALID_ARG;
    if (cache->batch == 0 || cache->max_kv == 0) return TMS_OK;
    AttnParams a{};
    a.c = view_of(cache);
    a.q = (const char*)args->q;
    a.lse = const_cast<float*>(args->lse);
    a.score_out = args->out ? args->out : cache->scores;
    a.qt = 2 * args->q_stride[0];
    a.qh = 2 * args->q_stride[1];
    a.q_heads = args->q_heads;
    a.group = args->q_heads / cache->kv_heads;
    a.window = args->window > 0 && args->window < kMaxLen ? args->window : 0;
    a.sinks = std::min(args->sinks, kMaxLen);
    set_scale(a, args->scale);
    if (cache->dtype == TMS_DTYPE_BF16) launch_scores<Bf16>(a, cache->max_kv, cache->max_q, stream);
    else launch_scores<F16>(a, cache->max_kv, cache->max_q, stream);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
