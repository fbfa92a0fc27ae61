// tms_scores.hip -- the attention weight that new tokens give to each cached
// key (tms_kv_add_scores): score[j] += sum over rows of 2^(s_j - lse), with
// s and lse to base 2.  One matrix product, S^T = K Q^T, and no exchange
// between workgroups: a wave keeps its keys in registers and passes over the
// rows that see them, so a key's sum is one wave's, in row order.
#include <algorithm>
#include <cmath>

#include "tms_attn.h"

namespace tms {

// Sums of x[i] over the 32 lanes of a half wave; the lane gets that of
// i = row_key(lane), each twice.
__device__ __forceinline__ int row_key(int n32) { return (n32 & 1) << 3 | (n32 & 2) << 1 | (n32 & 4) >> 1 | (n32 & 8) >> 3; }

template <int BIT, int HALF> __device__ __forceinline__ void give_half(float* x, int n32) {
    const bool up = n32 & BIT;
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
        const float give = up ? x[i] : x[i + HALF], keep = up ? x[i + HALF] : x[i];
        x[i] = keep + __shfl_xor(give, BIT);
    }
}

__device__ __forceinline__ float sum_rows(float* x, int n32) {
    give_half<1, 8>(x, n32);
    give_half<2, 4>(x, n32);
    give_half<4, 2>(x, n32);
    give_half<8, 1>(x, n32);
    return x[0] + __shfl_xor(x[0], 16);
}

// Four waves of 32 keys of one key head.  The rows that see any of the 128 come
// by 64 through LDS, loaded there (as the chunk kernel loads its keys) while the 64
// before are used, and the weights of 32 rows are summed among the products of the
// next 32.  Bound by the vector pipe: 16 cycles of a SIMD for the exponentials of 64
// weights and 8 for scaling and sum, beside 10 (D = 80) to 32 (D = 256) of the matrix
// pipe (1024 and 777 tokens over 6000 and 4097, 8 heads of 2 of 80 dimensions, fp16: 51 us, of
// which exponentials alone take 15; 153 us with rows read by each wave from memory).
template <typename T, int ROWB, int KS>
__global__ __launch_bounds__(256, KS > 8 ? 2 : 3) void score_kernel(AttnParams a) {
    constexpr int RQ = 64, C = ROWB / 16, RPI = 64 / C, NI = RQ / (4 * RPI);
    __shared__ __attribute__((aligned(128))) char sm[2][RQ * ROWB];
    __shared__ float sm_lse[2][RQ];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31, hh = lane >> 5;
    const int pair = blockIdx.x, b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    SeqView sq = seq_view(a.c, b);
    sq.len = min(sq.len, a.max_kv);
    const int g0 = blockIdx.y * 128, t0 = g0 + wave * 32;
    if (g0 >= sq.len) return;
    const int G = a.group, D = a.c.head_dim;
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;

    // Rows that see a key of the workgroup's: from the first at or past its
    // first key to the last whose window still reaches its last key.
    const int g1 = min(g0 + 128, sq.len) - 1;
    const int first = min(max(g0 - sq.p0, 0), sq.n);
    int last = sq.n - 1;
    if (a.window > 0 && g0 >= a.sinks) last = min(last, g1 - sq.p0 + a.window - 1);
    const float inv = 1.0f / (float)G;
    const int rbegin = first * G, rend = (last + 1) * G;

    // A tile has whole tokens (`step` rows, at most 64), so a lane's offsets from
    // its first token are the same in every tile; a group of more than 64 has none
    // whole, and its offsets are worked out for each tile.
    const bool whole = G <= RQ;
    const int step = whole ? RQ / G * G : RQ;
    const char* qbase = a.q + (int64_t)sq.q0 * a.qt + (int64_t)h * G * a.qh;
    const float* lbase = a.lse + (int64_t)sq.q0 * a.q_heads + h * G;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)&sm[0][0];
    uint32_t off[NI];
    int loff, tok0 = first;   // the lane's row's lse; the token that the offsets count from
    // A place of the tile without a row (past its last whole token, past the last row of
    // all) has its first row, at no weight: zeros there, times an infinite key, would be no number.
    auto offsets = [&](int hd0) __attribute__((always_inline)) {   // rows from head hd0 of the token on
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int rr = (wave * NI + i) * RPI + lane / C, piece = (lane % C) ^ key_swizzle<ROWB>(rr);
            int tok, hd;
            split_row(rr < step ? hd0 + rr : hd0, G, inv, tok, hd);
            off[i] = piece * 8 < D ? (uint32_t)(tok * (int)a.qt + hd * (int)a.qh + piece * 16) : 0x80000000u;
        }
        int tok, hd;
        split_row(hd0 + lane, G, inv, tok, hd);
        loff = tok * a.q_heads + hd;
    };
    offsets(0);
    // The tile from row r (token tok0) on: its last row's end bounds the resource.
    auto load = [&](int r, int buf) __attribute__((always_inline)) {
        int hd0 = 0;
        if (!whole) {
            split_row(r, G, inv, tok0, hd0);
            offsets(hd0);
        }
        const char* base = qbase + (int64_t)__builtin_amdgcn_readfirstlane(tok0) * a.qt;
        const int left = rend - r;   // rows
        if (left < step) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int rr = (wave * NI + i) * RPI + lane / C, piece = (lane % C) ^ key_swizzle<ROWB>(rr);
                if (rr >= left && piece * 8 < D) off[i] = hd0 * (int)a.qh + piece * 16;
            }
        }
        const u32x4 res = (u32x4){(uint32_t)(uintptr_t)base, (uint32_t)((uintptr_t)base >> 32) & 0xFFFF, 0x7FFFFFFFu, 0x00020000u};
#pragma unroll
        for (int i = 0; i < NI; ++i)
            load_lds16(res, off[i], lds0 + buf * RQ * ROWB + (wave * NI + i) * 1024);
    };
    auto lse_of = [&](int r) __attribute__((always_inline)) {   // the first wave's: row r + lane; a row that is none gets no weight
        const float x = lbase[(int64_t)tok0 * a.q_heads + (lane < step && r + lane < rend ? loff : 0)];
        return lane < step && r + lane < rend && x != -__builtin_huge_valf() ? x * kLog2e : __builtin_huge_valf();
    };
    int prow[2];   // token of the lane's row of each half, from the tile's first on
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        int hd;
        split_row(32 * half + n32, G, inv, prow[half], hd);
    }
    const bool any = rbegin < rend;
    float lnext = 0.f;
    if (any) {
        load(rbegin, 0);
        if (wave == 0) lnext = lse_of(rbegin);
    }

    u32x4 kr[KS];
    const int j0 = t0 + n32, page = page_of(a.c, row, j0, sq.len);
    {
        const char* src = a.c.k + (int64_t)h * a.c.kh + (page < 0 ? 0 : (int64_t)page * a.c.kp + (int64_t)(j0 & a.c.smask) * a.c.ks);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + hh * 8;
            kr[s] = *(const u32x4*)(src + 2 * (d < D ? d : 0));
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int w = 0; w < 4; ++w) kr[s][w] = s * 16 + hh * 8 < D ? (kr[s][w] & a.qand) ^ a.qxor : 0u;
    }
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;

    // The scores of 32 rows, while the weights of the 32 before (`s`) are summed:
    // a matrix instruction, some weights, the operand of two steps on.
    auto stage = [&](const char* sq_rows, int half, f32x16& next, const f32x16& s, float lse) __attribute__((always_inline)) {
        u32x4 qf[3];
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.f;
        qf[0] = key_operand<ROWB>(sq_rows, lane, half, 0);
        qf[1] = key_operand<ROWB>(sq_rows, lane, half, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (ks + 2 < KS) qf[(ks + 2) % 3] = key_operand<ROWB>(sq_rows, lane, half, ks + 2);
            next = T::mfma32(kr[ks], qf[ks % 3], next);
#pragma unroll
            for (int e = 16 * ks / KS; e < 16 * (ks + 1) / KS; ++e) {
                sum[e] += __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, -lse));
                asm volatile("" : "+v"(sum[e]));   // (here, not past the branch that follows)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    f32x16 s0, s1;
    float lse0 = 0.f, lse1 = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s1[i] = -__builtin_huge_valf();   // nothing before the first

    int buf = 0;
    for (int r = rbegin; r < rend; r += step, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (wave == 0) sm_lse[buf][lane] = lnext;
        __syncthreads();
        int pf, pl, hd;   // positions of the tile's first row and last
        if (whole) {
            pf = sq.p0 + tok0;
            pl = min(pf + step / G, sq.p0 + last + 1) - 1;
        } else {
            split_row(r, G, inv, pf, hd);
            split_row(min(r + step, rend) - 1, G, inv, pl, hd);
            pf = sq.p0 + __builtin_amdgcn_readfirstlane(pf);
            pl = sq.p0 + __builtin_amdgcn_readfirstlane(pl);
        }
        if (r + step < rend) {
            if (whole) tok0 += step / G;
            load(r + step, buf ^ 1);
            if (wave == 0) lnext = lse_of(r + step);
        }
        if (t0 > pl || t0 >= sq.len || (a.window > 0 && t0 + 31 <= pf - a.window && t0 >= a.sinks)) continue;
        const bool edge = t0 + 31 > pf || (a.window > 0 && t0 <= pl - a.window && t0 + 32 > a.sinks);
        auto mask = [&](f32x16& x, int half, float& lse) __attribute__((always_inline)) {
            // A lse that is no number makes one of -inf no more: such a row's scores take its place.
            if (__any(lse != lse)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = lse != lse ? lse : x[i];
                lse = lse != lse ? 0.f : lse;
            }
            int pos = pf + prow[half];
            if (!whole) {
                split_row(r + 32 * half + n32, G, inv, pos, hd);
                pos += sq.p0;
            }
            if (32 * half + n32 >= min(step, rend - r)) pos = -1;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!sees(t0 + 8 * (i / 4) + 4 * hh + (i & 3), pos, a.window, a.sinks)) x[i] = -__builtin_huge_valf();
        };
        stage(sm[buf], 0, s0, s1, lse1);
        lse0 = sm_lse[buf][n32];
        if (edge) mask(s0, 0, lse0);
        stage(sm[buf], 1, s1, s0, lse0);
        lse1 = sm_lse[buf][32 + n32];
        if (edge) mask(s1, 1, lse1);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] += __builtin_amdgcn_exp2f(fmaf(s1[i], a.scale, -lse1));
    const float add = sum_rows(sum, n32);
    const int i = row_key(n32), key = 8 * (i / 4) + 4 * hh + (i & 3), its = __shfl(page, key);
    if (n32 < 16 && its >= 0) {
        const int64_t at = (((int64_t)its * a.c.kv_heads + h) << a.c.shift) + ((t0 + key) & a.c.smask);
        a.score_out[at] = a.c.scores[at] + add;
    }
}

// At most 32 rows (a decode step's): they are read straight into registers by
// each wave, which takes KT times 32 keys and waits for no other.
template <typename T, int KS, int KT>
__global__ __launch_bounds__(256, KS > 8 ? 2 : 3) void score_rows_kernel(AttnParams a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n32 = lane & 31, hh = lane >> 5;
    const int pair = blockIdx.x, b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    SeqView sq = seq_view(a.c, b);
    sq.len = min(sq.len, a.max_kv);
    const int t0 = (blockIdx.y * 4 + wave) * 32 * KT;
    if (t0 >= sq.len) return;
    const int G = a.group, rows = sq.n * G, D = a.c.head_dim;
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    int page[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) page[kt] = row[min(t0 + 32 * kt + n32, sq.len - 1) >> a.c.shift];

    const bool in = n32 < rows;
    const int tok = in ? n32 / G : 0, hd = in ? n32 - tok * G : 0, pos = in ? sq.p0 + tok : -1;
    const int64_t qrow = rows > 0 ? sq.q0 + tok : 0;   // (a sequence without rows may have no row to read)
    u32x4 qf[KS], kr[KT][KS];
    float lse = -__builtin_huge_valf();
    if (rows > 0) {
        lse = a.lse[qrow * a.q_heads + h * G + hd] * kLog2e;
        const char* src = a.q + qrow * a.qt + (int64_t)(h * G + hd) * a.qh;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = query_operand(a, src, s * 16 + hh * 8, in);
    }
    if (lse == -__builtin_huge_valf()) lse = -lse;   // the row saw nothing: no weight
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int j = t0 + 32 * kt + n32;
        if (j >= sq.len || (uint32_t)page[kt] >= (uint32_t)a.c.pages) page[kt] = -1;
        const char* src = a.c.k + (int64_t)h * a.c.kh + (page[kt] < 0 ? 0 : (int64_t)page[kt] * a.c.kp + (int64_t)(j & a.c.smask) * a.c.ks);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 16 + hh * 8;
            kr[kt][s] = *(const u32x4*)(src + 2 * (d < D ? d : 0));
        }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int i16 = row_key(n32), key = 8 * (i16 / 4) + 4 * hh + (i16 & 3), its = __shfl(page[kt], key);
        const int64_t at = (((int64_t)its * a.c.kv_heads + h) << a.c.shift) + ((t0 + 32 * kt + key) & a.c.smask);
        float add = 0.f, had = 0.f;
        if (n32 < 16 && its >= 0) had = a.c.scores[at];
        if (rows > 0) {
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int w = 0; w < 4; ++w) kr[kt][ks][w] = ks * 16 + hh * 8 < D ? kr[kt][ks][w] : 0u;
                s = T::mfma32(kr[kt][ks], qf[ks], s);
            }
            float weight[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool on = sees(t0 + 32 * kt + 8 * (i / 4) + 4 * hh + (i & 3), pos, a.window, a.sinks);
                weight[i] = on ? __builtin_amdgcn_exp2f(fmaf(s[i], a.scale, -lse)) : 0.f;
            }
            add = sum_rows(weight, n32);
        }
        if (n32 < 16 && its >= 0) a.score_out[at] = had + add;
    }
}

template <typename T>
static void launch_scores(const AttnParams& a, int max_kv, int max_q, hipStream_t stream) {
    const int D = a.c.head_dim, pairs = a.c.batch * a.c.kv_heads;
    if (max_q * a.group <= 32) {   // (32 sequences of 257 to 4096, one token each: 37 us, 55 by way of LDS)
        const dim3 grid(pairs, (max_kv + 255) / 256), grid1(pairs, (max_kv + 127) / 128);
        if (D <= 64) hipLaunchKernelGGL((score_rows_kernel<T, 4, 2>), grid, dim3(256), 0, stream, a);
        else if (D <= 96) hipLaunchKernelGGL((score_rows_kernel<T, 6, 2>), grid, dim3(256), 0, stream, a);
        else if (D <= 128) hipLaunchKernelGGL((score_rows_kernel<T, 8, 2>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((score_rows_kernel<T, 16, 1>), grid1, dim3(256), 0, stream, a);
        return;
    }
    const dim3 grid(pairs, (max_kv + 127) / 128);
    if (D <= 64) hipLaunchKernelGGL((score_kernel<T, 128, 4>), grid, dim3(256), 0, stream, a);
    else if (D <= 96) hipLaunchKernelGGL((score_kernel<T, 256, 6>), grid, dim3(256), 0, stream, a);
    else if (D <= 128) hipLaunchKernelGGL((score_kernel<T, 256, 8>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((score_kernel<T, 512, 16>), grid, dim3(256), 0, stream, a);
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
    if (cache->max_kv > TMS_SCORES_MAX_KV || (int64_t)cache->max_q * (args->q_heads / cache->kv_heads) > TMS_ATTENTION_MAX_ROWS ||
        args->q_stride[0] > TMS_SCORES_MAX_Q_STRIDE || args->q_stride[1] > TMS_SCORES_MAX_Q_STRIDE ||
        args->q_stride[1] * (args->q_heads / cache->kv_heads) > TMS_SCORES_MAX_Q_STRIDE)
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
    a.max_kv = cache->max_kv;
    a.window = args->window > 0 && args->window < kMaxLen ? args->window : 0;
    a.sinks = std::min(args->sinks, kMaxLen);
    set_scale(a, args->scale);
    if (cache->dtype == TMS_DTYPE_BF16) launch_scores<Bf16>(a, cache->max_kv, std::min(cache->max_q, cache->tokens), stream);
    else launch_scores<F16>(a, cache->max_kv, std::min(cache->max_q, cache->tokens), stream);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
