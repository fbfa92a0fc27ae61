// tms_attn.hip -- attention of new tokens over the paged cache
// (tms_paged_attention): single tokens, short chunks of drafts and long chunks
// of a prompt, with shared key heads, a sliding window and sinks.
//
// One pass over the keys with a running maximum m and sum l per row:
//   m' = max(m, max_j s_j), o = o * 2^(m - m') + sum_j 2^(s_j - m') v_j,
// with s_j = q . k_j * scale * log2(e).  Rows of one key head are taken
// together: row r of a sequence is token r / G and head r % G of the G query
// heads that share the key head, so a key read once serves them all.
//
// Both products are matrix instructions on transposed tiles: S^T = K Q^T and
// O^T = V^T P^T.  A lane then holds one row's scores for several keys (row =
// lane % 16): the softmax needs no exchange but two shuffles for a maximum,
// and the weights are already where the second product wants its right
// operand, since the order of its inner index (the keys) is free as long as
// V^T's is the same.
#include <stddef.h>

#include <algorithm>
#include <cmath>

#include "tms_attn.h"

namespace tms {

// ---- few rows: keys spread over waves ------------------------------------------------------------
//
// 16 * RT rows of one key head a workgroup.  Its four waves take the key
// tiles (32 keys) of the workgroup's split in turn, each with its own running
// maximum and sum, and join at the end.  Keys and values go from memory to
// registers, in the matrix instructions' layout, without LDS: nothing is
// shared between the waves.  A lane reads 16 bytes of a key (lane % 16 the
// key, 64 bytes of a row together), and 8 values' rows at the 16 bytes
// lane % 16; v_perm pairs those rows' halves into the left operand, one
// instruction for two values.  Value row piece `c` of 8 then is rows
// {8c + t} of O^T in its tile t, so a lane ends with 8 neighbouring values of
// its row.
template <typename T, int KS, int VB, int RT>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnParams a) {
    constexpr int RM = 16 * RT, VP = VB / 8 ? VB / 8 : 1, VW = VB >= 8 ? 4 : 2;   // pieces, words a piece
    __shared__ float sm_o[2][VB * RT * 4 * 64];
    __shared__ float sm_m[2][RM], sm_l[2][RM];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n16 = lane & 15, g4 = lane >> 4;
    const int pair = blockIdx.x, tile = blockIdx.y, split = blockIdx.z;
    const int b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    const SeqView sq = seq_view(a.c, b);
    const int G = a.group, rows = sq.n * G, r0 = tile * RM;
    if (r0 >= rows) return;
    const int D = a.c.head_dim;
    const int rlast = min(r0 + RM, rows) - 1;
    const TileList<32> tl(a.window, a.sinks, sq.p0 + r0 / G, sq.p0 + rlast / G, sq.len);
    const int v0 = split * a.split_tiles, v1 = a.splits == split + 1 ? tl.n : min(tl.n, v0 + a.split_tiles);

    // This lane's row of each 16: its query and its position.
    u32x4 qf[RT][KS];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + rt * 16 + n16;
        const bool in = r < rows;
        const int tok = in ? r / G : 0, hd = in ? r - tok * G : 0;
        pos[rt] = in ? sq.p0 + tok : -1;
        const char* src = a.q + (int64_t)(sq.q0 + tok) * a.qt + (int64_t)(h * G + hd) * a.qh;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = s * 32 + g4 * 8;
            qf[rt][s] = in && d < D ? (*(const u32x4*)(src + 2 * d) & a.qand) ^ a.qxor : (u32x4){0, 0, 0, 0};
        }
    }

    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const char* kbase = a.c.k + (int64_t)h * a.c.kh;
    const char* vbase = a.c.v + (int64_t)h * a.c.vh;
    u32x4 kr[2][KS];
    uint32_t vr[2][4][VP][VW];
    int kp[2], vp[2];

    auto pages = [&](int v) {
        const int t0 = tl.key(v);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            kp[kt] = page_of(a.c, row, t0 + 16 * kt + n16, sq.len);
            vp[kt] = page_of(a.c, row, t0 + 16 * kt + 4 * g4, sq.len);
        }
    };
    // A key that does not exist is read from the first slot of the pool, and masked.
    auto load_k = [&](int v) {
        const int t0 = tl.key(v);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int j = t0 + 16 * kt + n16;
            const char* src = kbase + (kp[kt] < 0 ? 0 : (int64_t)kp[kt] * a.c.kp + (int64_t)(j & a.c.smask) * a.c.ks);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = s * 32 + g4 * 8;
                kr[kt][s] = d < D ? *(const u32x4*)(src + 2 * d) : (u32x4){0, 0, 0, 0};
            }
        }
    };
    auto load_v = [&](int v) {
        const int t0 = tl.key(v);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int j = (t0 + 16 * kt + 4 * g4) & a.c.smask;
            const char* src = vbase + (vp[kt] < 0 ? 0 : (int64_t)vp[kt] * a.c.vp + (int64_t)j * a.c.vs);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int p = 0; p < VP; ++p) {
                    const int d = p * 128 + n16 * (2 * VW);
                    const char* at = src + (vp[kt] < 0 ? 0 : i * a.c.vs) + 2 * (d < D ? d : 0);
                    if constexpr (VW == 4) {
                        const u32x4 x = *(const u32x4*)at;
#pragma unroll
                        for (int w = 0; w < 4; ++w) vr[kt][i][p][w] = x[w];
                    } else {
                        const u32x2 x = *(const u32x2*)at;
                        vr[kt][i][p][0] = x[0];
                        vr[kt][i][p][1] = x[1];
                    }
                }
        }
    };

    f32x4 o[RT][VB];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_huge_valf();
        l[rt] = 0.f;
#pragma unroll
        for (int t = 0; t < VB; ++t) o[rt][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }

    int v = v0 + wave;
    if (v < v1) {
        pages(v);
        load_k(v);
        load_v(v);
    }
    for (; v < v1; v += 4) {
        const int t0 = tl.key(v);
        // Which of this lane's 8 keys of S^T (and value rows) are there.
        uint32_t there = 0;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                there |= (uint32_t)(vp[kt] >= 0 && t0 + 16 * kt + 4 * g4 + i < sq.len) << (4 * kt + i);
        const bool more = v + 4 < v1;
        f32x4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                s[rt][kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[rt][kt] = T::mfma16(kr[kt][ks], qf[rt][ks], s[rt][kt]);
            }
        int vpn[2];
        if (more) {
            vpn[0] = vp[0];
            vpn[1] = vp[1];
            pages(v + 4);
            load_k(v + 4);
        }
        // A tile that some row sees in part: rows' own bounds, and values of
        // keys that are not there set to zero.
        const int pfirst = sq.p0 + r0 / G, plast = sq.p0 + rlast / G;
        const bool edge = __any(there != 0xFF) || t0 + 31 > pfirst ||
                          (a.window > 0 && t0 <= plast - a.window && t0 + 32 > a.sinks);
        bool odd = false;   // a value that is no finite number in such a tile
        if (edge) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = t0 + 16 * kt + 4 * g4 + i;
                        const bool on = (there >> (4 * kt + i) & 1) && sees(j, pos[rt], a.window, a.sinks);
                        s[rt][kt][i] = on ? s[rt][kt][i] : -__builtin_huge_valf();
                    }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int p = 0; p < VP; ++p)
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            uint32_t& x = vr[kt][i][p][w];
                            x = (there >> (4 * kt + i) & 1) ? x : 0u;
                            odd |= (x & T::kExp) == T::kExp || (x >> 16 & T::kExp) == T::kExp;
                        }
            odd = __any(odd);
        }
        u32x4 pb[RT];
        float pw[RT][8];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float x[8], top = -__builtin_huge_valf();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = s[rt][e >> 2][e & 3] * a.scale;
                top = fmaxf(top, x[e]);
            }
            if (__any(top > m[rt])) {   // (most tiles leave every row's maximum where it was)
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top, m[rt]);
                const float f = __builtin_amdgcn_exp2f(m[rt] - (top == -__builtin_huge_valf() ? 0.f : top));
                m[rt] = top;
                l[rt] *= f;
#pragma unroll
                for (int t = 0; t < VB; ++t) o[rt][t] *= f;
            }
            const float base = m[rt] == -__builtin_huge_valf() ? 0.f : m[rt];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pw[rt][e] = __builtin_amdgcn_exp2f(x[e] - base);
                l[rt] += pw[rt][e];
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) pb[rt][w] = T::pack(pw[rt][2 * w], pw[rt][2 * w + 1]);
        }
        if (!odd) {
#pragma unroll
            for (int t = 0; t < VB; ++t) {
                const int p = t / 8, w = (t & 7) >> 1;
                const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;
                u32x4 av;
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    av[x] = __builtin_amdgcn_perm(vr[x >> 1][2 * (x & 1) + 1][p][w], vr[x >> 1][2 * (x & 1)][p][w], sel);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[rt][t] = T::mfma16(av, pb[rt], o[rt][t]);
            }
        } else {
            // A weight of zero times an infinity or NaN would reach rows that
            // do not see the key: key by key, only where the weight is not zero.
            const int32_t vpc[2] = {more ? vpn[0] : vp[0], more ? vpn[1] : vp[1]};
            for (int key = 0; key < 32; ++key) {
                const int from = n16 + 16 * ((key & 15) >> 2);   // the lane that has this row's weight
                const int page = __shfl(key < 16 ? vpc[0] : vpc[1], from);
                const char* src = vbase + (int64_t)max(page, 0) * a.c.vp + (int64_t)((t0 + key) & a.c.smask) * a.c.vs;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float w = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = __shfl(pw[rt][e], from);
                        if (e == (key >> 4) * 4 + (key & 3)) w = x;
                    }
                    if (w == 0.f || page < 0) continue;
#pragma unroll
                    for (int t = 0; t < VB; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int d = (t / 8) * 128 + (g4 * 4 + i) * (2 * VW) + (t & 7);
                            if (d < D) o[rt][t][i] = fmaf(w, T::up(*(const uint16_t*)(src + 2 * d)), o[rt][t][i]);
                        }
                }
            }
        }
        if (more) load_v(v + 4);
    }

    // The waves' shares to wave 0, in pairs: 2 and 3 into 0 and 1, 1 into 0.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
    }
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
            const int w = wave - half;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (g4 == 0) {
                    sm_m[w][rt * 16 + n16] = m[rt];
                    sm_l[w][rt * 16 + n16] = l[rt];
                }
#pragma unroll
                for (int t = 0; t < VB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sm_o[w][((rt * VB + t) * 4 + i) * 64 + lane] = o[rt][t][i];
            }
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float m2 = sm_m[wave][rt * 16 + n16], top = fmaxf(m[rt], m2);
                const float base = top == -__builtin_huge_valf() ? 0.f : top;
                const float f1 = __builtin_amdgcn_exp2f(m[rt] - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
                m[rt] = top;
                l[rt] = l[rt] * f1 + sm_l[wave][rt * 16 + n16] * f2;
#pragma unroll
                for (int t = 0; t < VB; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[rt][t][i] = o[rt][t][i] * f1 + sm_o[wave][((rt * VB + t) * 4 + i) * 64 + lane] * f2;
            }
        }
        __syncthreads();
    }
    if (wave != 0) return;

#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + rt * 16 + n16;
        if (r >= rows) continue;
        if (a.splits > 1) {
            const int64_t at = (((int64_t)pair * a.row_tiles + tile) * a.splits + split) * RM + rt * 16 + n16;
            if (g4 == 0) {
                a.part_ml[2 * at] = m[rt];
                a.part_ml[2 * at + 1] = l[rt];
            }
#pragma unroll
            for (int t = 0; t < VB; t += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = (t / 8) * 128 + (g4 * 4 + i) * (2 * VW) + (t & 7);
                    if (d < D)
                        *(f32x4*)(a.part_o + at * D + d) =
                            (f32x4){o[rt][t][i], o[rt][t + 1][i], o[rt][t + 2][i], o[rt][t + 3][i]};
                }
            continue;
        }
        const int tok = r / G, hd = h * G + r - tok * G;
        const float inv = l[rt] == 0.f ? 0.f : 1.0f / l[rt];   // (a NaN sum stays one)
        if (a.lse && g4 == 0)
            a.lse[(int64_t)(sq.q0 + tok) * a.q_heads + hd] = (m[rt] + log2f(l[rt])) * kLn2;
        char* dst = a.out + (int64_t)(sq.q0 + tok) * a.ot + (int64_t)hd * a.oh;
#pragma unroll
        for (int t = 0; t < VB; t += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = (t / 8) * 128 + (g4 * 4 + i) * (2 * VW) + (t & 7);
                if (d < D)
                    *(u32x2*)(dst + 2 * d) = (u32x2){T::pack(o[rt][t][i] * inv, o[rt][t + 1][i] * inv),
                                                     T::pack(o[rt][t + 2][i] * inv, o[rt][t + 3][i] * inv)};
            }
    }
}

// ---- the splits' shares of a row ---------------------------------------------------------------
//
// A wave a row: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), the
// splits in order.  A split whose sum is zero saw nothing.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams a, int rm) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int pair = blockIdx.x, tile = blockIdx.y, b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    const SeqView sq = seq_view(a.c, b);
    const int G = a.group, rows = sq.n * G, D = a.c.head_dim;
    const int in = blockIdx.z * 4 + wave, r = tile * rm + in;
    if (in >= rm || r >= rows) return;
    const int64_t base = ((int64_t)pair * a.row_tiles + tile) * a.splits;
    float M = -__builtin_huge_valf();
    for (int s = lane; s < a.splits; s += 64) M = fmaxf(M, a.part_ml[2 * ((base + s) * rm + in)]);
    for (int x = 32; x; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
    const float ref = M == -__builtin_huge_valf() ? 0.f : M;
    float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const int64_t at = (base + s) * rm + in;
        const float l = a.part_ml[2 * at + 1], f = __builtin_amdgcn_exp2f(a.part_ml[2 * at] - ref);
        if (l == 0.f) continue;
        L += l * f;
        if (4 * lane < D) {
            const f32x4 o = *(const f32x4*)(a.part_o + at * D + 4 * lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += o[i] * f;
        }
    }
    const int tok = r / G, hd = h * G + r - tok * G;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    if (a.lse && lane == 0) a.lse[(int64_t)(sq.q0 + tok) * a.q_heads + hd] = (M + log2f(L)) * kLn2;
    if (4 * lane < D)
        *(u32x2*)(a.out + (int64_t)(sq.q0 + tok) * a.ot + (int64_t)hd * a.oh + 8 * lane) =
            (u32x2){T::pack(acc[0] * inv, acc[1] * inv), T::pack(acc[2] * inv, acc[3] * inv)};
}

// ---- host ---------------------------------------------------------------------------------------

// The chunk kernel's offsets: a page's stride and what its slots span in 32
// bits, and of 8 slots below 2^31.
static bool short_strides(const tms_cache* c, const int64_t* stride) {
    return 2 * stride[0] < (int64_t)1 << 32 && stride[2] < 1 << 26 && 2 * stride[2] * c->page_size < (int64_t)1 << 32;
}

struct AttnPlan {
    bool chunk;        // the chunk kernel
    int rm;            // rows a workgroup
    int row_tiles;
    int tiles;         // most key tiles of a row tile
    int split_tiles, splits;
    size_t o_bytes, ml_bytes;
};

static int check_attention(const tms_cache* c, const tms_attention_args* a) {
    const int rc = check_cache(c, true, true);
    if (rc != TMS_OK) return rc;
    if (!a || a->q_heads < 1 || a->q_heads % c->kv_heads || a->sinks < 0 || !std::isfinite(a->scale)) return TMS_ERR_INVALID_ARG;
    for (int i = 0; i < 2; ++i)
        if (a->q_stride[i] < 0 || a->q_stride[i] % 8 || a->out_stride[i] < 0 || a->out_stride[i] % 8) return TMS_ERR_INVALID_ARG;
    if ((int64_t)c->max_q * (a->q_heads / c->kv_heads) > (1 << 24)) return TMS_ERR_CAPACITY;
    if (c->tokens > 0 && c->batch > 0 && (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out) || ((uintptr_t)a->lse & 3)))
        return TMS_ERR_INVALID_ARG;
    return TMS_OK;
}

static AttnPlan plan_attention(const tms_cache* c, const tms_attention_args* a) {
    AttnPlan p;
    const int rows = min(c->max_q, c->tokens) * (a->q_heads / c->kv_heads);
    p.chunk = rows > 64 && short_strides(c, c->k_stride) && short_strides(c, c->v_stride);
    const int rt = rows <= 16 || c->head_dim > 128 ? 1 : 2;
    p.rm = p.chunk ? kChunkRows : 16 * rt;
    p.row_tiles = (rows + p.rm - 1) / p.rm;
    int64_t keys = min(c->max_kv, kMaxLen);
    if (a->window > 0) keys = std::min<int64_t>(keys, (int64_t)a->window + p.rm + a->sinks + 128);
    const int kt = p.chunk ? chunk_keys(c->head_dim) : 32;
    p.tiles = (int)((keys + kt - 1) / kt);
    const int64_t items = (int64_t)c->batch * c->kv_heads * p.row_tiles;
    if (p.chunk) {
        // Workgroups enough for two a CU, with 16 tiles each at least.
        const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(items, 1));
        p.split_tiles = (int)std::max<int64_t>((p.tiles + want - 1) / want, 16);
    } else {
    // Workgroups enough for four a CU, with 16 tiles each at least (four a wave).
    const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(items, 1));
    int split = std::max<int64_t>((p.tiles + want - 1) / want, 16);
    if (split > 64) split = 64;
    if ((p.tiles + split - 1) / split > 256) split = (p.tiles + 255) / 256;
    p.split_tiles = (split + 3) / 4 * 4;
    }
    p.splits = std::max(1, (p.tiles + p.split_tiles - 1) / p.split_tiles);
    const size_t parts = p.splits > 1 ? (size_t)items * p.splits * p.rm : 0;
    p.o_bytes = parts * c->head_dim * 4;
    p.ml_bytes = parts * 8;
    return p;
}

template <typename T, int KS, int VB>
static void launch_rows(const AttnPlan& p, const AttnParams& a, dim3 grid, hipStream_t stream) {
    if constexpr (VB <= 8) {
        if (p.rm == 32) {
            hipLaunchKernelGGL((attn_rows_kernel<T, KS, VB, 2>), grid, dim3(256), 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((attn_rows_kernel<T, KS, VB, 1>), grid, dim3(256), 0, stream, a);
}

template <typename T>
static void launch_attention(const AttnPlan& p, const AttnParams& a, hipStream_t stream) {
    const int D = a.c.head_dim;
    const dim3 grid(a.c.batch * a.c.kv_heads, p.row_tiles, p.splits);
    if (p.chunk) launch_attn_chunk(a, std::is_same<T, Bf16>::value, grid, stream);
    else if (D <= 64) launch_rows<T, 2, 4>(p, a, grid, stream);
    else if (D <= 96) launch_rows<T, 3, 8>(p, a, grid, stream);
    else if (D <= 128) launch_rows<T, 4, 8>(p, a, grid, stream);
    else launch_rows<T, 8, 16>(p, a, grid, stream);
    if (p.splits > 1)
        hipLaunchKernelGGL((attn_join_kernel<T>), dim3(grid.x, p.row_tiles, (p.rm + 3) / 4), dim3(256), 0, stream, a, p.rm);
}

}  // namespace tms

extern "C" int64_t tms_paged_attention_workspace(const tms_cache* cache, const tms_attention_args* args) {
    const int rc = tms::check_attention(cache, args);
    if (rc != TMS_OK) return rc;
    const tms::AttnPlan p = tms::plan_attention(cache, args);
    return (int64_t)(p.o_bytes + p.ml_bytes);
}

extern "C" int tms_paged_attention(const tms_cache* cache, const tms_attention_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_attention(cache, args);
    if (rc != TMS_OK) return rc;
    if (cache->batch == 0 || cache->tokens == 0 || cache->max_q == 0) return TMS_OK;
    const AttnPlan p = plan_attention(cache, args);
    if (p.row_tiles > 65535) return TMS_ERR_CAPACITY;
    if (args->workspace_bytes < p.o_bytes + p.ml_bytes ||
        (p.splits > 1 && (!args->workspace || !aligned16(args->workspace))))
        return TMS_ERR_INVALID_ARG;
    AttnParams a;
    a.c = view_of(cache);
    a.q = (const char*)args->q;
    a.out = (char*)args->out;
    a.lse = args->lse;
    a.score_out = nullptr;
    a.qt = 2 * args->q_stride[0];
    a.qh = 2 * args->q_stride[1];
    a.ot = 2 * args->out_stride[0];
    a.oh = 2 * args->out_stride[1];
    a.q_heads = args->q_heads;
    a.group = args->q_heads / cache->kv_heads;
    a.window = args->window > 0 && args->window < kMaxLen ? args->window : 0;
    a.sinks = std::min(args->sinks, kMaxLen);
    set_scale(a, args->scale);
    a.split_tiles = p.split_tiles;
    a.splits = p.splits;
    a.row_tiles = p.row_tiles;
    a.part_o = (float*)args->workspace;
    a.part_ml = (float*)((char*)args->workspace + p.o_bytes);
    if (cache->dtype == TMS_DTYPE_BF16) launch_attention<Bf16>(p, a, stream);
    else launch_attention<F16>(p, a, stream);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
