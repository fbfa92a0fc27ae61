// tms_attn.hip -- attention of new tokens over the paged cache
// (tms_paged_attention): single tokens, short chunks of drafts and long chunks
// of a prompt, with shared key heads, a sliding window and sinks.
//
// One pass over the keys with a running reference m and sum l per row:
//   m' = max(m, max_j s_j - lift), o = o * 2^(m - m') + sum_j 2^(s_j - m') v_j,
// with s_j = q . k_j * scale * log2(e), and the lift 0, or what puts a row's weights
// where fp16 has its bits.  Weights are rounded to the cache's type, half a
// step, because that is what the matrix instructions take beside it (a second product
// for what rounding leaves would add half of the matrix work): an output is off
// by some 0.0008 of itself in bf16 so, beside 0.0017 by its own rounding.  Rows of one key head are taken
// together: row r of a sequence is token r / G and head r % G of the G query
// heads that share the key head, so a key read once serves them all.
//
// Both products are matrix instructions on transposed tiles: S^T = K Q^T and
// O^T = V^T P^T.  A lane then holds one row's scores for several keys (row =
// lane % 32): the softmax needs no exchange but one shuffle for a maximum,
// and the weights are already where the second product wants its right
// operand, since the order of its inner index (the keys) is free as long as
// V^T's is the same.
#include <stddef.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tms_attn.h"

namespace tms {

constexpr int kShareRows = 32;   // of a workgroup of the rows kernel
// What an item takes besides its tiles, in tiles (64 sequences of 40 to 2000
// positions: 90 us with 0, 59 with 4, 56 with 8, 60 with 32), and the shortest
// share in tiles: one for each wave.
constexpr int kItemCost = 8, kLeastShare = 4;

// ---- few rows: the keys of all sequences in equal shares ---------------------------------------
//
// Bound by memory: the keys and values of a call are read once.  All items
// (sequence, row tile, key head) lie behind each other on one axis of key
// tiles, and each workgroup takes an equal share of it, whatever the lengths;
// an item that its share holds whole is written out, the two at its ends go
// to the workspace as parts, which a second launch joins.
//
// Within an item the waves take the tiles (32 keys) in turn, each with
// its own running maximum and sum and its own piece of LDS: a tile's keys are
// loaded there while the values of the one before are used, and its values
// while its keys are, so that 8 waves a CU keep some 100 KB on the way without
// a register for it.  No wave waits for another before the item's end.
// (64 sequences of 257 to 8192, 8 key heads of 4 of 128 dimensions, bf16: 207 us, 5.4
// TB/s; keys and values in registers, shares of a sequence: 306 us.)

// An item's tiles (one at least: rows that see nothing have an output all the
// same) and what it takes besides, as tiles.
__device__ __forceinline__ int item_length(const AttnParams& a, int tiles) { return max(tiles, 1) + kItemCost; }

__device__ __forceinline__ int item_tiles(const AttnParams& a, int combo) {
    const int b = combo / a.row_tiles, tile = combo - b * a.row_tiles;
    const SeqView sq = seq_view(a.c, b);
    const int G = a.group, rows = sq.n * G, r0 = tile * kShareRows;
    if (r0 >= rows) return 0;
    return item_length(a, TileList<32>(a.window, a.sinks, sq.p0 + r0 / G, sq.p0 + (min(r0 + kShareRows, rows) - 1) / G, sq.len).n);
}

__device__ __forceinline__ int64_t share_of(const AttnParams& a, int64_t total, int shares) {
    return max((total + shares - 1) / shares, (int64_t)a.split_tiles);
}

// Four values of a row's output from dimension d on, and its lse.
template <typename T>
__device__ __forceinline__ void write_row(const AttnParams& a, const SeqView& sq, int h, int r, int d, float m, float l, f32x4 o) {
    const int tok = r / a.group, hd = h * a.group + r - tok * a.group;
    const float inv = l == 0.f ? 0.f : 1.0f / l;   // (a NaN sum stays one)
    if (a.lse && d == 0) a.lse[(int64_t)(sq.q0 + tok) * a.q_heads + hd] = (m + log2f(l)) * kLn2;
    *(u32x2*)(a.out + (int64_t)(sq.q0 + tok) * a.ot + (int64_t)hd * a.oh + 2 * d) =
        (u32x2){T::pack(o[0] * inv, o[1] * inv), T::pack(o[2] * inv, o[3] * inv)};
}

template <typename T, int ROWB, int KS, int DT, int NW>
__global__ __launch_bounds__(64 * NW, ROWB > 256 ? 1 : 2) void attn_rows_kernel(AttnParams a) {
    constexpr int RM = kShareRows, KT = 32, NL = KT * ROWB / 1024, RPI = 1024 / ROWB, PAD = 33;
    // LDS: the waves' pieces, and at an item's end their outputs, maxima and sums.
    constexpr int RING = NW * 2 * KT * ROWB;
    constexpr int MERGE = NW * DT * 32 * PAD * 4, ML = NW * 32 * 2 * 4;
    __shared__ __attribute__((aligned(128))) char sm[MERGE + ML > RING ? MERGE + ML : RING];
    float* const sm_ml = (float*)(sm + MERGE);   // [wave][row][maximum, sum]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n32 = lane & 31, hh = lane >> 5;
    const int H = a.c.kv_heads, G = a.group, D = a.c.head_dim;
    const int combos = a.c.batch * a.row_tiles;

    // The share: [x, end) of the axis, which starts in `combo` (a sequence's
    // row tile, all key heads one after another) at `at`.  Without shares, an
    // item a workgroup.
    int64_t share = 0, x = 0, end = 1, at = 0;
    int combo = blockIdx.x / H;
    if (a.split_tiles > 0) {
        int64_t* const wsum = (int64_t*)sm;   // [NW], then where the share starts
        const int per = (combos + 64 * NW - 1) / (64 * NW), c0 = min(t * per, combos), c1 = min(c0 + per, combos);
        int64_t mine = 0;
        for (int c = c0; c < c1; ++c) mine += item_tiles(a, c);
        int64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        if (lane == 63) wsum[wave] = upto;
        __syncthreads();
        int64_t total = 0, before = upto - mine;
        for (int w = 0; w < NW; ++w) {
            before += w < wave ? wsum[w] : 0;
            total += wsum[w];
        }
        share = share_of(a, total * H, gridDim.x);
        x = blockIdx.x * share;
        end = min(x + share, total * H);
        if (x >= end) return;
        if (x >= before * H && x < (before + mine) * H)
            for (int c = c0;; ++c) {
                const int n = item_tiles(a, c);
                if (x < (before + n) * H) {
                    wsum[NW] = c;
                    wsum[NW + 1] = before * H;
                    break;
                }
                before += n;
            }
        __syncthreads();
        combo = __builtin_amdgcn_readfirstlane((int)wsum[NW]);
        at = wsum[NW + 1];
        __syncthreads();
    }

    char* ring = sm + wave * 2 * KT * ROWB;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)ring;
    const uint32_t kslot = (uint32_t)a.c.ks, vslot = (uint32_t)a.c.vs;
    uint32_t koff[NL], voff[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int rr = i * RPI + lane / (ROWB / 16), lc = lane % (ROWB / 16);
        const int ck = lc ^ key_swizzle<ROWB>(rr), cv = lc ^ value_swizzle<ROWB>(rr);
        koff[i] = ck * 8 < D ? (rr & 7) * kslot + ck * 16 : 0x80000000u;
        voff[i] = cv * 8 < D ? (rr & 7) * vslot + cv * 16 : 0x80000000u;
    }

    while (x < end) {
        const int b = combo / a.row_tiles, tile = combo - b * a.row_tiles;
        const SeqView sq = seq_view(a.c, b);
        const int rows = sq.n * G, r0 = tile * RM;
        if (r0 >= rows) {
            if (a.split_tiles == 0) return;
            ++combo;
            continue;
        }
        const int nr = min(RM, rows - r0);
        const int pfirst = sq.p0 + r0 / G, plast = sq.p0 + (r0 + nr - 1) / G;
        const TileList<KT> tl(a.window, a.sinks, pfirst, plast, sq.len);
        const int n = max(tl.n, 1), axis = item_length(a, tl.n);
        int h = blockIdx.x - combo * H, k0 = 0, k1 = n;
        int64_t item = 0;
        if (a.split_tiles > 0) {
            if (x >= at + (int64_t)axis * H) {
                at += (int64_t)axis * H;
                ++combo;
                continue;
            }
            h = (int)((x - at) / axis);
            item = at + (int64_t)h * axis;
            k0 = (int)(x - item);
            k1 = (int)min((int64_t)n, end - item);
            x = min(item + axis, end);
            if (k0 >= n) continue;
        }
        const int kend = min(k1, tl.n);

        const int r = r0 + n32;
        const bool in = r < rows;
        const int tok = in ? r / G : 0, hd = in ? r - tok * G : 0;
        const int pos = in ? sq.p0 + tok : -1;
        u32x4 qf[KS];
        {
            const char* src = a.q + (int64_t)(sq.q0 + tok) * a.qt + (int64_t)(h * G + hd) * a.qh;
#pragma unroll
            for (int s = 0; s < KS; ++s) qf[s] = query_operand(a, src, s * 16 + hh * 8, in);
        }
        // Table entries of a tile's groups of 8 keys: by the scalar cache, whose
        // counter the loads into LDS do not share.
        typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
        const scalar_ptr row = (scalar_ptr)(uintptr_t)(a.c.tables + (int64_t)b * a.c.tstride);
        const char* kbase = a.c.k + (int64_t)h * a.c.kh;
        const char* vbase = a.c.v + (int64_t)h * a.c.vh;
        int page[4], next[4];
        auto entries = [&](int v) __attribute__((always_inline)) {
            const int t0 = tl.key(v);
#pragma unroll
            for (int g = 0; g < 4; ++g) next[g] = row[min(t0 + 8 * g, sq.len - 1) >> a.c.shift];
        };
        auto take = [&](int v) __attribute__((always_inline)) {   // bit g: group g of 8 keys is there
            const int t0 = tl.key(v);
            uint32_t there = 0;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const bool ok = t0 + 8 * g < sq.len && (uint32_t)next[g] < (uint32_t)a.c.pages;
                page[g] = ok ? next[g] : -1;
                there |= ok ? 1u << g : 0u;
            }
            return there;
        };
        auto load = [&](int v, const char* base, int64_t pstride, uint32_t slot, const uint32_t* off, uint32_t to) __attribute__((always_inline)) {
            const int t0 = tl.key(v);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int j = t0 + 8 * g;
                const uint32_t p = max(page[g], 0), sl = page[g] < 0 ? 0 : j & a.c.smask;
                const u32x4 res = slots_rsrc(base + p * pstride + (uint64_t)sl * slot, page[g] < 0 ? -1 : min(8, sq.len - j) - 1, slot, 2 * D);
#pragma unroll
                for (int i = g * 8 / RPI; i < (g + 1) * 8 / RPI; ++i) load_lds16(res, off[i], to + i * 1024);
            }
        };

        f32x16 o[DT];
        float m = -__builtin_huge_valf(), l = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
        int v = k0 + wave;
        uint32_t there = 0;
        if (v < kend) {
            entries(v);
            there = take(v);
            __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): what went before is not counted below
            load(v, kbase, a.c.kp, kslot, koff, lds0);
            load(v, vbase, a.c.vp, vslot, voff, lds0 + KT * ROWB);
            if (v + NW < kend) entries(v + NW);
        }
        for (; v < kend; v += NW) {
            const bool more = v + NW < kend;
            const int t0 = tl.key(v);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");   // the keys; the values may be on the way
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = T::mfma32(key_operand<ROWB>(ring, lane, 0, ks), qf[ks], s);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the keys are read: their place is free
            const uint32_t now = there;
            if (more) {
                there = take(v + NW);
                load(v + NW, kbase, a.c.kp, kslot, koff, lds0);
                if (v + 2 * NW < kend) entries(v + 2 * NW);
            }
            const bool edge = now != 15 || t0 + KT > sq.len || t0 + KT - 1 > pfirst ||
                              (a.window > 0 && t0 <= plast - a.window && t0 + KT > a.sinks);
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = t0 + 8 * (i / 4) + 4 * hh + (i & 3);
                    const bool on = (now >> (i / 4) & 1) && j < sq.len && sees(j, pos, a.window, a.sinks);
                    s[i] = on ? s[i] : -__builtin_huge_valf();
                }
            }
            float top = -__builtin_huge_valf();
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
            top *= a.scale;
            if (__any(top > m + T::kMost)) {   // (as in the chunk kernel)
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top - T::kLift, m);
                const float f = __builtin_amdgcn_exp2f(m - (top == -__builtin_huge_valf() ? 0.f : top));
                m = top;
                l *= f;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
            }
            const float base = m == -__builtin_huge_valf() ? 0.f : m;
            float sum = 0.f;   // (small weights add up before they meet a large sum)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, -base));
                sum += s[e];
            }
            l += sum;
            u32x4 pf[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int w = 0; w < 4; ++w) pf[u][w] = T::pack(s[8 * u + 2 * w], s[8 * u + 2 * w + 1]);
            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");   // the values; the next keys may be on the way
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            char* sv = ring + KT * ROWB;
            if (edge) {
                // A weight of zero times an infinity or NaN would reach rows that
                // do not see the value: such values go, key by key, to the rows
                // whose weight is not zero (which weight does not matter), and are
                // zero in the product.
                bool odd = false;
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    const u32x4 y = *(const u32x4*)(sv + i * 1024 + lane * 16);
#pragma unroll
                    for (int w = 0; w < 4; ++w) odd |= (y[w] & T::kExp) == T::kExp || (y[w] >> 16 & T::kExp) == T::kExp;
                }
                if (__any(odd)) {
                    uint32_t mine = 0;
#pragma unroll
                    for (int e = 0; e < 16; ++e) mine |= s[e] != 0.f ? 1u << e : 0u;
                    const uint32_t other = __shfl_xor(mine, 32);
#pragma unroll 1
                    for (int key = 0; key < KT; ++key) {
                        const uint32_t w = (key >> 2 & 1) == hh ? mine : other;
                        if (!(w >> (key / 8 * 4 + (key & 3)) & 1)) continue;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const u32x2 val = *(const u32x2*)(sv + key * ROWB + 16 * ((4 * dt + c) ^ value_swizzle<ROWB>(key)) + 8 * hh);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t bits = val[i / 2] >> 16 * (i & 1) & 0xFFFF;
                                    o[dt][4 * c + i] += (bits & T::kExp) == T::kExp ? T::up(bits) : 0.f;
                                }
                            }
                    }
#pragma unroll 1
                    for (int i = 0; i < NL; ++i) {
                        u32x4 y = *(const u32x4*)(sv + i * 1024 + lane * 16);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if ((y[w] & T::kExp) == T::kExp) y[w] &= 0xFFFF0000u;
                            if ((y[w] >> 16 & T::kExp) == T::kExp) y[w] &= 0x0000FFFFu;
                        }
                        *(u32x4*)(sv + i * 1024 + lane * 16) = y;
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int u = 0; u < 2; ++u) o[dt] = T::mfma32(value_operand<ROWB>(sv, lane, dt, u), pf[u], o[dt]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) load(v + NW, vbase, a.c.vp, vslot, voff, lds0 + KT * ROWB);
        }

        // The waves' shares of the item's rows, by way of LDS: an array
        // [dimension][row] a wave.
        const bool whole = k0 == 0 && k1 == n;
        const int64_t part = 2 * (int64_t)blockIdx.x + (k0 == 0 ? 1 : 0);
        const int item_id = combo * H + h;
        if (k0 == 0 && t == 0 && a.split_tiles > 0)
            a.item_parts[item_id] = make_int2(blockIdx.x, whole ? 0 : (int)((item + n - 1) / share) - (int)blockIdx.x + 1);
        l += __shfl_xor(l, 32);
        __syncthreads();
        if (hh == 0) {
            sm_ml[(wave * 32 + n32) * 2] = m;
            sm_ml[(wave * 32 + n32) * 2 + 1] = l;
        }
        float* to = (float*)sm + wave * DT * 32 * PAD;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) to[(32 * dt + 8 * (i / 4) + 4 * hh + (i & 3)) * PAD + n32] = o[dt][i];
        __syncthreads();
        const int quads = D / 4;
        for (int e = t; e < nr * quads; e += 64 * NW) {
            const int rr = e / quads, d = 4 * (e - rr * quads);
            float M = -__builtin_huge_valf(), L = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, sm_ml[(w * 32 + rr) * 2]);
            const float ref = M == -__builtin_huge_valf() ? 0.f : M;
            f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm_ml[(w * 32 + rr) * 2] - ref);
                L += sm_ml[(w * 32 + rr) * 2 + 1] * f;
                const float* from = (const float*)sm + (w * DT * 32 + d) * PAD + rr;
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += from[i * PAD] * f;
            }
            if (!whole) {
                const int64_t row_at = part * RM + rr;
                *(f32x4*)(a.part_o + row_at * D + d) = acc;
                if (d == 0) {
                    a.part_ml[2 * row_at] = M;
                    a.part_ml[2 * row_at + 1] = L;
                }
            } else {
                write_row<T>(a, sq, h, r0 + rr, d, M, L, acc);
            }
        }
        if (a.split_tiles == 0) return;
        __syncthreads();
    }
}

// ---- the parts of a row --------------------------------------------------------------------------
//
// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).  LPR lanes (4 dimensions
// each) take a part; `sub` such groups take a row's parts in turn, each with
// its own maximum, and meet in LDS, so a long list is some loads deep and a
// workgroup has several rows where the lists are short.  The rows kernel
// leaves lists: the first part lies at the end of a share, the others at the
// beginning of the shares that follow.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnParams a, int rm, int sub) {
    __shared__ float sm[256 / LPR][4 * LPR + 2];
    const int g = threadIdx.x / LPR, lane = threadIdx.x % LPR, sg = g % sub;
    const int pair = blockIdx.x, tile = blockIdx.y, b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    const SeqView sq = seq_view(a.c, b);
    const int rows = sq.n * a.group, D = a.c.head_dim, n_in = 256 / LPR / sub;
    const int in = blockIdx.z * n_in + g / sub, r = tile * rm + in;
    if (tile * rm + (int)blockIdx.z * n_in >= rows) return;
    int64_t base, first;   // the part before the second one, and the first
    int parts, step;
    if (a.item_parts) {
        const int2 ip = a.item_parts[((int64_t)b * a.row_tiles + tile) * a.c.kv_heads + h];
        parts = ip.y;
        if (parts == 0) return;   // written by one workgroup
        base = 2 * (int64_t)ip.x;
        first = base + 1;
        step = 2;
    } else {
        parts = a.splits;
        base = first = ((int64_t)pair * a.row_tiles + tile) * a.splits;
        step = 1;
    }
    const bool on = in < rm && r < rows;
    auto place = [&](int s) { return (s == 0 ? first : base + (int64_t)s * step) * rm + in; };
    float M = -__builtin_huge_valf(), L = 0.f;
    f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int d = 4 * lane < D ? 4 * lane : 0;
    for (int s0 = sg; on && s0 < parts; s0 += sub * LPR) {   // LPR parts: a lane has one's maximum and sum
        const int s = s0 + sub * lane, count = min((parts - s0 + sub - 1) / sub, LPR);
        const float2 ml = lane < count ? *(const float2*)(a.part_ml + 2 * place(s)) : make_float2(-__builtin_huge_valf(), 0.f);
        float top = ml.x;
#pragma unroll
        for (int x = LPR / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, LPR));
        top = fmaxf(top, M);
        const float ref = top == -__builtin_huge_valf() ? 0.f : top;
        const float f0 = __builtin_amdgcn_exp2f(M - ref), f = __builtin_amdgcn_exp2f(ml.x - ref);
        M = top;
        L *= f0;
        acc *= f0;
        float sum = ml.y * f;
#pragma unroll
        for (int x = LPR / 2; x; x >>= 1) sum += __shfl_xor(sum, x, LPR);
        L += sum;
        for (int i = 0; i < count; i += 4) {
            f32x4 o[4];
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = min(i + k, count - 1);
                w[k] = __shfl(f, at, LPR);
                o[k] = *(const f32x4*)(a.part_o + place(s0 + sub * at) * D + d);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < count) acc += o[k] * w[k];
        }
    }
    if (sub > 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sm[g][4 * lane + e] = acc[e];
        if (lane == 0) {
            sm[g][4 * LPR] = M;
            sm[g][4 * LPR + 1] = L;
        }
        __syncthreads();
        if (sg != 0) return;
        for (int i = 1; i < sub; ++i) M = fmaxf(M, sm[g + i][4 * LPR]);
        const float ref = M == -__builtin_huge_valf() ? 0.f : M;
        L = 0.f;
        acc = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < sub; ++i) {
            const float f = __builtin_amdgcn_exp2f(sm[g + i][4 * LPR] - ref);
            L += sm[g + i][4 * LPR + 1] * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += sm[g + i][4 * lane + e] * f;
        }
    }
    if (on && 4 * lane < D) write_row<T>(a, sq, h, r, 4 * lane, M, L, acc);
}

// ---- host ---------------------------------------------------------------------------------------

// A page's stride and what its slots span in 32 bits: the chunk kernel's offsets.
static bool short_strides(const tms_cache* c, const int64_t* stride) {
    return 2 * stride[0] < (int64_t)1 << 32 && 2 * stride[2] * c->page_size < (int64_t)1 << 32;
}

// Up to this many tiles a workgroup of eight waves takes an item whole, with
// nothing to join (64 sequences of 40 to 1000 positions: 34 us, 35 in shares;
// one of 500: 12 and 14; one of 1000: 16 and 14).
constexpr int kWholeTiles = 32;

struct AttnPlan {
    bool chunk;        // the chunk kernel
    bool fits;         // its items are counted in 32 bits
    int rm;            // rows a workgroup
    int row_tiles;
    int split_tiles, splits;
    int shares;        // workgroups of the rows kernel
    int waves;         // of one of them
    bool join;
    int rows, most_parts;   // bounds: of a sequence and key head, and of a row's parts
    size_t o_bytes, ml_bytes, item_bytes;
};

static int check_attention(const tms_cache* c, const tms_attention_args* a) {
    const int rc = check_cache(c, true, true);
    if (rc != TMS_OK) return rc;
    if (!a || a->q_heads < 1 || a->q_heads % c->kv_heads || a->sinks < 0 || !std::isfinite(a->scale)) return TMS_ERR_INVALID_ARG;
    for (int i = 0; i < 2; ++i)
        if (a->q_stride[i] < 0 || a->q_stride[i] % 8 || a->out_stride[i] < 0 || a->out_stride[i] % 8) return TMS_ERR_INVALID_ARG;
    if ((int64_t)c->max_q * (a->q_heads / c->kv_heads) > TMS_ATTENTION_MAX_ROWS) return TMS_ERR_CAPACITY;
    if (c->k_stride[2] >= TMS_ATTENTION_MAX_SLOT_STRIDE || c->v_stride[2] >= TMS_ATTENTION_MAX_SLOT_STRIDE) return TMS_ERR_CAPACITY;
    if (c->tokens > 0 && c->batch > 0 && (!a->q || !a->out || !aligned16(a->q) || !aligned16(a->out) || ((uintptr_t)a->lse & 3)))
        return TMS_ERR_INVALID_ARG;
    return TMS_OK;
}

static AttnPlan plan_attention(const tms_cache* c, const tms_attention_args* a) {
    AttnPlan p;
    const int rows = p.rows = min(c->max_q, c->tokens) * (a->q_heads / c->kv_heads);
    p.chunk = rows > kShareRows && short_strides(c, c->k_stride) && short_strides(c, c->v_stride);
    p.rm = p.chunk ? kChunkRows : kShareRows;
    p.row_tiles = (rows + p.rm - 1) / p.rm;
    int64_t keys = min(c->max_kv, kMaxLen);
    if (a->window > 0) keys = std::min<int64_t>(keys, (int64_t)a->window + p.rm + a->sinks + 128);
    const int64_t items = (int64_t)c->batch * c->kv_heads * p.row_tiles;
    int64_t parts;
    p.fits = p.chunk || items <= INT32_MAX;
    p.splits = p.shares = 0;
    p.item_bytes = 0;
    if (p.chunk) {
        // Workgroups enough for two a CU, with 4 tiles each at least.
        const int kt = chunk_keys(c->head_dim);
        const int tiles = (int)((keys + kt - 1) / kt);
        const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(items, 1));
        p.split_tiles = (int)std::max<int64_t>((tiles + want - 1) / want, 4);
        p.splits = std::max(1, (tiles + p.split_tiles - 1) / p.split_tiles);
        p.join = p.splits > 1;
        p.most_parts = p.splits;
        parts = p.join ? items * p.splits : 0;
    } else {
        const int64_t tiles = std::max<int64_t>((keys + 31) / 32, 1);
        p.waves = c->head_dim <= 128 && tiles <= kWholeTiles && items <= 1 << 20 ? 8 : 4;
        p.join = p.waves == 4;
        p.split_tiles = p.join ? kLeastShare : 0;
        p.shares = (int)(p.join ? std::min<int64_t>(c->head_dim > 128 ? 256 : 512, (tiles + kItemCost) * items / kLeastShare) : items);
        parts = p.join ? 2 * (int64_t)p.shares : 0;
        p.most_parts = (int)std::min<int64_t>(tiles / kLeastShare + 2, p.shares);
        p.item_bytes = p.join ? (size_t)(items * 8 + 15) / 16 * 16 : 0;
    }
    p.o_bytes = (size_t)parts * p.rm * c->head_dim * 4;
    p.ml_bytes = (size_t)parts * p.rm * 8;
    return p;
}

template <typename T, int ROWB, int KS, int DT>
static void launch_rows(const AttnPlan& p, const AttnParams& a, hipStream_t stream) {
    if constexpr (ROWB <= 256) {
        if (p.waves == 8) {
            hipLaunchKernelGGL((attn_rows_kernel<T, ROWB, KS, DT, 8>), dim3(p.shares), dim3(512), 0, stream, a);
            return;
        }
    }
    hipLaunchKernelGGL((attn_rows_kernel<T, ROWB, KS, DT, 4>), dim3(p.shares), dim3(256), 0, stream, a);
}

template <typename T, int LPR>
static void launch_join(const AttnPlan& p, const AttnParams& a, int pairs, hipStream_t stream) {
    int sub = 1;
    while (sub < 256 / LPR && sub < p.most_parts) sub *= 2;
    const int n_in = 256 / LPR / sub;
    hipLaunchKernelGGL((attn_join_kernel<T, LPR>), dim3(pairs, p.row_tiles, (std::min(p.rm, p.rows) + n_in - 1) / n_in), dim3(256), 0, stream, a,
                       p.rm, sub);
}

template <typename T>
static void launch_attention(const AttnPlan& p, const AttnParams& a, hipStream_t stream) {
    const int D = a.c.head_dim, pairs = a.c.batch * a.c.kv_heads;
    if (p.chunk) launch_attn_chunk(a, std::is_same<T, Bf16>::value, dim3(pairs, p.row_tiles, p.splits), stream);
    else if (D <= 64) launch_rows<T, 128, 4, 2>(p, a, stream);
    else if (D <= 96) launch_rows<T, 256, 6, 3>(p, a, stream);
    else if (D <= 128) launch_rows<T, 256, 8, 4>(p, a, stream);
    else launch_rows<T, 512, 16, 8>(p, a, stream);
    if (!p.join) return;
    if (D <= 64) launch_join<T, 16>(p, a, pairs, stream);
    else if (D <= 128) launch_join<T, 32>(p, a, pairs, stream);
    else launch_join<T, 64>(p, a, pairs, stream);
}

}  // namespace tms

extern "C" int64_t tms_paged_attention_workspace(const tms_cache* cache, const tms_attention_args* args) {
    const int rc = tms::check_attention(cache, args);
    if (rc != TMS_OK) return rc;
    const tms::AttnPlan p = tms::plan_attention(cache, args);
    if (!p.fits) return TMS_ERR_CAPACITY;
    return (int64_t)(p.o_bytes + p.ml_bytes + p.item_bytes);
}

extern "C" int tms_paged_attention(const tms_cache* cache, const tms_attention_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_attention(cache, args);
    if (rc != TMS_OK) return rc;
    if (cache->batch == 0 || cache->tokens == 0 || cache->max_q == 0) return TMS_OK;
    const AttnPlan p = plan_attention(cache, args);
    if (!p.fits) return TMS_ERR_CAPACITY;
    if (args->workspace_bytes < p.o_bytes + p.ml_bytes + p.item_bytes ||
        (p.join && (!args->workspace || !aligned16(args->workspace))))
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
    a.item_parts = p.chunk ? nullptr : (int2*)((char*)args->workspace + p.o_bytes + p.ml_bytes);
    if (cache->dtype == TMS_DTYPE_BF16) launch_attention<Bf16>(p, a, stream);
    else launch_attention<F16>(p, a, stream);
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}
