// tms_attn_chunk.h -- attention over the paged cache for many rows a key head: one row tile's
// pass over its keys, for chunks of a prompt (tms_attn_chunk.hip) and drafted trees (tms_attn_tree.hip).
#pragma once

#include <type_traits>

#include "tms_attn.h"

namespace tms {

template <int ROWB, int NK, int NW, bool TREE>
struct ChunkShared {
    static constexpr int KT = 32 * NK, NV = ROWB > 256 ? 3 : 2;   // keys of a tile; value buffers
    __attribute__((aligned(128))) char k[2][KT * ROWB];
    __attribute__((aligned(128))) char v[NV][KT * ROWB];
};
template <int ROWB, int NK, int NW>
struct ChunkShared<ROWB, NK, NW, true> : ChunkShared<ROWB, NK, NW, false> {
    TreeRows<32 * NW> tree;
};

// A row tile of one sequence and key head: its list's key tiles [v0, v1), to the output, or as part
// `part` to the workspace (-1: all are there).
template <typename T, int ROWB, int KS, int DT, int NK, int NW, bool TREE>
__device__ __forceinline__ void chunk_item(const AttnParams& a, ChunkShared<ROWB, NK, NW, TREE>& sm, const SeqView& sq, int b, int h, int tile,
                                           const TileList<32 * NK>& tl, int v0, int v1, int64_t part) {
    constexpr int KT = 32 * NK, RM = 32 * NW;
    constexpr int C = ROWB / 16, RPI = 64 / C, NI = KT / (NW * RPI);   // pieces a row; rows a load; loads a wave
    constexpr uint32_t ALL = (1u << KT / 8) - 1;
    constexpr bool FUSED = ROWB > 256;
    static_assert(NK == (FUSED ? 1 : 2), "a tile's keys by 32");
    static_assert(NI * RPI % 8 == 0 && NI * RPI >= 8, "a wave loads whole groups of 8 keys");
    constexpr int NV = ChunkShared<ROWB, NK, NW, TREE>::NV;
    auto& sm_k = sm.k;
    auto& sm_v = sm.v;
    int thread = threadIdx.x;
    if constexpr (TREE) asm volatile("" : "+v"(thread));   // (what follows from it is not kept from item to item)
    const int lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int n32 = lane & 31, hh = lane >> 5;
    const int G = a.group, rows = sq.n * G, r0 = tile * RM;
    const int D = a.c.head_dim;
    // Positions of the workgroup's rows.  A tree's row sees no key past the prefix but its
    // own line, and stands at p0 or behind.
    const int gfirst = TREE ? sq.p0 : sq.p0 + r0 / G, glast = sq.p0 + (min(r0 + RM, rows) - 1) / G, gall = TREE ? sq.p0 - 1 : gfirst;

    // The wave's rows, and the lane's: its query and its position.
    const int w0 = r0 + wave * 32, r = w0 + n32;
    const bool in = r < rows;
    const int pfirst = TREE ? sq.p0 : sq.p0 + w0 / G, plast = w0 < rows ? sq.p0 + (min(w0 + 32, rows) - 1) / G : -1;
    const int tok = in ? r / G : 0, hd = in ? r - tok * G : 0;
    const int pos = in ? sq.p0 + tok : -1;
    // (a share of the prefix alone needs none of the tree, but for a window)
    const bool lines = TREE && (a.window > 0 || (v0 < v1 && tl.key(v1 - 1) + KT > sq.p0));
    [[maybe_unused]] typename TreeRows<RM>::template Parents<64 * NW> parents;
    if constexpr (TREE) {
        if (lines) parents.fetch(a, sq, glast - sq.p0 + 1);
    }
    u32x4 qf[KS];
    {
        const char* src = a.q + (int64_t)(sq.q0 + tok) * a.qt + (int64_t)(h * G + hd) * a.qh;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = query_operand(a, src, s * 16 + hh * 8, in);
    }

    // Loads into LDS: an instruction moves 64 pieces, RPI whole rows, of 8
    // keys that share a resource.  That ends with the last of them that exists,
    // and a page that does not has none: what lies past is written as zeros,
    // and so are the pieces past head_dim.
    const int32_t* row = a.c.tables + (int64_t)b * a.c.tstride;
    const char* kbase = a.c.k + (int64_t)h * a.c.kh;
    const char* vbase = a.c.v + (int64_t)h * a.c.vh;
    const uint32_t lds_k = (uint32_t)(uintptr_t)(lds_void*)&sm_k[0][0], lds_v = (uint32_t)(uintptr_t)(lds_void*)&sm_v[0][0];
    const uint32_t kslot = (uint32_t)a.c.ks, vslot = (uint32_t)a.c.vs, kpage = (uint32_t)a.c.kp, vpage = (uint32_t)a.c.vp;
    uint32_t koff[NI], voff[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int rr = (wave * NI + i) * RPI + lane / C, lc = lane % C;
        const int ck = lc ^ key_swizzle<ROWB>(rr), cv = lc ^ value_swizzle<ROWB>(rr);
        koff[i] = ck * 8 < D ? (rr & 7) * kslot + ck * 16 : 0x80000000u;
        voff[i] = cv * 8 < D ? (rr & 7) * vslot + cv * 16 : 0x80000000u;
    }
    // Table entries of the tile's groups of 8 keys, a lane each; -1 past the end.
    auto entries = [&](int v) {
        const int j = tl.key(v) + 8 * (lane & 7);
        return (unsigned)j < (unsigned)sq.len ? row[j >> a.c.shift] : -1;
    };
    auto load = [&](int v, int kbuf, int vbuf, int pg) __attribute__((always_inline)) {
        const int t0 = tl.key(v);
#pragma unroll
        for (int g = 0; g < NI * RPI / 8; ++g) {
            const int at = wave * NI * RPI + 8 * g, j = t0 + at;
            const uint32_t entry = __builtin_amdgcn_readlane(pg, at / 8);
            const bool ok = entry < (uint32_t)a.c.pages;
            const uint32_t page = ok ? entry : 0, slot = ok ? j & a.c.smask : 0;
            const int last = ok ? min(8, sq.len - j) - 1 : -1;
            const u32x4 kres = slots_rsrc(kbase + (uint64_t)page * kpage + slot * kslot, last, kslot, 2 * D);
            const u32x4 vres = slots_rsrc(vbase + (uint64_t)page * vpage + slot * vslot, last, vslot, 2 * D);
#pragma unroll
            for (int i = g * 8 / RPI; i < (g + 1) * 8 / RPI; ++i) {
                const uint32_t to = (wave * NI + i) * RPI * ROWB;
                load_lds16(kres, koff[i], lds_k + kbuf * KT * ROWB + to);
                load_lds16(vres, voff[i], lds_v + vbuf * KT * ROWB + to);
            }
        }
    };

    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
    float m = -__builtin_huge_valf(), l = 0.f;

    // The parts of a tile's work, by 32 keys.
    auto scores = [&](const char* sk, int kt, f32x16& s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s = T::mfma32(key_operand<ROWB>(sk, lane, kt, ks), qf[ks], s);
    };
    // The reference point lies 2^kLift below the maximum, and follows it once some
    // row's has grown past 2^kMost above: weights stay below that, in either type's range.
    auto refer = [&](float top) __attribute__((always_inline)) {
        top *= a.scale;
        if (__any(top > m + T::kMost)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            top = fmaxf(top - T::kLift, m);
            const float f = __builtin_amdgcn_exp2f(m - (top == -__builtin_huge_valf() ? 0.f : top));
            m = top;
            l *= f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= f;
        }
    };
    auto most = [&](const f32x16& s, float top) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
        return top;
    };
    auto weigh = [&](f32x16& s, u32x4 (&pf)[2]) __attribute__((always_inline)) {
        const float base = m == -__builtin_huge_valf() ? 0.f : m;
        float sum = 0.f;   // (small weights add up before they meet a large sum)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, -base));
            sum += s[e];
        }
        l += sum;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int w = 0; w < 4; ++w) pf[t][w] = T::pack(s[8 * t + 2 * w], s[8 * t + 2 * w + 1]);
    };
    auto outputs = [&](const char* sv, int kt, const u32x4 (&pf)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int t = 0; t < 2; ++t) o[dt] = T::mfma32(value_operand<ROWB>(sv, lane, dt, 2 * kt + t), pf[t], o[dt]);
    };
    const float low = -__builtin_huge_valf();
    // Scores of 32 keys, while the weights of the 32 before (`s`) are worked out
    // and go to the outputs; returns the maximum.  The order is written out: a
    // matrix instruction, some weights, the operands of two steps on.
    auto fused = [&](const char* sk, f32x16& next, f32x16& s, const char* sv) __attribute__((always_inline)) {
        const float base = m == low ? 0.f : m;
        u32x4 kf[3], vf[3], pf[2];
        float sum = 0.f, top = low;
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.f;
        kf[0] = key_operand<ROWB>(sk, lane, 0, 0);
        kf[1] = key_operand<ROWB>(sk, lane, 0, 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (ks + 2 < KS) kf[(ks + 2) % 3] = key_operand<ROWB>(sk, lane, 0, ks + 2);
            else vf[ks + 2 - KS] = value_operand<ROWB>(sv, lane, (ks + 2 - KS) / 2, (ks + 2 - KS) % 2);
            next = T::mfma32(kf[ks % 3], qf[ks], next);
#pragma unroll
            for (int e = 16 * ks / KS; e < 16 * (ks + 1) / KS; ++e) {
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, -base));
                sum += s[e];
                if (e & 1) pf[e / 8][e % 8 / 2] = T::pack(s[e - 1], s[e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i) {
            if (i + 2 < 2 * DT) vf[(i + 2) % 3] = value_operand<ROWB>(sv, lane, (i + 2) / 2, i % 2);
            o[i / 2] = T::mfma32(vf[i % 3], pf[i % 2], o[i / 2]);
            if (i >= 2 * DT - 2) {
#pragma unroll
                for (int e = 8 * (i - 2 * DT + 2); e < 8 * (i - 2 * DT + 3); ++e) top = fmaxf(top, next[e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
        return top;
    };

    // A tile of which some row of the workgroup does not see all.
    auto edge_step = [&](int t0, const char* sk, char* sv, uint32_t there) __attribute__((always_inline)) {
        bool odd = false;
        {
            // Some row has a weight of zero: does the tile hold an infinity or NaN?
#pragma unroll
            for (int i = 0; i < KT * ROWB / 1024; ++i) {
                const u32x4 x = *(const u32x4*)(sv + i * 1024 + lane * 16);
#pragma unroll
                for (int w = 0; w < 4; ++w) odd |= (x[w] & T::kExp) == T::kExp || (x[w] >> 16 & T::kExp) == T::kExp;
            }
            odd = __any(odd);
            const bool none = t0 > plast || (a.window > 0 && t0 + KT <= pfirst - a.window + 1 && t0 >= a.sinks);
            if (none && !odd) return;
        }
        f32x16 s[NK];
        u32x4 pf[NK][2];
        float top = low;
#pragma unroll
        for (int kt = 0; kt < NK; ++kt) {
            scores(sk, kt, s[kt]);
            uint32_t seen = 0;
            if constexpr (TREE) seen = in ? sm.tree.sees(a, sq.p0, tok - r0 / G, t0 + 32 * kt) : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int j = t0 + 32 * kt + 8 * (i / 4) + 4 * hh + (i & 3);
                const bool on = (there >> (4 * kt + i / 4) & 1) && j < sq.len &&
                                (TREE ? seen >> (j - t0 - 32 * kt) & 1 : sees(j, pos, a.window, a.sinks));
                s[kt][i] = on ? s[kt][i] : low;
            }
            top = most(s[kt], top);
        }
        refer(top);
#pragma unroll
        for (int kt = 0; kt < NK; ++kt) weigh(s[kt], pf[kt]);
        {
            // A weight of zero times an infinity or NaN would reach rows that
            // do not see the value: such values go, key by key, to the rows whose
            // weight is not zero (which weight does not matter), and are zero in
            // the product.
            if (odd) {
                uint32_t mine = 0;
#pragma unroll
                for (int e = 0; e < 16 * NK; ++e) mine |= s[e / 16][e % 16] != 0.f ? 1u << e : 0u;
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
                __syncthreads();
                for (int i = thread; i < KT * ROWB / 16; i += 64 * NW) {
                    u32x4 x = *(const u32x4*)(sv + 16 * i);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        if ((x[w] & T::kExp) == T::kExp) x[w] &= 0xFFFF0000u;
                        if ((x[w] >> 16 & T::kExp) == T::kExp) x[w] &= 0x0000FFFFu;
                    }
                    *(u32x4*)(sv + 16 * i) = x;
                }
                __syncthreads();
            }
        }

#pragma unroll
        for (int kt = 0; kt < NK; ++kt) outputs(sv, kt, pf[kt]);
    };

    int pg = v0 < v1 ? entries(v0) : -1, ahead = v0 + 1 < v1 ? entries(v0 + 1) : -1;
    uint32_t there = (uint32_t)__ballot((unsigned)pg < (unsigned)a.c.pages) & ALL;
    if (v0 < v1) load(v0, 0, 0, pg);
    if constexpr (TREE) {
        if (lines) sm.tree.find(a, sq, r0 / G, glast - sq.p0 - r0 / G + 1, parents);
    }
    int v = v0, kb = 0, vb = 0;   // the tile, its key and value buffers
    // Takes tile v when it has come: the wave's loads are in, and after the
    // barrier all are, and the buffers that the next tile's go to are free: no wave
    // has left to do but the last values of the tile before.
    uint32_t now = 0;
    auto arrive = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        pg = ahead;
        now = there;
        there = (uint32_t)__ballot((unsigned)pg < (unsigned)a.c.pages) & ALL;
        __syncthreads();
        if (v + 1 < v1) load(v + 1, kb ^ 1, vb == NV - 1 ? 0 : vb + 1, pg);
        if (v + 2 < v1) ahead = entries(v + 2);
    };
    auto advance = [&]() __attribute__((always_inline)) {
        ++v;
        kb ^= 1;
        vb = vb == NV - 1 ? 0 : vb + 1;
    };
    auto is_edge = [&](int t0, uint32_t bits) {
        return bits != ALL || t0 + KT > sq.len || t0 + KT - 1 > gall || (a.window > 0 && t0 <= glast - a.window && t0 + KT > a.sinks);
    };
    while (v < v1) {
        // Tiles that every row sees all of.
        if constexpr (FUSED) {
            if (!is_edge(tl.key(v), there)) {
                f32x16 sa, sb;
                u32x4 pf[2];
                arrive();
                scores(sm_k[kb], 0, sa);
                refer(most(sa, low));
                for (;;) {
                    sb = sa;
                    if (v + 1 >= v1 || is_edge(tl.key(v + 1), there)) break;
                    const char* before = sm_v[vb];
                    advance();
                    arrive();
                    refer(fused(sm_k[kb], sa, sb, before));
                }
                weigh(sb, pf);
                outputs(sm_v[vb], 0, pf);
                advance();
            }
        } else {
            // The products' operands are read three steps ahead, the second 32 keys'
            // weights are worked out among the first's outputs, and a wave in its
            // products goes before one in its weights: the two workgroups of a CU
            // fall into turns (2048 new tokens over 16384, 32 heads of 8 of 128: 499 us with
            // the operands ahead alone, 493 with the weights between, 473 with all).
            while (v < v1 && !is_edge(tl.key(v), there)) {
                f32x16 s[NK];
                u32x4 pf[NK][2], kf[4], vf[4];
                float top = low, sum = 0.f, w[16];
                arrive();
                const char* sk = sm_k[kb];
                const char* sv = sm_v[vb];
#pragma unroll
                for (int kt = 0; kt < NK; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < 3; ++i) kf[i] = key_operand<ROWB>(sk, lane, i % NK, i / NK);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NK * KS; ++i) {
                    if (i + 3 < NK * KS) kf[(i + 3) % 4] = key_operand<ROWB>(sk, lane, (i + 3) % NK, (i + 3) / NK);
                    s[i % NK] = T::mfma32(kf[i % 4], qf[i / NK], s[i % NK]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
#pragma unroll
                for (int kt = 0; kt < NK; ++kt) top = most(s[kt], top);
                refer(top);
                weigh(s[0], pf[0]);
                const float base = m == low ? 0.f : m;
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < 3; ++i) vf[i] = value_operand<ROWB>(sv, lane, i % DT, i / DT);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 2 * NK * DT; ++i) {
                    if (i + 3 < 2 * NK * DT) vf[(i + 3) % 4] = value_operand<ROWB>(sv, lane, (i + 3) % DT, (i + 3) / DT);
                    o[i % DT] = T::mfma32(vf[i % 4], pf[i / DT / 2][i / DT % 2], o[i % DT]);
                    if (i < 2 * DT) {
#pragma unroll
                        for (int e = 16 * i / (2 * DT); e < 16 * (i + 1) / (2 * DT); ++e) {
                            w[e] = __builtin_amdgcn_exp2f(fmaf(s[1][e], a.scale, -base));
                            sum += w[e];
                            if (e & 1) pf[1][e / 8][e % 8 / 2] = T::pack(w[e - 1], w[e]);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_s_setprio(0);
                l += sum;
                advance();
            }
        }
        while (v < v1 && is_edge(tl.key(v), there)) {
            arrive();
            edge_step(tl.key(v), sm_k[kb], sm_v[vb], now);
            advance();
        }
    }
    l += __shfl_xor(l, 32);
    if (!in) return;

    if (part >= 0) {
        const int64_t at = part * RM + (r - r0);
        if (hh == 0) {
            a.part_ml[2 * at] = m;
            a.part_ml[2 * at + 1] = l;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int d = 32 * dt + 8 * c + 4 * hh;
                if (d < D)
                    *(f32x4*)(a.part_o + at * D + d) =
                        (f32x4){o[dt][4 * c], o[dt][4 * c + 1], o[dt][4 * c + 2], o[dt][4 * c + 3]};
            }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;   // (a NaN sum stays one)
    if (a.lse && hh == 0) a.lse[(int64_t)(sq.q0 + tok) * a.q_heads + h * G + hd] = (m + log2f(l)) * kLn2;
    char* dst = a.out + (int64_t)(sq.q0 + tok) * a.ot + (int64_t)(h * G + hd) * a.oh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = 32 * dt + 8 * c + 4 * hh;
            if (d < D)
                *(u32x2*)(dst + 2 * d) = (u32x2){T::pack(o[dt][4 * c] * inv, o[dt][4 * c + 1] * inv),
                                                 T::pack(o[dt][4 * c + 2] * inv, o[dt][4 * c + 3] * inv)};
        }
}

}  // namespace tms
