// tms_attn.h -- what the attention and the score kernels share: the 16-bit
// types' matrix instructions, a call's parameters, and which key tiles a
// group of rows sees.
#pragma once

#include <algorithm>
#include <limits>

#include "tms_cache.h"
#include "../../include/tmtree_hip.h"

namespace tms {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Bf16 {
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {   // to nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, bf16x2));
    }
    static __device__ __forceinline__ float up(uint32_t bits16) { return __uint_as_float(bits16 << 16); }
    static constexpr uint32_t kExp = 0x7F80u;   // exponent bits: all set in infinities and NaN
    static constexpr float kLift = 0.f, kMost = 8.f;   // of a weight's exponent: a row's largest, and what it may grow to
};

struct F16 {
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {   // to nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){lo, hi}, f16x2));
    }
    static __device__ __forceinline__ float up(uint32_t bits16) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
    }
    static constexpr uint32_t kExp = 0x7C00u;
    // Below 2^-14 the type has fewer bits and below 2^-25 none, above it nearly 2^16:
    // a row's largest weight is taken as 2^11, so that one 2^-25 of it has all bits yet.
    static constexpr float kLift = 11.f, kMost = 15.f;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnParams {
    CacheView c;
    const char* q;
    char* out;
    float* lse;            // attention: written; scores: read
    float* score_out;
    int64_t qt, qh;        // bytes between tokens, heads
    int64_t ot, oh;
    int group, q_heads;
    int window, sinks;     // window 0: none
    int max_kv;            // scores: positions past it are left out
    float scale;           // above 0, times log2(e): exponentials are taken to base 2
    uint32_t qand, qxor;   // a query's bits are taken through these: a scale below 0 flips its sign, 0 clears it
    int split_tiles;       // chunk kernel: key tiles a split has; rows kernel and trees: the least that a share has
    int splits;            // chunk kernel
    int row_tiles;
    float* part_o;         // parts of rows, [part][rows a tile][head_dim]
    float* part_ml;        // [part][rows a tile][2]: maximum, sum
    int2* item_parts;      // rows kernel and trees, [pairs * row_tiles]: the first share and the number of shares with a part
    const int32_t* parents;   // trees
};

// The key tiles of `KT` keys that the rows at positions [pmin, pmax] see, as
// a list of `n`: the sinks' tiles that lie before the window's first tile,
// `lo`, then [lo, end).  A row of the group may see none of a tile.
template <int KT>
struct TileList {
    int sink, lo, n;
    __device__ __forceinline__ TileList(int window, int sinks, int pmin, int pmax, int len) {
        const int end = (min(pmax + 1, len) + KT - 1) / KT;
        lo = 0;
        sink = 0;
        if (window > 0) {
            lo = min(max(max(pmin, 0) - window + 1, 0) / KT, max(end, 0));
            sink = min((min(sinks, len) + KT - 1) / KT, lo);
        }
        n = max(sink + end - lo, 0);
    }
    __device__ __forceinline__ int key(int i) const { return (i < sink ? i : i - sink + lo) * KT; }
};

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// A tile lies in LDS by rows of `ROWB` bytes, a key's (value's) 16-byte pieces
// permuted within its row so that the reads of the matrix operands fall on
// different banks: the key operand takes one piece of 32 rows, the value
// operand (transposed on the way, ds_read_b64_tr_b16) 64 bytes of 4 rows.
template <int ROWB> __device__ __forceinline__ int key_swizzle(int row) { return ROWB == 128 ? row >> 1 & 7 : row & 15; }
template <int ROWB> __device__ __forceinline__ int value_swizzle(int row) { return ROWB == 128 ? (row >> 1 & 1) << 2 : (row & 3) << 2; }

// 16 bytes a lane from `off` of the resource to LDS at `lds` (wave-uniform) +
// 16 * lane; zeros where the resource ends before.  Counted by vmcnt only:
// the loop waits for it, the compiler does not know of it.  (A wait state
// lies between m0's write and the load that reads it.  m0 is reserved: the compiler
// keeps nothing in it and takes no clobber of it, and nothing else in these kernels uses it.)
__device__ __forceinline__ void load_lds16(u32x4 rsrc, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory");
}

// The resource of the last + 1 slots at `p`, none of them where `last` < 0.
__device__ __forceinline__ u32x4 slots_rsrc(const char* p, int last, uint32_t stride, int bytes) {
    const uint64_t at = (uint64_t)p;
    return (u32x4){(uint32_t)at, (uint32_t)(at >> 32) & 0xFFFF, last < 0 ? 0u : (uint32_t)(last * stride + bytes), 0x00020000u};
}

// Row r as token and head of its group, r below 2^21: a product with 1 / G is off
// by one at most.
__device__ __forceinline__ void split_row(int r, int G, float inv, int& tok, int& hd) {
    tok = (int)((float)r * inv);
    hd = r - tok * G;
    if (hd < 0) {
        --tok;
        hd += G;
    } else if (hd >= G) {
        ++tok;
        hd -= G;
    }
}

// A row's 8 values from dimension d on as the operand of the scores, zeros
// past head_dim and for a row that is none (`src` is some row in any case:
// loads without a branch between them are in flight together).
__device__ __forceinline__ u32x4 query_operand(const AttnParams& a, const char* src, int d, bool in) {
    const bool is = in && d < a.c.head_dim;
    const u32x4 x = *(const u32x4*)(src + 2 * (d < a.c.head_dim ? d : 0));
    u32x4 y;
#pragma unroll
    for (int w = 0; w < 4; ++w) y[w] = is ? (x[w] & a.qand) ^ a.qxor : 0u;
    return y;
}

// The operand of S^T = K Q^T: 32 keys from `tile` on, dimensions 16 ks...
template <int ROWB> __device__ __forceinline__ u32x4 key_operand(const char* sk, int lane, int tile, int ks) {
    const int key = tile * 32 + (lane & 31);
    return *(const u32x4*)(sk + key * ROWB + 16 * ((2 * ks + (lane >> 5)) ^ key_swizzle<ROWB>(key)));
}

// The operand of O^T = V^T P^T: value columns 32 dt..., the keys of weights
// 8 t .. 8 t + 7 of a lane, which are 16 t + 4 (lane / 32) + 0..3 and 8 more on.
template <int ROWB> __device__ __forceinline__ u32x4 value_operand(const char* sv, int lane, int dt, int t) {
    const int q16 = lane & 15;
    u32x4 vf;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int key = 16 * t + 8 * u + 4 * (lane >> 5) + (q16 >> 2);
        const int piece = 4 * dt + 2 * (lane >> 4 & 1) + (q16 >> 1 & 1);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4*)(sv + key * ROWB + 16 * (piece ^ value_swizzle<ROWB>(key)) + 8 * (q16 & 1)));
        const u32x2 y = __builtin_bit_cast(u32x2, x);
        vf[2 * u] = y[0];
        vf[2 * u + 1] = y[1];
    }
    return vf;
}

// The scale of a call, split into one above 0 and what becomes of the query:
// masked scores are -inf before the scale and stay so.  (A scale near the type's
// largest number stays finite: a score of 0 stays 0.)
inline void set_scale(AttnParams& a, float scale) {
    a.qand = scale == 0.f ? 0u : ~0u;
    a.qxor = scale < 0.f ? 0x80008000u : 0u;
    a.scale = scale == 0.f ? 1.f : std::min((scale < 0.f ? -scale : scale) * kLog2e, std::numeric_limits<float>::max());
}

constexpr int kChunkRows = 128;   // of a workgroup of the chunk kernel
inline int chunk_keys(int head_dim) { return head_dim > 128 ? 32 : 64; }   // of its tile
void launch_attn_chunk(const AttnParams& a, bool bf16, dim3 grid, hipStream_t stream);
void launch_attn_chunk_tree(const AttnParams& a, bool bf16, int rows, int workgroups, hipStream_t stream);   // `rows` of a workgroup

__device__ __forceinline__ bool sees(int j, int p, int window, int sinks) {
    return j <= p && (window <= 0 || j > p - window || j < sinks);
}

// Trees in the chunk kernel: all items (sequence, row tile, key head) lie behind each other on
// one axis of key tiles, and each workgroup takes an equal share of it, as in the rows kernel
// (8 sequences of 9000 to 16384, trees of 64 nodes, on one card: 142 us; 160 with four splits of each sequence, 184
// with as many splits as its length asks for, which leaves a second round of workgroups).
// An item takes kTreeItemCost tiles besides its own.
constexpr int kTreeItemCost = 4, kTreeLeastShare = 4;
template <int KT, int RM>
struct TreeAxis {
    static __device__ __forceinline__ int tiles(const AttnParams& a, const SeqView& sq, int tile) {
        const int last = min((tile + 1) * RM, sq.n * a.group) - 1;
        return TileList<KT>(a.window, a.sinks, sq.p0, sq.p0 + last / a.group, sq.len).n;
    }
    static __device__ __forceinline__ int length(int tiles) { return max(tiles, 1) + kTreeItemCost; }
    // A sequence's row tile's share of the axis, for one key head.
    static __device__ __forceinline__ int combo(const AttnParams& a, int c) {
        const int b = c / a.row_tiles, tile = c - b * a.row_tiles;
        const SeqView sq = seq_view(a.c, b);
        return tile * RM < sq.n * a.group ? length(tiles(a, sq, tile)) : 0;
    }
};

// A barrier for what goes through LDS alone: loads in flight stay so.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Trees: what the tokens of a group of rows see of the new tokens, a bit each, found by
// climbing from node to parent in LDS (some 100 cycles a step), and their depths.  With a
// window a node's own line is cut by it here, and climbed twice.  A workgroup climbs for each item of whose new tokens it
// has keys, so deep lines show (4 heads a key head of 128, a chain and a tree one deep, 508 positions before it: 64 nodes
// 34 and 27 us, 512 nodes 99 and 43, with a window of 256 113 and 39; 16 sequences of 512 nodes after 2000 534 and 384).
constexpr int kTreeWords = TMS_TREE_MAX_NODES / 32;
template <int TOKENS>
struct TreeRows {
    int16_t up[TMS_TREE_MAX_NODES];
    uint32_t seen[TOKENS][kTreeWords + 1];
    int depth[TOKENS];

    // The parents of nodes below `end`, a thread's in registers: on the way with the queries, and in LDS
    // while the first keys come.
    template <int NT>
    struct Parents {
        int up[TMS_TREE_MAX_NODES / NT];
        __device__ __forceinline__ void fetch(const AttnParams& a, const SeqView& sq, int end) {
#pragma unroll
            for (int k = 0; k < TMS_TREE_MAX_NODES / NT; ++k) {
                const int i = k * NT + (int)threadIdx.x;
                up[k] = i < end ? a.parents[sq.q0 + i] : -1;
            }
        }
    };

    // What tokens [tok0, tok0 + n) of the sequence see; by all threads of the workgroup.
    template <int NT>
    __device__ __forceinline__ void find(const AttnParams& a, const SeqView& sq, int tok0, int n, const Parents<NT>& p) {
        const int t = threadIdx.x;
#pragma unroll
        for (int k = 0; k < TMS_TREE_MAX_NODES / NT; ++k) {
            const int i = k * NT + t;
            up[i] = (int16_t)(p.up[k] >= 0 && p.up[k] < i ? p.up[k] : -1);
        }
        lds_barrier();
        for (int i = t; i < n; i += NT) {
            for (int w = 0; w <= kTreeWords; ++w) seen[i][w] = 0;
            int far = 0;
            if (a.window > 0)
                for (int x = up[tok0 + i]; x >= 0; x = up[x]) ++far;
            depth[i] = far;
            int back = 0;
            for (int x = tok0 + i; x >= 0; x = up[x], ++back)
                if (a.window <= 0 || back < a.window || sq.p0 + far - back < a.sinks) seen[i][x >> 5] |= 1u << (x & 31);
        }
        lds_barrier();
    }

    // Bit e: token `i` of these sees key t0 + e.
    __device__ __forceinline__ uint32_t sees(const AttnParams& a, int p0, int i, int t0) const {
        const int first = t0 - p0;   // the node that the first key is
        uint32_t m = ~0u;
        if (first >= 0) {
            const int w = min(first >> 5, kTreeWords), s = first & 31;
            m = (uint32_t)(((uint64_t)(w < kTreeWords ? seen[i][w + 1] : 0u) << 32 | seen[i][w]) >> s);
        } else if (first > -32) {
            m = seen[i][0] << -first | ((1u << -first) - 1);
        }
        if (a.window > 0) {   // the prefix ends with p0, and is hidden from `sinks` to the window
            const int lo = max(a.sinks - t0, 0), hi = min(min(p0 + depth[i] - a.window, p0 - 1) - t0, 31);
            if (lo <= hi) m &= ~((~0u >> (31 - (hi - lo))) << lo);
        }
        return m;
    }
};

}  // namespace tms
