// tms_attn.h -- what the attention and the score kernels share: the 16-bit
// types' matrix instructions, a call's parameters, and which key tiles a
// group of rows sees.
#pragma once

#include "tms_cache.h"

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
    float scale;           // above 0, times log2(e): exponentials are taken to base 2
    uint32_t qand, qxor;   // a query's bits are taken through these: a scale below 0 flips its sign, 0 clears it
    int split_tiles;       // key tiles a split has
    int splits;
    int row_tiles;
    float* part_o;         // [pairs * row_tiles][splits][rows a tile][head_dim]
    float* part_ml;        // [pairs * row_tiles][splits][rows a tile][2]: maximum, sum
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

// The scale of a call, split into one above 0 and what becomes of the query:
// masked scores are -inf before the scale and stay so.
inline void set_scale(AttnParams& a, float scale) {
    a.qand = scale == 0.f ? 0u : ~0u;
    a.qxor = scale < 0.f ? 0x80008000u : 0u;
    a.scale = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * kLog2e;
}

constexpr int kChunkRows = 128;   // of a workgroup of the chunk kernel
inline int chunk_keys(int head_dim) { return head_dim > 128 ? 32 : 64; }   // of its tile
constexpr float kSlack = 8.f;
void launch_attn_chunk(const AttnParams& a, bool bf16, dim3 grid, hipStream_t stream);

__device__ __forceinline__ bool sees(int j, int p, int window, int sinks) {
    return j <= p && (window <= 0 || j > p - window || j < sinks);
}

}  // namespace tms
