// tms_rotary.hip -- rotary positions: heads turned by their tokens' positions
// (tms_rotary), and the same on the way into the paged cache (tms_kv_append_rotary).
//
// Pair (x, y) of angle a = position * frequency becomes (x cos a - y sin a, y cos a +
// x sin a).  At positions of some 10^6 an fp32 angle is off by a tenth of a radian, so the
// angle is reduced in fp64, as quarter turns k + r, |r| <= 1/2; cos and sin of r pi / 2 are
// their Taylor series (to r^10 and r^9: off by 2^-25 at most) in fp32.
//
// Bound by memory for a prompt, by latency for a decode step.  An angle serves all of a
// token's heads: a thread takes one unit (16 bytes, with two halves 2 x 16) of several heads.
// 16385 tokens, 32 + 8 heads of 128, bf16, pairs, 336 MB: 63 us, 5.3 TB/s.  Into the cache, half
// layout, 7 prompts of 333 to 2381 tokens, fp16, 234 MB: 58 us, 4.0 TB/s, with two heads' loads ahead (63 with one, 65 with
// four; 135 with turning and copying by the same threads, whose registers then hold both).  The 64 tokens of a
// decode step: 7 us, of which the kernel has 4.
#include <algorithm>
#include <cmath>

#include "tms_cache.h"
#include "../../include/tmtree_hip.h"

namespace tms {

struct TurnParams {
    CacheView c;              // append alone
    const char* x;            // queries
    char* out;
    const char* k;
    const char* v;
    int64_t xt, xh, ot, oh;   // bytes between tokens, heads
    int64_t kt, kh, vt, vh;
    const int32_t* positions;
    const float* freqs;
    float scale;
    int tokens, q_heads, heads;   // heads: keys too
    int head_dim, rotary_dim;
    int groups;               // a thread that turns takes every groups-th head
    int turned, ends, odd;    // units of a head that turn, and that are copied: `odd` of these single values
    int copies;               // threads of a token that copy
    int turn_blocks;          // of a sequence
};

typedef uint16_t u16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct TurnF32 {
    typedef float elem;
    static constexpr int kPiece = 4;   // values in 16 bytes
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
struct TurnF16 {
    typedef u16 elem;
    static constexpr int kPiece = 8;
    static __device__ __forceinline__ float up(u16 x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ u16 down(float x) { return __builtin_bit_cast(u16, (_Float16)x); }
};
struct TurnBf16 {
    typedef u16 elem;
    static constexpr int kPiece = 8;
    static __device__ __forceinline__ float up(u16 x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ u16 down(float x) { return __builtin_bit_cast(u16, (__bf16)x); }
};

// cos and sin of `position` * f, f in quarter turns a position.  An angle past fp64's
// whole numbers, or none, gives some cosine or NaN.
__device__ __forceinline__ void turn_of(double position, double f, float scale, float& co, float& si) {
    const double q = position * f, t = q - 4.0 * rint(0.25 * q);   // |t| <= 2
    const double k = rint(t);
    const float r = (float)(t - k) * 1.57079632679489662f, z = r * r;
    float s = fmaf(z, 1.f / 362880, -1.f / 5040), c = fmaf(z, -1.f / 3628800, 1.f / 40320);
    s = fmaf(z, s, 1.f / 120);
    c = fmaf(z, c, -1.f / 720);
    s = fmaf(z, s, -1.f / 6);
    c = fmaf(z, c, 1.f / 24);
    s = fmaf(r * z, s, r);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.f);
    const int quarter = (int)k & 3;
    co = quarter & 1 ? s : c;
    si = quarter & 1 ? c : s;
    co = (quarter == 1 || quarter == 2 ? -co : co) * scale;
    si = (quarter >= 2 ? -si : si) * scale;
}

// E values a piece (1: a value at a time, where the pairs do not fall on 16-byte pieces).
// In the half layout a unit is piece u and the one rotary_dim / 2 on, in pairs it is one
// piece (two values with E = 1).
template <typename T, bool PAIRS, int E, bool APPEND>
__global__ __launch_bounds__(256) void turn_kernel(TurnParams a) {
    typedef typename T::elem elem;
    constexpr int NP = PAIRS && E == 1 ? 2 : E;          // values in a turned unit's piece
    constexpr int ANGLES = PAIRS ? NP / 2 : E, AHEAD = PAIRS ? 4 : 2;   // heads whose loads are in flight
    typedef elem Piece __attribute__((ext_vector_type(NP), aligned(E == 1 ? sizeof(elem) : 16)));
    // The last blocks of a sequence copy: values, and the heads' ends that do not turn.
    const bool copies = blockIdx.x >= (unsigned)a.turn_blocks;
    const int b = APPEND ? blockIdx.y : 0;
    SeqView sq;
    if constexpr (APPEND) sq = seq_view(a.c, b);
    else sq = SeqView{0, a.tokens, 0, 0};
    const int per = copies ? a.copies : a.groups * a.turned;   // a token's threads
    const int64_t start = (int64_t)(blockIdx.x - (copies ? a.turn_blocks : 0)) * 256, tok0 = start / per;
    const int at = (int)(start - tok0 * per) + (int)threadIdx.x, more = at / per, w = at - more * per;
    const int64_t i64 = tok0 + more;
    if (i64 >= sq.n) return;
    const int i = (int)i64;
    const int64_t tok = sq.q0 + i;
    int page = -1, slot = 0;
    if constexpr (APPEND) {
        page = page_of(a.c, a.c.tables + (int64_t)b * a.c.tstride, sq.p0 + i, sq.len);
        slot = (sq.p0 + i) & a.c.smask;
    }
    auto source = [&](int h) {
        return APPEND && h >= a.q_heads ? a.k + tok * a.kt + (h - a.q_heads) * a.kh : a.x + tok * a.xt + h * a.xh;
    };
    auto target = [&](int h) {
        return APPEND && h >= a.q_heads ? a.c.k + (int64_t)page * a.c.kp + (h - a.q_heads) * a.c.kh + (int64_t)slot * a.c.ks
                                        : a.out + tok * a.ot + h * a.oh;
    };
    auto is = [&](int h) { return h < a.heads && (!APPEND || h < a.q_heads || page >= 0); };

    if (copies) {
        const int ends = a.heads * a.ends;
        if (w < ends) {   // the values up to whole pieces one by one, then those
            const int h = w / a.ends, u = w - h * a.ends;
            if (!is(h)) return;
            if (u < a.odd) *((elem*)target(h) + a.rotary_dim + u) = *((const elem*)source(h) + a.rotary_dim + u);
            else {
                const int e = a.rotary_dim + a.odd + (u - a.odd) * T::kPiece;
                *(u32x4*)(target(h) + e * sizeof(elem)) = *(const u32x4*)(source(h) + e * sizeof(elem));
            }
        } else if constexpr (APPEND) {   // 16 bytes of a value
            const int hv = a.head_dim / 8, p = w - ends, h = p / hv, d = p - h * hv;
            const u32x4 y = *(const u32x4*)(a.v + tok * a.vt + h * a.vh + 16 * d);
            if (page < 0) return;
            *(u32x4*)(a.c.v + (int64_t)page * a.c.vp + h * a.c.vh + (int64_t)slot * a.c.vs + 16 * d) = y;
            if (d == 0 && a.c.scores) a.c.scores[(((int64_t)page * a.c.kv_heads + h) << a.c.shift) + slot] = 0.f;
        }
        return;
    }
    const int g = w / a.turned, u = w - g * a.turned;
    const int lo = u * NP, hi = lo + a.rotary_dim / 2;   // first values of the unit's pieces
    float co[ANGLES], si[ANGLES];
    {
        const double position = a.positions ? a.positions[tok] : sq.p0 + i;
#pragma unroll
        for (int e = 0; e < ANGLES; ++e)
            turn_of(position, (double)a.freqs[u * ANGLES + e] * 0.63661977236758134308, a.scale, co[e], si[e]);
    }
    for (int h0 = g; h0 < a.heads; h0 += AHEAD * a.groups) {
        Piece y[AHEAD][PAIRS ? 1 : 2];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
            if (is(h0 + n * a.groups)) {
                const char* s = source(h0 + n * a.groups);
                y[n][0] = *(const Piece*)(s + lo * sizeof(elem));
                if constexpr (!PAIRS) y[n][1] = *(const Piece*)(s + hi * sizeof(elem));
            }
#pragma unroll
        for (int n = 0; n < AHEAD; ++n)
            if (is(h0 + n * a.groups)) {
                char* d = target(h0 + n * a.groups);
#pragma unroll
                for (int e = 0; e < ANGLES; ++e) {
                    constexpr int Y = PAIRS ? 0 : 1;
                    const int ex = PAIRS ? 2 * e : e, ey = PAIRS ? 2 * e + 1 : e;
                    const float vx = T::up(y[n][0][ex]), vy = T::up(y[n][Y][ey]);
                    y[n][0][ex] = T::down(fmaf(vx, co[e], -(vy * si[e])));
                    y[n][Y][ey] = T::down(fmaf(vy, co[e], vx * si[e]));
                }
                *(Piece*)(d + lo * sizeof(elem)) = y[n][0];
                if constexpr (!PAIRS) *(Piece*)(d + hi * sizeof(elem)) = y[n][1];
            }
    }
}

// One head a thread while the card has room for more threads, up to eight past that.
static void divide(TurnParams& a, int piece, bool pairs, bool wide, int64_t tokens) {
    const int e = wide ? piece : 1;
    a.turned = pairs ? a.rotary_dim / (wide ? e : 2) : a.rotary_dim / 2 / e;
    a.odd = (piece - a.rotary_dim % piece) % piece;
    a.ends = a.odd + (a.head_dim - a.rotary_dim - a.odd) / piece;
    a.groups = std::max(a.heads, 1);
    while (a.groups > (a.heads + 7) / 8 && tokens * a.turned * a.groups > 1 << 18) a.groups = (a.groups + 1) / 2;
}

template <typename T, bool PAIRS, bool APPEND>
static void launch_turn(const TurnParams& a, bool wide, dim3 grid, hipStream_t stream) {
    if (wide) hipLaunchKernelGGL((turn_kernel<T, PAIRS, T::kPiece, APPEND>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((turn_kernel<T, PAIRS, 1, APPEND>), grid, dim3(256), 0, stream, a);
}

template <bool APPEND>
static int launch_turns(TurnParams& a, int dtype, bool pairs, int64_t tokens, int batch, hipStream_t stream) {
    const int piece = dtype == TMS_DTYPE_F32 ? 4 : 8;
    const bool wide = (pairs ? a.rotary_dim : a.rotary_dim / 2) % piece == 0;
    divide(a, piece, pairs, wide, tokens * batch);
    a.copies = a.heads * a.ends + (APPEND ? a.c.kv_heads * (a.head_dim / 8) : 0);
    const int64_t turn_blocks = (tokens * a.groups * a.turned + 255) / 256, blocks = turn_blocks + (tokens * a.copies + 255) / 256;
    if (blocks >= 1 << 24) return TMS_ERR_CAPACITY;   // a launch has fewer than 2^32 threads
    a.turn_blocks = (int)turn_blocks;
    const dim3 grid((unsigned)blocks, (unsigned)batch);
    if (dtype == TMS_DTYPE_F32) {
        if constexpr (!APPEND) {
            if (pairs) launch_turn<TurnF32, true, false>(a, wide, grid, stream);
            else launch_turn<TurnF32, false, false>(a, wide, grid, stream);
        }
    } else if (dtype == TMS_DTYPE_F16) {
        if (pairs) launch_turn<TurnF16, true, APPEND>(a, wide, grid, stream);
        else launch_turn<TurnF16, false, APPEND>(a, wide, grid, stream);
    } else {
        if (pairs) launch_turn<TurnBf16, true, APPEND>(a, wide, grid, stream);
        else launch_turn<TurnBf16, false, APPEND>(a, wide, grid, stream);
    }
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}

static bool bad_stride(const int64_t* s, int n) {
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || s[i] % 8) return true;
    return false;
}

// An output that is the input has its strides.
static bool bad_output(const void* x, const int64_t* xs, const void* out, const int64_t* os) {
    return x == out && (xs[0] != os[0] || xs[1] != os[1]);
}

static bool bad_rotary(int rotary_dim, int head_dim, int interleaved, float scale) {
    return rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim || (interleaved != 0 && interleaved != 1) || !std::isfinite(scale);
}

}  // namespace tms

extern "C" int tms_rotary(const tms_rotary_args* args, hipStream_t stream) {
    using namespace tms;
    if (!args || args->reserved != 0) return TMS_ERR_INVALID_ARG;
    if (args->dtype != TMS_DTYPE_F32 && args->dtype != TMS_DTYPE_F16 && args->dtype != TMS_DTYPE_BF16) return TMS_ERR_INVALID_ARG;
    if (args->tokens < 0 || args->heads < 0 || args->head_dim < 8 || args->head_dim % 8) return TMS_ERR_INVALID_ARG;
    if (bad_rotary(args->rotary_dim, args->head_dim, args->interleaved, args->scale)) return TMS_ERR_INVALID_ARG;
    if (bad_stride(args->x_stride, 2) || bad_stride(args->out_stride, 2)) return TMS_ERR_INVALID_ARG;
    if (args->head_dim > TMS_ROTARY_MAX_HEAD_DIM || args->heads > TMS_ROTARY_MAX_HEADS || args->tokens > TMS_CACHE_MAX_TOKENS)
        return TMS_ERR_CAPACITY;
    if (args->tokens == 0 || args->heads == 0) return TMS_OK;
    if (!args->x || !args->out || !aligned16(args->x) || !aligned16(args->out) || !args->positions || !args->freqs ||
        ((uintptr_t)args->positions & 3) || ((uintptr_t)args->freqs & 3))
        return TMS_ERR_INVALID_ARG;
    if (bad_output(args->x, args->x_stride, args->out, args->out_stride)) return TMS_ERR_INVALID_ARG;
    const int size = args->dtype == TMS_DTYPE_F32 ? 4 : 2;
    TurnParams a{};
    a.x = (const char*)args->x;
    a.out = (char*)args->out;
    a.xt = size * args->x_stride[0];
    a.xh = size * args->x_stride[1];
    a.ot = size * args->out_stride[0];
    a.oh = size * args->out_stride[1];
    a.positions = args->positions;
    a.freqs = args->freqs;
    a.scale = args->scale;
    a.tokens = args->tokens;
    a.q_heads = a.heads = args->heads;
    a.head_dim = args->head_dim;
    a.rotary_dim = args->rotary_dim;
    return launch_turns<false>(a, args->dtype, args->interleaved != 0, args->tokens, 1, stream);
}

extern "C" int tms_kv_append_rotary(const tms_cache* cache, const tms_append_rotary_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_cache(cache, true, true);
    if (rc != TMS_OK) return rc;
    if (!args || bad_stride(args->k_new_stride, 2) || bad_stride(args->v_new_stride, 2)) return TMS_ERR_INVALID_ARG;
    if (args->q_heads < 0 || (args->q_heads > 0 && (bad_stride(args->q_stride, 2) || bad_stride(args->out_stride, 2))))
        return TMS_ERR_INVALID_ARG;
    if (bad_rotary(args->rotary_dim, cache->head_dim, args->interleaved, args->scale)) return TMS_ERR_INVALID_ARG;
    if (cache->batch > TMS_APPEND_MAX_BATCH || (int64_t)args->q_heads + cache->kv_heads > TMS_ROTARY_MAX_HEADS) return TMS_ERR_CAPACITY;
    if (cache->batch == 0 || cache->tokens == 0 || cache->max_q == 0) return TMS_OK;
    if (!args->k_new || !args->v_new || !aligned16(args->k_new) || !aligned16(args->v_new)) return TMS_ERR_INVALID_ARG;
    if (args->q_heads > 0 && (!args->q || !args->out || !aligned16(args->q) || !aligned16(args->out))) return TMS_ERR_INVALID_ARG;
    if (!args->freqs || ((uintptr_t)args->freqs & 3) || ((uintptr_t)args->positions & 3)) return TMS_ERR_INVALID_ARG;
    if (args->q_heads > 0 && bad_output(args->q, args->q_stride, args->out, args->out_stride)) return TMS_ERR_INVALID_ARG;
    if (cache->k == cache->v) return TMS_ERR_INVALID_ARG;
    TurnParams a{};
    a.c = view_of(cache);
    a.x = (const char*)args->q;
    a.out = (char*)args->out;
    a.k = (const char*)args->k_new;
    a.v = (const char*)args->v_new;
    a.xt = 2 * args->q_stride[0];
    a.xh = 2 * args->q_stride[1];
    a.ot = 2 * args->out_stride[0];
    a.oh = 2 * args->out_stride[1];
    a.kt = 2 * args->k_new_stride[0];
    a.kh = 2 * args->k_new_stride[1];
    a.vt = 2 * args->v_new_stride[0];
    a.vh = 2 * args->v_new_stride[1];
    a.positions = args->positions;
    a.freqs = args->freqs;
    a.scale = args->scale;
    a.tokens = cache->tokens;
    a.q_heads = args->q_heads;
    a.heads = args->q_heads + cache->kv_heads;
    a.head_dim = cache->head_dim;
    a.rotary_dim = args->rotary_dim;
    return launch_turns<true>(a, cache->dtype, args->interleaved != 0, std::min(cache->max_q, cache->tokens), cache->batch, stream);
}
