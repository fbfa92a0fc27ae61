// tms_verify_tree.hip -- drafted trees verified against the target's probabilities, with
// given random numbers (tms_verify_tree).
//
// At node c, R = p_c and S = 1; child j (token x) is accepted where u_j q_c(x) S < R(x),
// and refused it leaves R = max(R - S q_c, 0), S = sum R.  R / S is the residual
// distribution max(R / S - q, 0) over its sum without a division; R - S q is exact or rounded
// once in fp64, so products with S below 1 shrink but lose nothing.  With given drafts q is a single id, and
// what is left of S after refusing x is S - R(x): the walk needs two numbers a node and no row.
//
// Bound by latency: the walk is a chain, and what it reads depends on it.  A refusal
// of a drawn draft and the last draw are passes over the vocabulary, so a sequence is divided
// among `parts` workgroups, each with its stretch of ids.  All of them make the walk, with
// the same numbers in the same order; a pass's sums by part go through a word each in
// global memory, written once, its top bit saying that it is there.  No answer depends on a
// wait: one that runs out works the missing part's sum out itself, to the same bits.
#include <algorithm>
#include <atomic>

#include "tms_cache.h"
#include "tms_device.h"
#include "../../include/tmtree_hip.h"

namespace tms {

constexpr int kVerThreads = 512, kVerWaves = kVerThreads / 64;
constexpr int kVerNodes = TMS_TREE_MAX_NODES, kVerSets = kVerNodes / 64;
constexpr int kVerSteps = 8;             // loads of 16 bytes a thread has of its part's row, at most
constexpr int kVerPolls = 256;           // some 0.2 ms, where a call takes 10 to 60 us
constexpr uint64_t kThere = 1ull << 63;

struct VerifyParams {
    const void* target;
    const void* draft;
    int64_t tstride, dstride;   // elements
    int vocab, tokens, max_q;
    const int32_t* ids;
    const int32_t* parents;
    const int32_t* q_start;
    const double* uniforms;
    int32_t* path;
    int32_t* kept;
    int32_t* token;
    uint64_t* slots;            // [batch][max_q + 1 passes][parts]
    int parts, steps;
    int polls;                  // of a wait for another part's sum
};

struct TreeView {
    int q0, n;
};
__device__ __forceinline__ TreeView tree_view(const VerifyParams& a, int b) {
    TreeView s;
    s.q0 = min(max(a.q_start[b], 0), a.tokens);
    s.n = min(min(max(a.q_start[b + 1], s.q0), a.tokens) - s.q0, a.max_q);
    return s;
}

__global__ __launch_bounds__(256) void verify_clear_kernel(VerifyParams a) {
    const int b = blockIdx.x;
    const int64_t all = (int64_t)(tree_view(a, b).n + 1) * a.parts;
    uint64_t* s = a.slots + (int64_t)b * (a.max_q + 1) * a.parts;
    for (int64_t i = threadIdx.x; i < all; i += 256) st_agent(s + i, (uint64_t)0);
}

// Entries that are no probability count as 0.
__device__ __forceinline__ double clean(float p) { return p > 0.f && p <= 3.402823466e38f ? (double)p : 0.0; }

__device__ __forceinline__ double wave_sum(double x) {   // the same in every lane
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

__device__ __forceinline__ double wave_upto(double x, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}

template <typename T, bool DRAWN>
struct Verify {
    static constexpr int VEC = Elt<T>::kVec, STEP = kVerThreads * VEC, NB = 16 / VEC;   // NB steps' values in registers
    struct Shared {
        double u[kVerNodes], left[kVerNodes], q[kVerNodes];   // R(x) and q(x) of a node under its parent
        double hist[kVerNodes];                               // S before each refusal at the current node
        double cell[kVerSteps * kVerWaves];                   // sums of a wave's 64 VEC ids
        double part[64];
        int32_t id[kVerNodes];
        int16_t up[kVerNodes], path[kVerNodes];
        uint32_t gone[DRAWN ? 1 : kVerSteps * STEP / 32];     // given drafts refused, of a part's ids
        uint64_t missing;
    };
    const VerifyParams& a;
    Shared& sm;
    const int b, own, t, lane, wave;
    const TreeView tree;
    int up[kVerSets], id[kVerSets];   // the lane's nodes, 64 k + lane: parent and token
    int cells_of = -1;                // the part that sm.cell is of
    int pass = 0;

    __device__ Verify(const VerifyParams& a_, Shared& sm_, int b_, int part)
        : a(a_), sm(sm_), b(b_), own(part), t(threadIdx.x), lane(threadIdx.x & 63),
          wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), tree(tree_view(a_, b_)) {}

    __device__ const T* target_row(int c) const { return (const T*)a.target + (int64_t)(tree.q0 + c) * a.tstride; }
    __device__ const T* draft_row(int c) const { return (const T*)a.draft + (int64_t)(tree.q0 + c) * a.dstride; }

    // The tree, and each node's two numbers.
    __device__ void load() {
        for (int i = t; i < tree.n; i += kVerThreads) {
            const int p = a.parents[tree.q0 + i], x = a.ids[tree.q0 + i];
            const bool in = p >= 0 && p < i && (unsigned)x < (unsigned)a.vocab;
            sm.u[i] = a.uniforms[tree.q0 + i];
            sm.id[i] = x;
            sm.up[i] = (int16_t)(p >= 0 && p < i ? p : -1);
            sm.left[i] = in ? clean(Elt<T>::scalar(target_row(p) + x)) : 0.0;
            sm.q[i] = !DRAWN ? 1.0 : in ? clean(Elt<T>::scalar(draft_row(p) + x)) : 0.0;
        }
#pragma unroll
        for (int k = 0; k < kVerSets; ++k) {
            const int i = 64 * k + lane;
            up[k] = -1;
            id[k] = 0;
            if (i < tree.n) {
                const int p = a.parents[tree.q0 + i];
                up[k] = p >= 0 && p < i ? p : -1;
                id[k] = a.ids[tree.q0 + i];
            }
        }
        lds_sync();
    }

    // The first child of c past node j, -1 without one.
    __device__ int child(int c, int j) const {
#pragma unroll
        for (int k = 0; k < kVerSets; ++k)
            if (64 * k < tree.n && 64 * k + 63 > j) {
                const uint64_t m = __ballot(up[k] == c && 64 * k + lane > j);
                if (m) return 64 * k + __builtin_ctzll(m);
            }
        return -1;
    }
    // Given drafts: an earlier child of c has the token of j.
    __device__ bool twice(int c, int j) const {
        const int x = sm.id[j];
        bool same = false;
#pragma unroll
        for (int k = 0; k < kVerSets; ++k)
            if (64 * k < j) same |= up[k] == c && 64 * k + lane < j && id[k] == x;
        return __any(same);
    }

    __device__ uint4 fetch(const T* row, int at) const {   // VEC entries from id `at` on, zeros past the vocabulary
        if (at + VEC <= a.vocab) return ld_any(row + at);
        uint32_t w[4] = {0, 0, 0, 0};
        for (int e = 0; e < VEC && at + e < a.vocab; ++e) {
            if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(Elt<T>::scalar(row + at + e));
            else w[e / 2] |= (uint32_t)*(const uint16_t*)(row + at + e) << 16 * (e & 1);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }

    // R of NB steps from `step` on of a part, after `m` refusals at c; `whole`: the row as it is.
    __device__ void residual(int part, int step, int n, int c, int m, bool whole, double (&r)[NB][VEC]) const {
        const int at = part * a.steps * STEP + step * STEP + t * VEC;
        uint4 pq[NB], dq[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k)
            if (k < n) {
                pq[k] = fetch(target_row(c), at + k * STEP);
                if (DRAWN && m > 0) dq[k] = fetch(draft_row(c), at + k * STEP);
            }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[k][e] = k < n ? clean(elt<T>(pq[k], e)) : 0.0;
            if (!DRAWN && !whole && k < n) {
                const int from = (step + k) * STEP + t * VEC;
                const uint32_t bits = sm.gone[from / 32] >> (from & 31);
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (bits >> e & 1) r[k][e] = 0.0;
            }
        }
        if constexpr (DRAWN) {
            for (int i = 0; i < m; ++i) {
                const double s = sm.hist[i];
#pragma unroll
                for (int k = 0; k < NB; ++k)
                    if (k < n)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) r[k][e] = fmax(r[k][e] - s * clean(elt<T>(dq[k], e)), 0.0);
            }
        }
    }

    __device__ double lane_sum(const double (&r)[VEC]) const {
        double s = r[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) s += r[e];
        return s;
    }

    // The sum of R over a part's ids, by cells of sm.cell.
    __device__ double sum_part(int part, int c, int m, bool whole) {
        lds_sync();   // sm.cell and sm.gone are free, sm.hist is there
        if (!DRAWN && !whole) {
            const int words = a.steps * STEP / 32, first = part * a.steps * STEP;
            for (int i = t; i < words; i += kVerThreads) sm.gone[i] = 0;
            lds_sync();
            for (int i = t; i < tree.n; i += kVerThreads) {
                const int64_t x = (int64_t)sm.id[i] - first;
                if (sm.up[i] == c && x >= 0 && x < a.steps * STEP) atomicOr(&sm.gone[x / 32], 1u << (x & 31));
            }
            lds_sync();
        }
        for (int step = 0; step < a.steps; step += NB) {
            const int n = min(NB, a.steps - step);
            double r[NB][VEC];
            residual(part, step, n, c, m, whole, r);
#pragma unroll
            for (int k = 0; k < NB; ++k)
                if (k < n) {
                    const double s = wave_sum(lane_sum(r[k]));
                    if (lane == 0) sm.cell[(step + k) * kVerWaves + wave] = s;
                }
        }
        lds_sync();
        cells_of = part;
        double s = 0.0;
        for (int i = 0; i < a.steps * kVerWaves; ++i) s += sm.cell[i];
        return s;
    }

    // The sum over the whole vocabulary; sm.part has the parts'.
    __device__ double sum_all(int c, int m, bool whole) {
        const double mine = sum_part(own, c, m, whole);
        if (a.parts == 1) return mine;
        uint64_t* const slot = a.slots + ((int64_t)b * (a.max_q + 1) + pass) * a.parts;
        ++pass;
        if (t == 0) st_agent(slot + own, __builtin_bit_cast(uint64_t, mine) | kThere);
        if (wave == 0) {
            uint64_t v = lane < a.parts ? 0 : kThere, none = 0;
            if (lane == own) v = __builtin_bit_cast(uint64_t, mine) | kThere;
            none = __ballot(v == 0);
            for (int it = 0; none && it < a.polls; ++it) {
                if (v == 0) v = ld_agent(slot + lane);
                none = __ballot(v == 0);
                if (none) __builtin_amdgcn_s_sleep(1);
            }
            sm.part[lane] = __builtin_bit_cast(double, v & ~kThere);
            if (lane == 0) sm.missing = none;
        }
        lds_sync();
        for (uint64_t none = sm.missing; none; none &= none - 1) {
            const int p = __builtin_ctzll(none);
            const double s = sum_part(p, c, m, whole);
            if (t == 0) sm.part[p] = s;
        }
        lds_sync();
        return __shfl(wave_upto(sm.part[lane], lane), 63);
    }

    // The first id with more than `rest` up to it, of this workgroup's part.
    __device__ void pick(int c, int m, bool whole, double rest) {
        if (cells_of != own) sum_part(own, c, m, whole);
        double run = 0.0, before = 0.0;
        int cell = -1;
        for (int i = 0; i < a.steps * kVerWaves; ++i) {
            const double s = sm.cell[i];
            if (s > 0.0) {
                cell = i;
                before = run;
                if (run + s > rest) break;
            }
            run += s;
        }
        if (cell < 0 || cell % kVerWaves != wave) return;
        const int step = cell / kVerWaves;
        double r[NB][VEC];
        residual(own, step, 1, c, m, whole, r);
        const double s = lane_sum(r[0]), upto = wave_upto(s, lane);
        const uint64_t over = __ballot(s > 0.0 && before + upto > rest), some = __ballot(s > 0.0);
        const int who = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        const double below = __shfl_up(upto, 1);
        if (lane != who) return;
        double at = before + (lane ? below : 0.0);
        int found = -1;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (r[0][e] > 0.0 && (found < 0 || !(at > rest))) found = e;
            at += r[0][e];
        }
        a.token[b] = own * a.steps * STEP + step * STEP + t * VEC + found;
    }

    __device__ void run() {
        load();
        int c = 0, m = 0, len = 1, j = 0;
        double S = 1.0;
        while ((j = child(c, j)) >= 0) {
            const double r = !DRAWN && twice(c, j) ? 0.0 : sm.left[j];
            if (sm.u[j] * sm.q[j] * S < r) {
                if (t == 0) sm.path[len] = (int16_t)j;
                ++len;
                c = j;
                S = 1.0;
                m = 0;
            } else if (DRAWN) {
                lds_sync();   // sm.left and sm.hist have been read
                for (int i = t; i < tree.n; i += kVerThreads)
                    if (sm.up[i] == c) sm.left[i] = fmax(sm.left[i] - S * sm.q[i], 0.0);
                if (t == 0) sm.hist[m] = S;
                ++m;
                S = sum_all(c, m, false);
            } else {
                S -= r;
            }
        }
        bool whole = false;
        double total = DRAWN && m > 0 ? S : sum_all(c, m, false);
        if (!(total > 0.0)) {   // nothing is left
            whole = true;
            m = 0;
            total = sum_all(c, m, true);
        }
        if (own == 0) {
            if (t == 0) sm.path[0] = 0;
            lds_sync();
            for (int i = t; i < a.max_q; i += kVerThreads) a.path[(int64_t)b * a.max_q + i] = i < len ? sm.path[i] : -1;
            if (t == 0) {
                a.kept[b] = len;
                if (!(total > 0.0)) a.token[b] = -1;
            }
        }
        if (!(total > 0.0)) return;
        const double aim = fmax(sm.u[0] * total, 0.0);   // (a NaN gives 0)
        double before = 0.0;
        if (a.parts > 1) {
            const double s = sm.part[lane], upto = wave_upto(s, lane);
            const uint64_t over = __ballot(s > 0.0 && upto > aim), some = __ballot(s > 0.0);
            const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            if (who != own) return;
            before = own ? __shfl(upto, own - 1) : 0.0;
        }
        pick(c, m, whole, aim - before);
    }
};

template <typename T, bool DRAWN>
__global__ __launch_bounds__(kVerThreads) void verify_tree_kernel(VerifyParams a) {
    __shared__ typename Verify<T, DRAWN>::Shared sm;
    const int b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
    if (tree_view(a, b).n == 0) {
        if (part == 0) {
            for (int i = threadIdx.x; i < a.max_q; i += kVerThreads) a.path[(int64_t)b * a.max_q + i] = -1;
            if (threadIdx.x == 0) {
                a.kept[b] = 0;
                a.token[b] = -1;
            }
        }
        return;
    }
    Verify<T, DRAWN> v(a, sm, b, part);
    v.run();
}

struct VerifyPlan {
    int parts, steps;
    size_t bytes;
};

// As many parts as bring the card some workgroups a CU, up to 64, with one step each at least.
static VerifyPlan plan_verify(const tms_verify_tree_args* a) {
    VerifyPlan p;
    const int step = kVerThreads * (a->dtype == TMS_DTYPE_F32 ? 4 : 8);
    const int steps = (a->vocab + step - 1) / step;   // of the vocabulary
    const int want = std::max(1, std::min(64, 1024 / std::max(a->batch, 1)));
    p.steps = std::min(std::max(1, (steps + want - 1) / want), kVerSteps);
    p.parts = (steps + p.steps - 1) / p.steps;
    p.bytes = p.parts > 1 ? (size_t)a->batch * (a->max_q + 1) * p.parts * 8 : 0;
    return p;
}
static_assert(TMS_VERIFY_MAX_VOCAB <= 64 * kVerSteps * kVerThreads * 4, "64 parts hold a vocabulary");

static std::atomic<int> g_polls{kVerPolls};

static int check_verify(const tms_verify_tree_args* a) {
    if (!a || a->reserved != 0) return TMS_ERR_INVALID_ARG;
    if (a->dtype != TMS_DTYPE_F32 && a->dtype != TMS_DTYPE_F16 && a->dtype != TMS_DTYPE_BF16) return TMS_ERR_INVALID_ARG;
    if (a->vocab < 1 || a->batch < 0 || a->tokens < 0 || a->max_q < 0) return TMS_ERR_INVALID_ARG;
    if (a->target_stride < a->vocab || (a->draft && a->draft_stride < a->vocab)) return TMS_ERR_INVALID_ARG;
    if (a->vocab > TMS_VERIFY_MAX_VOCAB || a->batch > TMS_VERIFY_MAX_BATCH || a->max_q > TMS_TREE_MAX_NODES ||
        a->tokens > TMS_CACHE_MAX_TOKENS)
        return TMS_ERR_CAPACITY;
    if (a->batch == 0) return TMS_OK;
    const uintptr_t low = a->dtype == TMS_DTYPE_F32 ? 3 : 1;
    if (!a->q_start || !a->kept || !a->token || (a->max_q > 0 && !a->path)) return TMS_ERR_INVALID_ARG;
    if (a->tokens > 0 && (!a->target || !a->draft_tokens || !a->parents || !a->uniforms || ((uintptr_t)a->target & low) ||
                          ((uintptr_t)a->draft & low) || ((uintptr_t)a->uniforms & 7)))
        return TMS_ERR_INVALID_ARG;
    return TMS_OK;
}

template <typename T>
static void launch_verify(const VerifyParams& a, int batch, hipStream_t stream) {
    const dim3 grid((unsigned)(batch * a.parts));
    if (a.draft) hipLaunchKernelGGL((verify_tree_kernel<T, true>), grid, dim3(kVerThreads), 0, stream, a);
    else hipLaunchKernelGGL((verify_tree_kernel<T, false>), grid, dim3(kVerThreads), 0, stream, a);
}

}  // namespace tms

extern "C" int64_t tms_verify_tree_workspace(const tms_verify_tree_args* args) {
    const int rc = tms::check_verify(args);
    return rc != TMS_OK ? rc : (int64_t)tms::plan_verify(args).bytes;
}

extern "C" int tms_verify_tree(const tms_verify_tree_args* args, hipStream_t stream) {
    using namespace tms;
    const int rc = check_verify(args);
    if (rc != TMS_OK) return rc;
    if (args->batch == 0) return TMS_OK;
    const VerifyPlan p = plan_verify(args);
    if (args->workspace_bytes < p.bytes || (p.bytes > 0 && (!args->workspace || !aligned16(args->workspace)))) return TMS_ERR_INVALID_ARG;
    VerifyParams a{};
    a.target = args->target;
    a.draft = args->draft;
    a.tstride = args->target_stride;
    a.dstride = args->draft_stride;
    a.vocab = args->vocab;
    a.tokens = args->tokens;
    a.max_q = args->max_q;
    a.ids = args->draft_tokens;
    a.parents = args->parents;
    a.q_start = args->q_start;
    a.uniforms = args->uniforms;
    a.path = args->path;
    a.kept = args->kept;
    a.token = args->token;
    a.slots = (uint64_t*)args->workspace;
    a.parts = p.parts;
    a.steps = p.steps;
    a.polls = g_polls.load(std::memory_order_relaxed);
    if (a.parts > 1) hipLaunchKernelGGL(verify_clear_kernel, dim3(args->batch), dim3(256), 0, stream, a);
    switch (args->dtype) {
        case TMS_DTYPE_F32: launch_verify<float>(a, args->batch, stream); break;
        case TMS_DTYPE_F16: launch_verify<_Float16>(a, args->batch, stream); break;
        default: launch_verify<Bf16>(a, args->batch, stream);
    }
    return hipGetLastError() == hipSuccess ? TMS_OK : TMS_ERR_HIP;
}

extern "C" int tms_debug_verify_polls(int polls) {
    tms::g_polls.store(polls < 0 ? tms::kVerPolls : polls, std::memory_order_relaxed);
    return TMS_OK;
}
