// tms_verify_tree.hip -- drafted trees verified against the target's probabilities, with
// given random numbers (tms_verify_tree).
//
// At node c, R = p_c and S = 1; child j (token x) is accepted where u_j q_c(x) S < R(x),
// and refused it leaves R = max(R - S q_c, 0), S = sum R.  R / S is the residual
// distribution max(R / S - q, 0) over its sum without a division.  R - S q in fp64 is rounded once at a
// node's first refusal, where S is 1, and past it twice, the product and the difference: by 2^-53 of each.
// With given drafts q is a single id, and what is left of S after refusing x is S - R(x): the walk
// needs two numbers a node and no row.
//
// Bound by latency: the walk is a chain, and what it reads depends on it.  A refusal
// of a drawn draft and the last draw are passes over the vocabulary, so a sequence is divided
// among `parts` workgroups, each with its stretch of ids.  All of them make the walk, with
// the same numbers in the same order; a pass's sums by part go through a word each in
// global memory, written once, its top bit saying that it is there.  No answer depends on a
// wait: one that runs out works the missing part's sum out itself, to the same bits.
//
// R stays in registers from refusal to refusal, so a row is read once a node.  32 sequences of 9
// to 25 drawn nodes over 128256 ids, fp32: 28 to 36 us, some 2.9 a pass (1.4 of them the exchange
// between XCDs, 1.0 the sum; 90 us with R worked out from the rows at each refusal).  64 of 16 given nodes over 151936
// ids, bf16: 15 us (3.4 the tree, 4.3 the row, 2.2 the exchange).
#include <algorithm>
#include <atomic>

#include "tms_cache.h"
#include "tms_device.h"
#include "../../include/tmtree_hip.h"

namespace tms {

constexpr int kVerThreads = 512, kVerWaves = kVerThreads / 64;
constexpr int kVerNodes = TMS_TREE_MAX_NODES;
constexpr int kVerParts = 128;           // of a sequence, two a lane
constexpr int kVerPolls = 256;           // some 0.2 ms, where a call takes 10 to 60 us
constexpr uint64_t kThere = 1ull << 63;
static_assert(kVerNodes == kVerThreads, "a thread has a node");

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A part's ids: those whose R a thread keeps in registers, 16 (32 where it keeps them in 16 bits).
// A vocabulary of given drafts in 16 bits that fits 64 is one part: nothing to clear or to exchange
// (5 sequences of 8 nodes over 32000 ids 9.1 us, 10.7 in two parts; 64 of them 9.9 and 11.0.  In fp32, whose rows are
// twice as long, it takes longer from a few sequences on: 5 11.3 and 9.8, 64 13.1 and 10.4).
constexpr int kVerMost = kVerThreads * 64;
constexpr int verify_ids(bool wide, bool drawn) { return kVerThreads * (wide || drawn ? 16 : 32); }

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
    uint64_t* slots;            // [batch][passes][parts]
    int64_t words;              // of them
    int passes, parts;
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

// One workgroup for few words to clear (1.4 us; workgroups on all XCDs take 4), four for more (32 sequences of
// 9 to 25 drawn nodes, 13312 words: 36.0 us a call, 37.1 with one).
__global__ __launch_bounds__(256) void verify_clear_kernel(VerifyParams a) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < a.words; i += (int64_t)gridDim.x * blockDim.x)
        st_agent(a.slots + i, (uint64_t)0);
}

// Entries that are no probability count as 0.
__device__ __forceinline__ double clean(float p) { return p > 0.f && p <= 3.402823466e38f ? (double)p : 0.0; }

// x of the lane that `CTRL` names, 0 where that is none or the row is not in ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ double lane_move(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 15, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 15, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sums up to each lane: within rows of 16 by shifts of 1, 2, 4 and 8, then the last lane of a row
// to the next one, and of the first two rows to the others.
__device__ __forceinline__ double wave_upto(double x) {
    x += lane_move<0x111, 15>(x);
    x += lane_move<0x112, 15>(x);
    x += lane_move<0x114, 15>(x);
    x += lane_move<0x118, 15>(x);
    x += lane_move<0x142, 10>(x);
    x += lane_move<0x143, 12>(x);
    return x;
}

template <typename T, bool DRAWN, bool ONE>
struct Verify {
    // Of a part's ids a wave has CELL one after another, in steps of STEP, VEC of them a lane.
    static constexpr int VEC = Elt<T>::kVec, STEP = 64 * VEC;
    static constexpr int PART = ONE ? kVerMost : verify_ids(sizeof(T) == 4, DRAWN), CELL = PART / kVerWaves, STEPS = CELL / STEP;
    struct Shared {
        double u[kVerNodes], left[kVerNodes], q[DRAWN ? kVerNodes : 1];   // R(x) and q(x) of a node under its parent
        double hist[DRAWN ? kVerNodes : 1];                               // S before each refusal at the current node
        double cell[kVerWaves], other[kVerWaves];                         // sums of the waves' ids
        double part[kVerParts];
        int32_t id[DRAWN ? 1 : kVerNodes];
        int16_t up[kVerNodes], path[kVerNodes];   // (given drafts: the parent of a node that it accepts, else -1)
        int16_t kin[DRAWN ? 1 : kVerNodes];       // given drafts: the parent
        uint64_t missing[2];
    };
    const VerifyParams& a;
    Shared& sm;
    const int b, own, t, lane, wave;
    const TreeView tree;
    int up_t;                         // the thread's node, t: parent, R(x) and q(x)
    double left_t, q_t;
    u32x4 row[STEPS];                 // the part's ids: p, with drawn drafts q
    double rest[DRAWN ? STEPS : 1][VEC];   // and R
    int pass = 0;

    __device__ Verify(const VerifyParams& a_, Shared& sm_, int b_, int part)
        : a(a_), sm(sm_), b(b_), own(part), t(threadIdx.x), lane(threadIdx.x & 63),
          wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), tree(tree_view(a_, b_)) {}

    __device__ const T* target_row(int c) const { return (const T*)a.target + (int64_t)(tree.q0 + c) * a.tstride; }
    __device__ const T* draft_row(int c) const { return (const T*)a.draft + (int64_t)(tree.q0 + c) * a.dstride; }

    // The tree, and each node's two numbers.
    __device__ void load() {
        int p = -1, x = -1;
        double u = 0.0;
        if (t < tree.n) {
            p = a.parents[tree.q0 + t];
            x = a.ids[tree.q0 + t];
            u = a.uniforms[tree.q0 + t];
        }
        up_t = p < t ? p : -1;
        const bool in = up_t >= 0 && (unsigned)x < (unsigned)a.vocab;
        left_t = q_t = 0.0;
        if (in) {
            const float y = Elt<T>::scalar(target_row(up_t) + x), z = DRAWN ? Elt<T>::scalar(draft_row(up_t) + x) : 0.f;
            left_t = clean(y);
            q_t = clean(z);
        }
        up_t = max(up_t, -1);
        sm.u[t] = u;
        sm.left[t] = left_t;
        if constexpr (DRAWN) {
            sm.up[t] = (int16_t)up_t;
            sm.q[t] = q_t;
        } else {
            // Whether a node would be accepted depends on its elder siblings alone: S is 1 without
            // what they have, a token that several of them have counting once.
            sm.kin[t] = (int16_t)up_t;
            sm.id[t] = x;
            lds_sync();
            bool twice = false;
            for (int i = up_t + 1; i < t && t < tree.n; ++i) twice |= sm.kin[i] == up_t && sm.id[i] == x;
            lds_sync();
            if (twice) sm.left[t] = left_t = 0.0;
            lds_sync();
            double S = 1.0;
            for (int i = up_t + 1; i < t && t < tree.n; ++i) S -= sm.kin[i] == up_t ? sm.left[i] : 0.0;
            sm.up[t] = (int16_t)(u * S < left_t ? up_t : -1);
        }
        lds_sync();
    }

    // The first child of c past node j (given drafts: that is accepted), -1 without one.
    __device__ int child(int c, int j) const {
        for (int k = (j + 1) & ~63; k < tree.n; k += 64) {
            const uint64_t m = __ballot(sm.up[k + lane] == c && k + lane > j);
            if (m) return k + __builtin_ctzll(m);
        }
        return -1;
    }
    // A row's entries of a part's steps from `step` on: zeros past the vocabulary.
    template <int N>
    __device__ void fetch(const T* r, int part, int step, u32x4 (&w)[N]) const {
        const int first = part * PART + wave * CELL + step * STEP, end = a.vocab - a.vocab % VEC;   // past it is one piece that is not whole
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int at = first + k * STEP + lane * VEC;
            w[k] = (u32x4){0, 0, 0, 0};
            if (at < end) {
                const uint4 x = ld_any(r + at);
                w[k] = (u32x4){x.x, x.y, x.z, x.w};
            }
        }
        const int cut = end - first;
        if (end < a.vocab && cut >= 0 && cut < N * STEP && cut % STEP / VEC == lane) {
            u32x4 x = (u32x4){0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < VEC - 1; ++e)
                if (end + e < a.vocab) {
                    if constexpr (sizeof(T) == 4) x[e] = *(const uint32_t*)(r + end + e);
                    else x[e / 2] |= (uint32_t)*(const uint16_t*)(r + end + e) << 16 * (e & 1);
                }
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (cut / STEP == k) w[k] = x;
        }
    }
    // Entries that are no probability as 0: those whose bits are not below infinity's.
    static __device__ u32x4 cleaned(u32x4 w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = w[i] < 0x7F800000u ? w[i] : 0;
            } else {
                constexpr uint32_t inf = __is_same(T, Bf16) ? 0x7F80u : 0x7C00u;
                w[i] = (w[i] & 0xFFFFu) < inf ? w[i] : w[i] & 0xFFFF0000u;
                w[i] = w[i] < inf << 16 ? w[i] : w[i] & 0xFFFFu;
            }
        }
        return w;
    }
    static __device__ double entry(u32x4 w, int e) { return (double)elt<T>(make_uint4(w[0], w[1], w[2], w[3]), e); }

    // Given drafts: the tokens of c's children, all refused, out of the entries of `fetch`.
    template <int N>
    __device__ void without(u32x4 (&w)[N], int c, int part, int step) const {
        const int first = part * PART + wave * CELL + step * STEP;
        for (int k = c & ~63; k < tree.n; k += 64) {
            const int id = sm.id[k + lane];
            for (uint64_t m = __ballot(sm.kin[k + lane] == c && id >= first && id - first < N * STEP); m; m &= m - 1) {
                const int x = __builtin_amdgcn_readlane(id, __builtin_ctzll(m)) - first;
                if (x % STEP / VEC != lane) continue;
                const int word = x % VEC * (int)sizeof(T) / 4;
                const uint32_t keep = sizeof(T) == 4 ? 0u : x & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (x / STEP == n && word == i) w[n][i] &= keep;
            }
        }
    }

    // R of the part's ids at node c: the target row, with given drafts (not `whole`) without c's children.
    __device__ void begin(int c, bool whole) {
        u32x4 p[STEPS];
        fetch(target_row(c), own, 0, p);
        if constexpr (DRAWN) {
            if (!whole) fetch(draft_row(c), own, 0, row);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                p[k] = cleaned(p[k]);
                row[k] = cleaned(row[k]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) rest[k][e] = entry(p[k], e);
            }
        } else {
            if (!whole) without(p, c, own, 0);
#pragma unroll
            for (int k = 0; k < STEPS; ++k) row[k] = cleaned(p[k]);
        }
    }
    // R of a step's ids, and their sum.  (The entries are widened each time: kept in fp64
    // they would not fit the registers.)
    __device__ void values(int k, double (&r)[VEC]) const {
        if constexpr (DRAWN) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[e] = rest[k][e];
        } else {
            u32x4 w = row[k];
            asm volatile("" : "+v"(w));
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[e] = entry(w, e);
        }
    }
    static __device__ double sum_of(const double (&r)[VEC]) {
        double s = r[0];
#pragma unroll
        for (int e = 1; e < VEC; ++e) s += r[e];
        return s;
    }
    __device__ void refuse(double S) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            u32x4 w = row[k];
            asm volatile("" : "+v"(w));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < VEC; ++e) rest[DRAWN ? k : 0][e] = fmax(rest[DRAWN ? k : 0][e] - S * entry(w, e), 0.0);
        }
    }

    static __device__ double cells_sum(const double (&cell)[kVerWaves]) {
        double s = cell[0];
#pragma unroll
        for (int w = 1; w < kVerWaves; ++w) s += cell[w];
        return s;
    }

    // The sum of the part's R, by cells.  (A barrier has passed since sm.cell was read.)
    __device__ double sum_own() {
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            double r[VEC];
            values(k, r);
            s += sum_of(r);
        }
        s = wave_upto(s);
        if (lane == 63) sm.cell[wave] = s;
        lds_sync();
        return cells_sum(sm.cell);
    }

    // The same of another part, after `m` refusals at c: the same operations in the same order.
    __device__ double sum_other(int part, int c, int m, bool whole) {
        lds_sync();
        double s = 0.0;
#pragma unroll 1
        for (int k = 0; k < STEPS; ++k) {
            u32x4 p[1], q[1] = {(u32x4){0, 0, 0, 0}};
            fetch(target_row(c), part, k, p);
            if (DRAWN && m > 0) fetch(draft_row(c), part, k, q);
            if (!DRAWN && !whole) without(p, c, part, k);
            p[0] = cleaned(p[0]);
            q[0] = cleaned(q[0]);
            double r[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                r[e] = entry(p[0], e);
                if constexpr (DRAWN) {
                    const double y = entry(q[0], e);
                    for (int i = 0; i < m; ++i) r[e] = fmax(r[e] - sm.hist[i] * y, 0.0);
                }
            }
            s += sum_of(r);
        }
        s = wave_upto(s);
        if (lane == 63) sm.other[wave] = s;
        lds_sync();
        return cells_sum(sm.other);
    }

    // The sum over the whole vocabulary; sm.part has the parts'.
    __device__ double sum_all(int c, int m, bool whole) {
        const double mine = sum_own();
        if (ONE || a.parts == 1) return mine;
        uint64_t* const slot = a.slots + ((int64_t)b * a.passes + pass) * a.parts;
        ++pass;
        if (t == 0) st_agent(slot + own, __builtin_bit_cast(uint64_t, mine) | kThere);
        if (wave == 0) {
            uint64_t v[2], none[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[i] = 2 * lane + i == own ? __builtin_bit_cast(uint64_t, mine) | kThere : 2 * lane + i < a.parts ? 0 : kThere;
                none[i] = __ballot(v[i] == 0);
            }
            for (int it = 0; (none[0] | none[1]) && it < a.polls; ++it) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (v[i] == 0) v[i] = ld_agent(slot + 2 * lane + i);
#pragma unroll
                for (int i = 0; i < 2; ++i) none[i] = __ballot(v[i] == 0);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sm.part[2 * lane + i] = __builtin_bit_cast(double, v[i] & ~kThere);
                if (lane == 0) sm.missing[i] = none[i];
            }
        }
        lds_sync();
        bool any = false;
        for (int i = 0; i < 2; ++i)
            for (uint64_t none = sm.missing[i]; none; none &= none - 1) {
                const int p = 2 * __builtin_ctzll(none) + i;
                const double s = sum_other(p, c, m, whole);
                if (t == 0) sm.part[p] = s;
                any = true;
            }
        if (any) lds_sync();
        return readlane_f64(wave_upto(sm.part[2 * lane] + sm.part[2 * lane + 1]), 63);
    }

    // The first id with more than `aim` up to it, of this workgroup's part, which has some.
    __device__ void pick(double aim) {
        double at = 0.0, run = 0.0;
        int cell = -1;
#pragma unroll
        for (int w = 0; w < kVerWaves; ++w) {
            if (sm.cell[w] > 0.0 && (cell < 0 || !(run > aim))) {
                cell = w;
                at = run;
            }
            run += sm.cell[w];
        }
        if (cell != wave) return;
        int found = -1;
        for (int k = 0; k < STEPS; ++k) {
            double r[VEC];
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
                if (i == k) values(i, r);
            const double mine = sum_of(r), here = wave_upto(mine);
            const uint64_t some = __ballot(mine > 0.0), over = __ballot(mine > 0.0 && at + here > aim);
            if (found >= 0 && at > aim) break;   // (a sum's last bit)
            if (some) {   // the last step with some where none goes past
                const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
                double x = who ? at + readlane_f64(here, who - 1) : at;
                int e0 = -1;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (r[e] > 0.0 && (e0 < 0 || !(x > aim))) e0 = e;
                    x += r[e];
                }
                found = own * PART + wave * CELL + k * STEP + who * VEC + __builtin_amdgcn_readlane(e0, who);
                if (over) break;
            }
            at += readlane_f64(here, 63);
        }
        if (lane == 0) a.token[b] = found;
    }

    __device__ void run() {
        load();
        int c = 0, m = 0, len = 1, j = 0;   // the node, refusals at it, nodes of the path, the child last tried
        double S = 1.0, total = 0.0;
        bool whole = false;
        for (;;) {
            bool refused = false;   // a drawn draft: a pass over the vocabulary
            while (j >= 0 && (j = child(c, j)) >= 0) {
                if (DRAWN && !(sm.u[j] * sm.q[j] * S < sm.left[j])) {
                    refused = true;
                    break;
                }
                if (t == 0) sm.path[len] = (int16_t)j;
                ++len;
                c = j;
                S = 1.0;
                m = 0;
            }
            if (refused || whole || m == 0) {   // (else the last refusal's sum is R's)
                if (m == 0) begin(c, whole);
                lds_sync();   // sm.left, sm.hist and sm.cell have been read
                if (DRAWN && refused) {
                    if (up_t == c) sm.left[t] = left_t = fmax(left_t - S * q_t, 0.0);
                    if (t == 0) sm.hist[m] = S;
                    refuse(S);
                    ++m;
                }
                total = sum_all(c, m, whole);
                if (refused) {
                    S = total;
                    continue;
                }
            }
            if (total > 0.0 || whole) break;
            whole = true;   // nothing is left
            m = 0;
        }
        if (own == 0) {
            if (t == 0) sm.path[0] = 0;
            lds_sync();
            if (t < a.max_q) a.path[(int64_t)b * a.max_q + t] = t < len ? sm.path[t] : -1;
            if (t == 0) {
                a.kept[b] = len;
                if (!(total > 0.0)) a.token[b] = -1;
            }
        }
        if (!(total > 0.0)) return;
        const double aim = fmax(sm.u[0] * total, 0.0);   // (a NaN gives 0)
        double before = 0.0;
        if (!ONE && a.parts > 1) {
            const double s0 = sm.part[2 * lane], s1 = sm.part[2 * lane + 1], s = s0 + s1, upto = wave_upto(s);
            const uint64_t over = __ballot(s > 0.0 && upto > aim), some = __ballot(s > 0.0);
            const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            if (who) before = readlane_f64(upto, who - 1);
            const double first = readlane_f64(s0, who), second = readlane_f64(s1, who);
            const bool next = second > 0.0 && !(first > 0.0 && before + first > aim);
            if (own != 2 * who + next) return;
            if (next) before += first;
        }
        pick(aim - before);
    }
};

template <typename T, bool DRAWN, bool ONE>
__global__ __launch_bounds__(kVerThreads, DRAWN || ONE ? 4 : 8) void verify_tree_kernel(VerifyParams a) {
    __shared__ typename Verify<T, DRAWN, ONE>::Shared sm;
    const int b = blockIdx.x / a.parts, part = blockIdx.x - b * a.parts;
    if (tree_view(a, b).n == 0) {
        if (part == 0) {
            if ((int)threadIdx.x < a.max_q) a.path[(int64_t)b * a.max_q + threadIdx.x] = -1;
            if (threadIdx.x == 0) {
                a.kept[b] = 0;
                a.token[b] = -1;
            }
        }
        return;
    }
    Verify<T, DRAWN, ONE> v(a, sm, b, part);
    v.run();
}

struct VerifyPlan {
    int parts, passes;
    size_t words, bytes;
};

static VerifyPlan plan_verify(const tms_verify_tree_args* a) {
    VerifyPlan p;
    const int ids = verify_ids(a->dtype == TMS_DTYPE_F32, a->draft != nullptr);
    p.parts = !a->draft && a->dtype != TMS_DTYPE_F32 && a->vocab <= kVerMost ? 1 : (a->vocab + ids - 1) / ids;
    p.passes = a->draft ? a->max_q + 1 : 2;   // the refusals, the last draw, and that again where nothing is left
    p.words = p.parts > 1 ? (size_t)a->batch * p.passes * p.parts : 0;
    p.bytes = p.words * 8;
    return p;
}
static_assert(TMS_VERIFY_MAX_VOCAB <= kVerParts * verify_ids(true, true), "the parts hold a vocabulary");

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
    if (a.draft) hipLaunchKernelGGL((verify_tree_kernel<T, true, false>), grid, dim3(kVerThreads), 0, stream, a);
    else if (sizeof(T) == 2 && a.parts == 1 && a.vocab > verify_ids(false, false))
        hipLaunchKernelGGL((verify_tree_kernel<T, false, sizeof(T) == 2>), grid, dim3(kVerThreads), 0, stream, a);
    else hipLaunchKernelGGL((verify_tree_kernel<T, false, false>), grid, dim3(kVerThreads), 0, stream, a);
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
    a.passes = p.passes;
    a.words = (int64_t)p.words;
    a.polls = g_polls.load(std::memory_order_relaxed);
    if (a.parts > 1) hipLaunchKernelGGL(verify_clear_kernel, dim3(a.words <= 1 << 11 ? 1 : a.words <= 1 << 15 ? 4 : 256), dim3(256), 0, stream, a);
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
