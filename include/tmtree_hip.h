/*
 * tmtree_hip.h -- C ABI of speculative decoding with trees of drafts over the
 * paged cache (gfx950), in the same library as tmcache_hip.h and by its rules:
 * device pointers, a tms_cache, a hipStream_t, an int status; nothing is
 * allocated, synchronised or kept, calls are stream-ordered, can be captured into
 * a HIP graph and run on the current device.
 * TensorMark drafts chains only and verifies them on the host
 * (spec_generate_greedy, tensormark/llama.h:5127-5131); its rotary positions are
 * the model's own: these calls have no counterpart to cite line by line.
 *
 * Trees.  A sequence's new tokens of a call, q_start[b] <= t < q_start[b + 1],
 * are its tree; node i is token q_start[b] + i.  parents[t] is the parent's i, or
 * -1 for a node without one; a parent that is not below the node's own i counts
 * as -1.  Node i is cached at position p0 + i, with p0 = kv_len[b] - (q_start[b + 1]
 * - q_start[b]) as everywhere, and stands at position p0 + depth in the text, its
 * depth being the number of its ancestors: its keys are turned by that.
 * Trees have up to TMS_TREE_MAX_NODES nodes (`max_q`).
 *
 * One step: tms_kv_append_rotary, tms_tree_attention, the model's rest,
 * tms_verify_tree, tms_kv_compact.
 */
#ifndef TMTREE_HIP_H
#define TMTREE_HIP_H

#include "tmcache_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TMS_TREE_MAX_NODES 512
#define TMS_ROTARY_MAX_HEADS 65536
#define TMS_ROTARY_MAX_HEAD_DIM 1024
#define TMS_VERIFY_MAX_VOCAB 1048576
#define TMS_VERIFY_MAX_BATCH 65535
#define TMS_COMPACT_MAX_KEPT 4194304

/*
 * Turn the first rotary_dim values of each head by its token's position: with
 * the angle a_i = position * freqs[i], pair i = (x, y) becomes
 *   (x cos a_i - y sin a_i, y cos a_i + x sin a_i) * scale.
 * Pair i is values i and i + rotary_dim / 2, with `interleaved` values 2 i and 2 i + 1;
 * the values from rotary_dim on are copied.  Angles are reduced in fp64, products and sums
 * are fp32, rounded once to dtype.  The call with negative positions is its gradient, and with
 * 1 / scale undoes it.
 */
typedef struct tms_rotary_args {
    const void* x;            /* device, [tokens][heads][head_dim]; 16-byte aligned */
    void* out;                /* device, like x; may be x itself with x's strides, and
                                 shares no other memory with the inputs */
    int64_t x_stride[2];      /* elements between tokens, heads: multiples of 8 */
    int64_t out_stride[2];
    const int32_t* positions; /* device, [tokens]; any numbers */
    const float* freqs;       /* device, [rotary_dim / 2]: radians a position */
    int32_t dtype;            /* TMS_DTYPE_* */
    int32_t tokens;
    int32_t heads;            /* up to TMS_ROTARY_MAX_HEADS */
    int32_t head_dim;         /* a multiple of 8 up to TMS_ROTARY_MAX_HEAD_DIM */
    int32_t rotary_dim;       /* even, 2..head_dim */
    int32_t interleaved;      /* 0 or 1 */
    float scale;              /* finite */
    int32_t reserved;         /* must be 0 */
} tms_rotary_args;
/* Tokens times threads of a token (a thread turns 16 bytes, or twice 16, of up to eight heads, or copies 16;
 * a value or two, where rotary_dim is not whole pieces) are below 2^32, here and in the next call with
 * max_q for the tokens. */
int tms_rotary(const tms_rotary_args* args, hipStream_t stream);

/*
 * tms_kv_append with the keys turned on their way into the cache, and the
 * queries of the same tokens turned into `out`.  Rows of q that belong to no new token
 * (past the last sequence's, or past max_q of one's) are left out; a token without a mapped
 * slot has its queries turned all the same.  cache->k and cache->v are pools of their own.
 */
typedef struct tms_append_rotary_args {
    const void* k_new;        /* as in tms_append_args */
    const void* v_new;
    int64_t k_new_stride[2];
    int64_t v_new_stride[2];
    const void* q;            /* device, [tokens][q_heads][head_dim] of the cache's dtype,
                                 16-byte aligned; unused with q_heads = 0 */
    void* out;                /* device, like q; may be q itself with q's strides, and
                                 shares no other memory with the inputs */
    int64_t q_stride[2];      /* elements between tokens, heads: multiples of 8 */
    int64_t out_stride[2];
    const int32_t* positions; /* device, [tokens]; null: the position in the cache */
    const float* freqs;       /* device, [rotary_dim / 2] */
    int32_t q_heads;          /* q_heads + kv_heads up to TMS_ROTARY_MAX_HEADS */
    int32_t rotary_dim;
    int32_t interleaved;
    float scale;
} tms_append_rotary_args;
int tms_kv_append_rotary(const tms_cache* cache, const tms_append_rotary_args* args, hipStream_t stream);

/*
 * tms_paged_attention for trees: a node sees the positions below p0, its
 * ancestors and itself (on mapped pages).  With window > 0 it sees those of them whose
 * position in the text is above its own - window or below `sinks`.  parents: device,
 * [tokens].  Everything else, what is rounded and the workspace too, is as there, with its own call for the
 * workspace's size; batch times kv_heads times tiles of 128 rows (32, where a page's stride or slots
 * span 2^32 bytes) is below 2^23.
 */
int64_t tms_tree_attention_workspace(const tms_cache* cache, const tms_attention_args* args);
int tms_tree_attention(const tms_cache* cache, const tms_attention_args* args, const int32_t* parents, hipStream_t stream);

/*
 * Verify drafted trees against the target's probabilities, with given random
 * numbers.  Node 0 of each tree is the last settled token; the walk starts there.  At
 * node c, with R = target row c and S = 1, its children j are tried in order,
 * token x with random number u_j:
 *   accepted where u_j q(x) S < R(x): the walk goes on at j;
 *   else R = max(R - S q, 0), S = sum of R.
 * q is draft row c, the distribution that c's children were drawn from,
 * independently.  Without draft rows the drafts are given: q(x) = 1, and after a refusal
 * R(x) = 0 and S loses what R(x) was.  The step's token is then drawn from what is left of
 * R at the last node: the first id v with R(0) + .. + R(v) > u_0 sum(R), u_0 being node
 * 0's number.  So each step's tokens are distributed as the target's as far as rows sum to 1,
 * what S is at first: by as much as they do not, as by their rounding to 16 bits, it is off.
 * Where nothing is left the token is drawn from the target row, and is -1 where that holds nothing.
 * Entries that are not finite numbers above 0 count as 0, as does a draft outside the vocabulary;
 * products and sums are fp64, sums in a fixed order.  Nodes that node 0 is no ancestor of are never tried.
 */
typedef struct tms_verify_tree_args {
    const void* target;       /* device, [tokens][target_stride] of dtype: row t holds the
                                 probabilities of what follows token t */
    const void* draft;        /* device, [tokens][draft_stride] of dtype, nullable */
    int64_t target_stride;    /* elements, >= vocab */
    int64_t draft_stride;
    int32_t dtype;            /* TMS_DTYPE_* */
    int32_t vocab;            /* up to TMS_VERIFY_MAX_VOCAB */
    int32_t batch;            /* up to TMS_VERIFY_MAX_BATCH */
    int32_t tokens;           /* rows of the tokens' arrays */
    int32_t max_q;            /* nodes of a tree, up to TMS_TREE_MAX_NODES; those past it are left out */
    int32_t reserved;         /* must be 0 */
    const int32_t* draft_tokens; /* device, [tokens]; a node 0's is not read */
    const int32_t* parents;   /* device, [tokens] */
    const int32_t* q_start;   /* device, [batch + 1] */
    const double* uniforms;   /* device, [tokens], in [0, 1) */
    int32_t* path;            /* device, [batch][max_q]: the nodes of the walk from 0 on, -1 past
                                 them; like kept and token it shares no memory with what the call
                                 reads */
    int32_t* kept;            /* device, [batch]: how many they are (the accepted drafts and node 0; 0
                                 without a tree) */
    int32_t* token;           /* device, [batch] */
    void* workspace;          /* device, 16-byte aligned, tms_verify_tree_workspace bytes;
                                 contents need not be kept or cleared */
    size_t workspace_bytes;
} tms_verify_tree_args;
/* Bytes of workspace that the call needs (0 is possible); a TMS_ERR_* code,
 * negative, for arguments that the call would refuse. */
int64_t tms_verify_tree_workspace(const tms_verify_tree_args* args);
int tms_verify_tree(const tms_verify_tree_args* args, hipStream_t stream);
/* Test hook: how often a workgroup of the process's later tms_verify_tree calls looks for
 * another's sum before it works that out itself; negative: the default. */
int tms_debug_verify_polls(int polls);

/*
 * Keep chosen entries of each sequence: entry base + kept[b][i] (key, value and
 * score, of all heads) goes to position base + i, i < n_kept[b], and new_len[b] is
 * base + n_kept[b], 0 at least.  base is p0 with cache->q_start (`kept` then names nodes: the
 * path of a tms_verify_tree), and 0 without.  In place, where kept[i] >= i for every i, the
 * result is as if all entries were read before any is written.  With dst_tables the entries go to the pages of
 * that table instead (of the same pools, and of none that the call reads), from any list.
 * Not copied are entries to or from unmapped pages, with kept[i] outside the sequence, and in
 * place those with kept[i] < i.  A page that two sequences share is written by both, in no order.
 * n_kept is taken as at most max_kept, and in place as at most the sequence's entries from base on.
 * Of the cache's fields `tokens`, `max_q` and `max_kv` are not used; `k` and `v` are pools of their own.
 */
typedef struct tms_compact_args {
    const int32_t* kept;      /* device, [batch][kept_stride] */
    int64_t kept_stride;      /* >= max_kept */
    const int32_t* n_kept;    /* device, [batch] */
    const int32_t* dst_tables; /* device, [batch][dst_table_stride], nullable: in place; not
                                 the cache's tables */
    int64_t dst_table_stride;
    int32_t* new_len;         /* device, [batch], nullable; none of the call's inputs */
    int32_t max_kept;         /* 0..TMS_COMPACT_MAX_KEPT */
    int32_t reserved;         /* must be 0 */
} tms_compact_args;
int tms_kv_compact(const tms_cache* cache, const tms_compact_args* args, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TMTREE_HIP_H */
