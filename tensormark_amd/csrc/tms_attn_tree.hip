// tms_attn_tree.hip -- attention of drafted trees over the paged cache for many rows a key head
// (tms_tree_attention); up to 32 rows take the rows kernel of tms_attn.hip.
//
// The mathematics of tms_attn_chunk.hip's: S^T = K Q^T, weights 2^(s - m), O^T = V^T P^T, m and
// the sum of weights running per row.  A row sees the prefix and the nodes of its own line, a
// bit each in LDS (TreeRows); the mask is read only in tiles that hold new tokens, or a window's edge.
//
// Few rows over long prefixes (8 nodes and 4 heads a key head are 32 rows): bound by memory, so a
// key is read once for all rows of its head, 256 of them in 8 waves where there are more than 128.  32 sequences of 257
// to 8192, 9 to 25 nodes, 8 key heads of 128, 4 heads each, bf16: 129 us, 562 MB, 4.4 TB/s (the card copies
// at 5.0).  8 of 9000 to 16384 with 64 nodes: 142 to 155 us by card and clock, 106 GFLOP, 680 to 740 TFLOP/s (a large
// product: 1230).  Products have 46 % of a SIMD's cycles there and vector instructions 45 %, where the same loop has 60
// and 54 % for a prompt's chunk, in two workgroups a CU: one workgroup's waves come to the barrier and to the
// weights of a tile's first half together, and wait a third of their time (22 % there).  At 142 us: 153 with 128 rows a
// workgroup; 164 with one half of the waves half a tile behind the other; 160 with four tiles on their way.
// Past 128 dimensions a wave's outputs and queries alone are 192 registers, so a workgroup has 128 rows, and more rows
// read the keys again: the 32 sequences with heads of 256 288 us, 3.9 TB/s, the 8 365 us, 580 TFLOP/s.
#include "tms_attn_chunk.h"

namespace tms {

__device__ __forceinline__ int64_t uniform(int64_t x) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

// A share of the axis (TreeAxis), or an item a workgroup.
template <typename T, int ROWB, int KS, int DT, int NK, int NW>
__global__ __launch_bounds__(64 * NW, 2 * (ROWB > 256 ? 1 : 2) / (NW / 2)) void attn_tree_kernel(AttnParams a) {
    constexpr int KT = 32 * NK, RM = 32 * NW;
    typedef TreeAxis<KT, RM> Axis;
    __shared__ ChunkShared<ROWB, NK, NW, true> sm;
    __shared__ int64_t wsum[NW + 2];   // then where the share starts
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int H = a.c.kv_heads, combos = a.c.batch * a.row_tiles;
    // The share: [x, end) of the axis, which starts in `combo` at `at`.  Without shares, an item a workgroup.
    int64_t share = 0, x = 0, end = 1, at = 0;
    int combo = blockIdx.x / H;
    if (a.split_tiles > 0) {
        const int per = (combos + 64 * NW - 1) / (64 * NW), c0 = min(t * per, combos), c1 = min(c0 + per, combos);
        int64_t mine = 0;
        for (int c = c0; c < c1; ++c) mine += Axis::combo(a, c);
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
        total = uniform(total) * H;
        share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)a.split_tiles);
        x = blockIdx.x * share;
        end = min(x + share, total);
        if (x >= end) return;
        if (x >= before * H && x < (before + mine) * H)
            for (int c = c0;; ++c) {
                const int n = Axis::combo(a, c);
                if (x < (before + n) * H) {
                    wsum[NW] = c;
                    wsum[NW + 1] = before * H;
                    break;
                }
                before += n;
            }
        __syncthreads();
        combo = __builtin_amdgcn_readfirstlane((int)wsum[NW]);
        at = uniform(wsum[NW + 1]);
    }
    while (x < end) {
        const int b = combo / a.row_tiles, tile = combo - b * a.row_tiles;
        const SeqView sq = seq_view(a.c, b);
        const int rows = sq.n * a.group, r0 = tile * RM;
        if (r0 >= rows) {
            if (a.split_tiles == 0) return;
            ++combo;
            continue;
        }
        const TileList<KT> tl(a.window, a.sinks, sq.p0, sq.p0 + (min(r0 + RM, rows) - 1) / a.group, sq.len);
        const int n = max(tl.n, 1), axis = Axis::length(tl.n);
        int h = blockIdx.x - combo * H, k0 = 0, k1 = n;
        bool whole = true;
        if (a.split_tiles > 0) {
            if (x >= at + (int64_t)axis * H) {
                at += (int64_t)axis * H;
                ++combo;
                continue;
            }
            h = (int)((x - at) / axis);
            const int64_t item = at + (int64_t)h * axis;
            k0 = (int)(x - item);
            k1 = (int)min((int64_t)n, end - item);
            x = min(item + axis, end);
            if (k0 >= n) continue;
            whole = k0 == 0 && k1 == n;
            if (k0 == 0 && t == 0)
                a.item_parts[combo * H + h] = make_int2(blockIdx.x, whole ? 0 : (int)((item + n - 1) / share) - (int)blockIdx.x + 1);
        }
        chunk_item<T, ROWB, KS, DT, NK, NW, true>(a, sm, sq, b, h, tile, tl, k0, min(k1, tl.n),
                                                  whole ? -1 : 2 * (int64_t)blockIdx.x + (k0 == 0 ? 1 : 0));
        if (a.split_tiles == 0) return;
        __syncthreads();   // its tiles are read
    }
}

template <typename T>
static void launch_tree_type(const AttnParams& a, int rows, int workgroups, hipStream_t stream) {
    const int D = a.c.head_dim;
    const dim3 grid(workgroups);
    if (D > 128) hipLaunchKernelGGL((attn_tree_kernel<T, 512, 16, 8, 1, 4>), grid, dim3(256), 0, stream, a);
    else if (rows == 128) {
        if (D <= 64) hipLaunchKernelGGL((attn_tree_kernel<T, 128, 4, 2, 2, 4>), grid, dim3(256), 0, stream, a);
        else if (D <= 96) hipLaunchKernelGGL((attn_tree_kernel<T, 256, 6, 3, 2, 4>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((attn_tree_kernel<T, 256, 8, 4, 2, 4>), grid, dim3(256), 0, stream, a);
    } else {
        if (D <= 64) hipLaunchKernelGGL((attn_tree_kernel<T, 128, 4, 2, 2, 8>), grid, dim3(512), 0, stream, a);
        else if (D <= 96) hipLaunchKernelGGL((attn_tree_kernel<T, 256, 6, 3, 2, 8>), grid, dim3(512), 0, stream, a);
        else hipLaunchKernelGGL((attn_tree_kernel<T, 256, 8, 4, 2, 8>), grid, dim3(512), 0, stream, a);
    }
}

void launch_attn_chunk_tree(const AttnParams& a, bool bf16, int rows, int workgroups, hipStream_t stream) {
    if (bf16) launch_tree_type<Bf16>(a, rows, workgroups, stream);
    else launch_tree_type<F16>(a, rows, workgroups, stream);
}

}  // namespace tms
