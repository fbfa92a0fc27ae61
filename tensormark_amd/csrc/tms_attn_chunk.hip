// tms_attn_chunk.hip -- attention over the paged cache for many rows a key
// head: chunks of a prompt, long drafts (tms_paged_attention).
//
// Bound by the matrix and the vector pipe about alike (a tile of 64 keys: 1024
// cycles of products, some 1030 of weights a wave), with LDS reads near.
//
// The same mathematics as tms_attn.hip's: S^T = K Q^T, weights 2^(s - m), O^T
// = V^T P^T, m and the sum of weights running per row.  128 rows of one key
// head a workgroup, 32 a wave, on 32x32x16 instructions; a tile of 64 keys and
// values goes to LDS once for the four waves, the next one on the way; two
// workgroups a CU.  Head dimensions past 128 (FUSED) have one workgroup's registers
// and a tile of 32 keys: there the scores of the next keys run among the weights of
// the last within a wave (2048 new tokens over 8192, 256 dimensions: 790 us
// without, 545 with; at 128 dimensions that spills: 526 and 775).
#include "tms_attn_chunk.h"

namespace tms {

template <typename T, int ROWB, int KS, int DT, int NK>
__global__ __launch_bounds__(256, ROWB > 256 ? 1 : 2) void attn_chunk_kernel(AttnParams a) {
    constexpr int KT = 32 * NK, RM = kChunkRows;
    __shared__ ChunkShared<ROWB, NK, 4, false> sm;
    const int pair = blockIdx.x, tile = a.row_tiles - 1 - blockIdx.y, split = blockIdx.z;
    const int b = pair / a.c.kv_heads, h = pair - b * a.c.kv_heads;
    const SeqView sq = seq_view(a.c, b);
    const int rows = sq.n * a.group, r0 = tile * RM;
    if (r0 >= rows) return;
    const TileList<KT> tl(a.window, a.sinks, sq.p0 + r0 / a.group, sq.p0 + (min(r0 + RM, rows) - 1) / a.group, sq.len);
    const int v0 = split * a.split_tiles, v1 = a.splits == split + 1 ? tl.n : min(tl.n, v0 + a.split_tiles);
    chunk_item<T, ROWB, KS, DT, NK, 4, false>(a, sm, sq, b, h, tile, tl, v0, v1,
                                              a.splits > 1 ? ((int64_t)pair * a.row_tiles + tile) * a.splits + split : -1);
}

template <typename T>
static void launch_chunk_type(const AttnParams& a, dim3 grid, hipStream_t stream) {
    const int D = a.c.head_dim;
    if (D <= 64) hipLaunchKernelGGL((attn_chunk_kernel<T, 128, 4, 2, 2>), grid, dim3(256), 0, stream, a);
    else if (D <= 96) hipLaunchKernelGGL((attn_chunk_kernel<T, 256, 6, 3, 2>), grid, dim3(256), 0, stream, a);
    else if (D <= 128) hipLaunchKernelGGL((attn_chunk_kernel<T, 256, 8, 4, 2>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((attn_chunk_kernel<T, 512, 16, 8, 1>), grid, dim3(256), 0, stream, a);
}

void launch_attn_chunk(const AttnParams& a, bool bf16, dim3 grid, hipStream_t stream) {
    if (bf16) launch_chunk_type<Bf16>(a, grid, stream);
    else launch_chunk_type<F16>(a, grid, stream);
}

}  // namespace tms
