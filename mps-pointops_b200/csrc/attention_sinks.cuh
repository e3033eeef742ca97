// Gradients of the keys that stay visible (sinks): every later query of a cloud
// sees them, so one block per key tile would outlast all others (5 times the
// kernel's time on clouds of 4096 points and a window of 512).  `shares` blocks
// divide the queries of a tile that holds sinks; each leaves its sums in float32,
//   partial[cloud * sink tiles + tile][key head][share][dk, dv][128][dim],
// and a second kernel adds them in the order of the shares.  shares == 1: no
// tile is divided.  The plan lists key tiles by their number within the cloud, so
// the tiles with sinks are among the first clouds * sink tiles of the list, and
// only those get `shares` blocks (all tiles with that many blocks, most of which
// ended at once, took 1102 against 897 us at 8 x 8192 points, 8 heads of 64, and 346
// against 292 us at 4 sinks of 128 elements).
#pragma once

#include "attention_exact.cuh"

namespace mpo {
namespace {

__host__ __device__ __forceinline__ int sink_tiles(const AttnArgs& A) {
    return (A.a.sinks + kAttnTile - 1) / kAttnTile;
}
// What block number x of the key/value kernels' list works on.
struct SinkBlock {
    int tile, share;
    bool divided;  // its tile is among those that may be shared out
};
__device__ __forceinline__ SinkBlock sink_block(int x, int divided, int shares) {
    if (x < divided * shares) return {x / shares, x % shares, true};
    return {x - divided * (shares - 1), 0, false};
}
// dk row of key j of a cloud in one share's sums; its dv row is kAttnTile * dim on.
__device__ __forceinline__ float* sink_sums(const AttnArgs& A, float* partial, int cloud, int j, int hk, int shares,
                                            int share) {
    const int64_t tile = (int64_t)cloud * sink_tiles(A) + j / kAttnTile;
    return partial +
           (((tile * A.a.kv_heads + hk) * shares + share) * 2 * kAttnTile + j % kAttnTile) * A.a.dim;
}

// grad_k and grad_v of the key tiles with sinks: the shares' sums in order.  A
// warp per key row.
template <typename T>
__global__ void __launch_bounds__(256)
attn_join_sinks_kernel(const __grid_constant__ AttnArgs A, int shares, const float* __restrict__ partial) {
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.k_tiles)[blockIdx.x];
    if (t.first >= A.a.sinks) return;
    const int lane = threadIdx.x & 31, hk = blockIdx.y, r = blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r < t.rows) {
        const float* src = sink_sums(A, const_cast<float*>(partial), t.cloud, t.first + r, hk, shares, 0);
        const int64_t at = (((int64_t)t.row + r) * A.a.kv_heads + hk) * A.a.dim;
        const int64_t half = (int64_t)kAttnTile * A.a.dim;
        bool nan = false;
        for (int d = lane; d < A.a.dim; d += 32) {
            float dk = 0.f, dv = 0.f;
#pragma unroll 4
            for (int z = 0; z < shares; ++z) {
                dk += src[z * 2 * half + d];
                dv += src[(z * 2 + 1) * half + d];
            }
            nan |= !isfinite(dk) | !isfinite(dv);
            static_cast<T*>(A.a.grad_k)[at + d] = Elem<T>::from(dk);
            static_cast<T*>(A.a.grad_v)[at + d] = Elem<T>::from(dv);
        }
        if (__any_sync(FULL_MASK, nan)) {
            __syncwarp();
            exact_grad_kv_row<T>(A, t.base, t.first + r, t.other, t.lq, t.lk, hk);
        }
    }
}

template <typename T>
int join_sinks(const AttnArgs& A, int divided, int shares, const float* partial, cudaStream_t s) {
    const dim3 grid((unsigned)divided, (unsigned)A.a.kv_heads, kAttnTile / 8);
    attn_join_sinks_kernel<T><<<grid, 256, 0, s>>>(A, shares, partial);
    return check_launch("attn_join_sinks_kernel");
}

}  // namespace

// Blocks that share a key tile with sinks: each about as many queries as see
// any other key tile, but no more blocks than fill the GPU (eight per SM).
inline int sink_shares(const AttnArgs& A) {
    if (A.a.sinks == 0) return 1;
    const int64_t window = (int64_t)A.left + A.right + kAttnTile;
    const int64_t tiles = (int64_t)A.a.clouds * sink_tiles(A) * A.a.kv_heads;
    return (int)max64(1, min64(A.a.max_rows / window, ceil_div(8 * sm_count(), max64(tiles, 1))));
}
// Key tiles, from the head of the list, that `shares` blocks divide where they hold sinks.
inline int sink_divided(const AttnArgs& A, int shares) {
    return shares == 1 ? 0 : (int)min64(A.a.k_tile_count, (int64_t)A.a.clouds * sink_tiles(A));
}
inline size_t sink_bytes(const AttnArgs& A) {
    const int shares = sink_shares(A);
    if (shares == 1) return 0;
    const int64_t tiles = (int64_t)A.a.clouds * sink_tiles(A);
    return (size_t)(tiles * A.a.kv_heads * shares * 2 * kAttnTile * A.a.dim) * sizeof(float);
}

}  // namespace mpo
