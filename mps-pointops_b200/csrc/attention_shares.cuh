// Gradients of keys that many queries see, or that few blocks would form: `shares`
// blocks divide the queries of a key tile; each leaves its sums in float32,
//   partial[tile][key head][share][dk, dv][128][dim],
// and a second kernel adds them in the order of the shares (key_shares below says
// which tiles).  The plan lists key tiles by their number within the cloud, so those
// that are divided stand at the head of the list, and only they get more than one
// block (`shares` blocks for all tiles, most of which ended at once, took 1102
// against 897 us at 8 x 8192 points, 8 heads of 64, and 346 against 292 us at 4 sinks
// of 128 elements).
#pragma once

#include "attention_exact.cuh"

namespace mpo {
namespace {

struct KeyShares {
    int tiles;   // at the head of the list that may be divided
    int limit;   // and are, where their first key is below this
    int shares;  // 1: none is
};
// What block number x of the key/value kernels' list works on.
struct ShareBlock {
    int tile, share;
    bool divided;  // its tile is among those that may be
};
__device__ __forceinline__ ShareBlock share_block(int x, const KeyShares& K) {
    if (x < K.tiles * K.shares) return {x / K.shares, x % K.shares, true};
    return {x - K.tiles * (K.shares - 1), 0, false};
}
// dk row r of a tile in one share's sums; its dv row is kAttnTile * dim on.
__device__ __forceinline__ float* share_sums(const AttnArgs& A, float* partial, int tile, int r, int hk, int shares,
                                             int share) {
    return partial +
           ((((int64_t)tile * A.a.kv_heads + hk) * shares + share) * 2 * kAttnTile + r) * A.a.dim;
}

// grad_k and grad_v of the tiles that are divided: the shares' sums in order.  A
// warp per key row.
template <typename T>
__global__ void __launch_bounds__(256, 3)
attn_join_shares_kernel(const __grid_constant__ AttnArgs A, const KeyShares K, const float* __restrict__ partial) {
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.k_tiles)[blockIdx.x];
    if (t.first >= K.limit) return;
    const int lane = threadIdx.x & 31, hk = blockIdx.y, r = blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r < t.rows) {
        const float* src = share_sums(A, const_cast<float*>(partial), blockIdx.x, r, hk, K.shares, 0);
        const int64_t at = (((int64_t)t.row + r) * A.a.kv_heads + hk) * A.a.dim;
        const int64_t half = (int64_t)kAttnTile * A.a.dim;
        bool nan = false;
        for (int d = lane; d < A.a.dim; d += 32) {
            float dk = 0.f, dv = 0.f;
#pragma unroll 4
            for (int z = 0; z < K.shares; ++z) {
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
int join_shares(const AttnArgs& A, const KeyShares& K, const float* partial, cudaStream_t s) {
    const dim3 grid((unsigned)K.tiles, (unsigned)A.a.kv_heads, kAttnTile / 8);
    attn_join_shares_kernel<T><<<grid, 256, 0, s>>>(A, K, partial);
    return check_launch("attn_join_shares_kernel");
}

}  // namespace

// Sinks: each block about as many queries as see any other key tile, but no more
// blocks than fill the GPU (eight per SM); otherwise one block per key tile with
// sinks would outlast all others (5 times the kernel's time on clouds of 4096 points
// and a window of 512).  All tiles: where there are fewer blocks than half of the SMs,
// as many as fill them, of 64 queries or more (undivided against divided and joined, us:
// float32, clouds of 304, 200 and 100 points, 4 heads of 128 over 1: 455, 70; 700 and 300
// points, 8 heads of 64 over 2, window 400, 4 sinks: 637, 171; bf16, 1024 and 900 points, 8
// over 2, window 600: 61, 26; 2048 points, 16 heads of 128 over 4, causal: 118, 80; one cloud
// of 1024 points, 4 heads of 32, window 256: 10.7, 10.6).  float32 divides the query heads of
// a key head too; with 16-bit types that gave the first of these shapes 23 against 21 us and took the
// registers of the table's kernel (987 against 897 us at 8 x 8192 points).
inline KeyShares key_shares(const AttnArgs& A) {
    const int64_t rows = A.a.max_rows, window = (int64_t)A.left + A.right + kAttnTile;
    const int64_t blocks = (int64_t)A.a.k_tile_count * A.a.kv_heads * (A.a.dtype == MPO_F32 ? 2 : 1);
    KeyShares K = {0, 0, 1};
    if (2 * blocks <= sm_count()) {
        const int64_t seen = (A.a.dtype == MPO_F32 ? A.group : 1) * (A.a.sinks ? rows : min64(rows, window));
        K.shares = (int)max64(1, min64(seen / 64, sm_count() / max64(blocks, 1)));
        if (K.shares > 1) {
            K.tiles = (int)A.a.k_tile_count;
            K.limit = kFar;
        }
    } else if (A.a.sinks) {
        const int64_t sink_tiles = (int64_t)A.a.clouds * ceil_div(A.a.sinks, kAttnTile);
        K.shares = (int)max64(1, min64(rows / window, ceil_div(8 * sm_count(), max64(sink_tiles * A.a.kv_heads, 1))));
        if (K.shares > 1) {
            K.tiles = (int)min64(A.a.k_tile_count, sink_tiles);
            K.limit = A.a.sinks;
        }
    }
    return K;
}
// Blocks of the key/value kernel, in planned tiles.
inline int64_t key_blocks(const AttnArgs& A, const KeyShares& K) {
    return A.a.k_tile_count + (int64_t)K.tiles * (K.shares - 1);
}
inline size_t share_bytes(const AttnArgs& A) {
    const KeyShares K = key_shares(A);
    return K.shares == 1 ? 0 : (size_t)K.tiles * A.a.kv_heads * K.shares * 2 * kAttnTile * A.a.dim * sizeof(float);
}

}  // namespace mpo
