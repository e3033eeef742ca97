// Attention of serialised clouds for float32 (definitions:
// attention_common.cuh): tiles of 64 x 64 pairs with fused multiply-adds.
//
// 128 threads; thread (ty, tx) = (tid / 16, tid % 16) holds rows 8 ty .. 8 ty + 7
// and columns tx, tx + 16, tx + 32, tx + 48 of a tile of scores, and rows
// 8 ty .. of the accumulated rows with the elements tx W .. (W = DP / 16).  Per
// four elements of a dot product a thread loads 8 + 4 vectors of 16 bytes for
// 128 multiply-adds, about half of what shared memory can deliver in that
// time.  3 ragged clouds of up to 4096 points, 4 heads of 32, window 512, a table:
// forward 126, queries 325, keys and values 287 us, where the products alone would
// take 30, 44 and 59 us of the FP32 pipes' 74 TFLOP/s: at 32 elements the bias of a
// pair (and the table's cells) costs more than its products, and there are at most
// 768 blocks of 64 rows, of unequal clouds.
#include <string>

#include "attention_shares.cuh"

namespace mpo {
namespace {

constexpr int kTR = 64;       // rows and columns of a tile
constexpr int kPS = kTR + 4;  // row pitch of the tile of weights
constexpr int kThreads = 128;

template <int DP>
struct Pitch {
    static constexpr int v = DP + 4;  // floats; keeps 16-byte rows and spreads the banks
};

struct SimtSmem {
    float* rows[4];  // operand tiles
    float* w;        // [64][kPS]
    float* lse2;     // [64]
    float* delta;    // [64]
    float* table;    // [kAttnMaxEntries], times log2(e)
    int* rpos;       // [3][64] positions of the resident side
    int* cpos;       // [3][64] positions of the streamed side
    uint8_t* map;    // [kAttnMaxMap]
    float* hist;     // [entries][64]
    static size_t bytes(int dp, int operands, int hist_entries) {
        size_t n = (size_t)operands * kTR * (dp + 4) * 4 + kTR * kPS * 4 + 2 * kTR * 4 +
                   kAttnMaxEntries * 4 + 6 * kTR * 4 + (kAttnMaxMap + 15) / 16 * 16;
        return n + (size_t)hist_entries * 64 * 4;
    }
    __device__ SimtSmem(unsigned char* p, int dp, int operands) {
        float* f = reinterpret_cast<float*>(p);
        for (int i = 0; i < 4; ++i) {
            rows[i] = f;
            if (i < operands) f += kTR * (dp + 4);
        }
        w = f;
        lse2 = w + kTR * kPS;
        delta = lse2 + kTR;
        table = delta + kTR;
        rpos = reinterpret_cast<int*>(table + kAttnMaxEntries);
        cpos = rpos + 3 * kTR;
        map = reinterpret_cast<uint8_t*>(cpos + 3 * kTR);
        hist = reinterpret_cast<float*>(map + (kAttnMaxMap + 15) / 16 * 16);
    }
};

// rows [r0, r0 + n) of one head as floats, zeros past n and past dim.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(float* dst, const void* base, int64_t r0, int n, int h,
                                          int64_t row_stride, int64_t head_stride, int dim) {
    constexpr int kChunks = DP / Elem<T>::kVec;
    for (int c = threadIdx.x; c < kTR * kChunks; c += kThreads) {
        const int r = c / kChunks, d = (c % kChunks) * Elem<T>::kVec;
        float x[Elem<T>::kVec];
#pragma unroll
        for (int e = 0; e < Elem<T>::kVec; ++e) x[e] = 0.f;
        if (r < n && d < dim)
            Elem<T>::unpack(*reinterpret_cast<const uint4*>(
                                attn_row<T>(base, r0 + r, h, row_stride, head_stride) + d), x);
#pragma unroll
        for (int e = 0; e < Elem<T>::kVec; e += 4)
            *reinterpret_cast<float4*>(dst + r * Pitch<DP>::v + d + e) =
                make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    }
}
__device__ __forceinline__ void load_pos(int* dst, const int32_t* pos, int64_t r0, int n, int axes) {
    for (int c = threadIdx.x; c < kTR * axes; c += kThreads) {
        const int r = c / axes, a = c % axes;
        dst[a * kTR + r] = r < n ? pos[(r0 + r) * axes + a] : 0;
    }
}
__device__ __forceinline__ void load_bias(const AttnArgs& A, const SimtSmem& S, int h) {
    for (int e = threadIdx.x; e < A.a.axes * A.a.buckets; e += kThreads)
        S.table[e] = table_entry(A.a, e, h) * kLog2e;
    if (A.a.map)
        for (int e = threadIdx.x; e <= 2 * A.a.reach; e += kThreads)
            S.map[e] = (uint8_t)min(max(A.a.map[e], 0), A.a.buckets - 1);
}

// acc[i][c] += sum_d a[8 ty + i][d] * b[tx + 16 c][d]
template <int DP>
__device__ __forceinline__ void product_nt(float (&acc)[8][4], const float* a, const float* b) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 y[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            y[c] = *reinterpret_cast<const float4*>(b + (tx + 16 * c) * Pitch<DP>::v + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(a + (8 * ty + i) * Pitch<DP>::v + d);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                acc[i][c] = fmaf(x.x, y[c].x, acc[i][c]);
                acc[i][c] = fmaf(x.y, y[c].y, acc[i][c]);
                acc[i][c] = fmaf(x.z, y[c].z, acc[i][c]);
                acc[i][c] = fmaf(x.w, y[c].w, acc[i][c]);
            }
        }
    }
}
// acc[i][e] += sum_k w[8 ty + i][k] * b[k][tx W + e]
template <int DP>
__device__ __forceinline__ void product_nn(float (&acc)[8][DP / 16], const float* w, const float* b) {
    constexpr int W = DP / 16;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 2
    for (int k = 0; k < kTR; k += 4) {
        float y[4][W];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float* src = b + (k + j) * Pitch<DP>::v + tx * W;
            if constexpr (W % 4 == 0) {
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(src + e);
                    y[j][e] = t.x; y[j][e + 1] = t.y; y[j][e + 2] = t.z; y[j][e + 3] = t.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) y[j][e] = src[e];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(w + (8 * ty + i) * kPS + k);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                acc[i][e] = fmaf(x.x, y[0][e], acc[i][e]);
                acc[i][e] = fmaf(x.y, y[1][e], acc[i][e]);
                acc[i][e] = fmaf(x.z, y[2][e], acc[i][e]);
                acc[i][e] = fmaf(x.w, y[3][e], acc[i][e]);
            }
        }
    }
}

// Scores of a tile in units of log2, -inf where invisible.  Rows are queries
// (TRANSPOSED: keys) of the resident side, columns the streamed side's.  `whole`:
// every pair of the tile is visible.
template <bool TRANSPOSED>
__device__ __forceinline__ void finish_scores(const AttnArgs& A, const SimtSmem& S, float (&s)[8][4],
                                              int p0, int rows, int j0, int cols, bool whole) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][c] *= A.scale_log2;
    for (int a = 0; a < A.a.axes; ++a) {
        const float* table = S.table + a * A.a.buckets;
        int cp[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) cp[c] = S.cpos[a * kTR + tx + 16 * c];
        const int4 lo = *reinterpret_cast<const int4*>(S.rpos + a * kTR + 8 * ty);
        const int4 hi = *reinterpret_cast<const int4*>(S.rpos + a * kTR + 8 * ty + 4);
        const int rp[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int d = TRANSPOSED ? rp[i] - cp[c] : cp[c] - rp[i];
                int b = min(max(d, -A.a.reach), A.a.reach) + A.a.reach;
                if (A.a.map) b = S.map[b];
                s[i][c] += table[b];
            }
    }
    if (whole) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int r = 8 * ty + i, col = tx + 16 * c;
            const int p = TRANSPOSED ? j0 + col : p0 + r, j = TRANSPOSED ? p0 + r : j0 + col;
            if (!(r < rows && col < cols && attn_visible(A, p, j))) s[i][c] = -INFINITY;
        }
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL_MASK, v, o));
    return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

// The 64 rows of a planned tile that this block owns; false when it has none.
struct Half {
    AttnTile t;
    int rows, p0;
    int64_t row;
    __device__ __forceinline__ bool load(const int32_t* tiles, int half) {
        t = reinterpret_cast<const AttnTile*>(tiles)[half >> 1];
        const int off = (half & 1) * kTR;
        rows = min(kTR, t.rows - off);
        p0 = t.first + off;
        row = (int64_t)t.row + off;
        return rows > 0;
    }
};

// ---------------------------------------------------------------- forward
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_simt_fwd_kernel(const __grid_constant__ AttnArgs A) {
    extern __shared__ __align__(16) unsigned char smem[];
    const SimtSmem S(smem, DP, 3);
    constexpr int W = DP / 16;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, h = blockIdx.y, hk = h / A.group;
    Half H;
    if (!H.load(A.a.q_tiles, blockIdx.x)) return;
    load_rows<T, DP>(S.rows[0], A.a.q, H.row, H.rows, h, A.a.q_row, A.a.q_head, A.a.dim);
    if (A.a.table) {
        load_bias(A, S, h);
        load_pos(S.rpos, A.a.qpos, H.row, H.rows, A.a.axes);
    }
    float o[8][W], m[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) o[i][e] = 0.f;
    }
    const KeySpan span = key_span(A, H.p0, H.p0 + H.rows - 1, H.t.lk, kTR);
    for (int t = 0; t < span.count(); ++t) {
        const int k0 = span.tile(t) * kTR, n = min(kTR, H.t.lk - k0);
        const int64_t kr = (int64_t)H.t.other + k0;
        __syncthreads();
        load_rows<T, DP>(S.rows[1], A.a.k, kr, n, hk, A.a.k_row, A.a.k_head, A.a.dim);
        load_rows<T, DP>(S.rows[2], A.a.v, kr, n, hk, A.a.v_row, A.a.v_head, A.a.dim);
        if (A.a.table) load_pos(S.cpos, A.a.kpos, kr, n, A.a.axes);
        __syncthreads();
        float s[8][4];
        product_nt<DP>(s, S.rows[0], S.rows[1]);
        finish_scores<false>(A, S, s, H.p0, H.rows, k0, n,
                             n == kTR && H.rows == kTR && all_visible(A, H.p0, H.p0 + kTR - 1, k0, k0 + kTR - 1));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float top = half_warp_max(fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
            const float mn = fmaxf(m[i], top), ref = mn == -INFINITY ? 0.f : mn;
            const float f = exp2_sfu(m[i] - ref);
            m[i] = mn;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float w = exp2_sfu(s[i][c] - ref);
                sum += w;
                S.w[(8 * ty + i) * kPS + tx + 16 * c] = w;
            }
            l[i] = fmaf(l[i], f, sum);  // this thread's columns only, joined at the end
#pragma unroll
            for (int e = 0; e < W; ++e) o[i][e] *= f;
        }
        __syncwarp();  // a row of weights is written and read by the same half warp
        product_nn<DP>(o, S.w, S.rows[2]);
    }
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float sum = half_warp_sum(l[i]);
        const int r = 8 * ty + i;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        bool nan = false;
        if (r < H.rows) {
            const int64_t at = ((H.row + r) * A.a.heads + h) * A.a.dim + tx * W;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float v = o[i][e] * inv;
                nan |= isnan(v);
                if (tx * W + e < A.a.dim) {
                    static_cast<T*>(A.a.out)[at + e] = Elem<T>::from(v);
                }
            }
            if (A.a.lse && tx == 0)
                A.a.lse[(int64_t)h * A.a.q_rows + H.row + r] =
                    sum == 0.f ? -INFINITY : fmaf(m[i], kLn2, logf(sum));
        }
        const unsigned b = __ballot_sync(FULL_MASK, nan);
        if (b & 0xffffu) bad |= 1u << i;
        if (b >> 16) bad |= 1u << (8 + i);
    }
    __syncwarp();
    for (; bad; bad &= bad - 1) {  // rows of this warp: 16 (warp) + bit
        const int r = (threadIdx.x >> 5) * 16 + __ffs(bad) - 1;
        exact_forward_row<T>(A, H.row + r, H.p0 + r, H.t.other, H.t.lk, h);
    }
}

// ---------------------------------------------------------------- backward: queries
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_simt_grad_q_kernel(const __grid_constant__ AttnArgs A, float* partial) {
    extern __shared__ __align__(16) unsigned char smem[];
    const SimtSmem S(smem, DP, 4);
    constexpr int W = DP / 16;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, h = blockIdx.y, hk = h / A.group;
    const int entries = A.a.axes * A.a.buckets;
    Half H;
    const bool mine = H.load(A.a.q_tiles, blockIdx.x);
    if (!mine) {
        if (partial)
            for (int e = threadIdx.x; e < entries; e += kThreads)
                partial[((int64_t)blockIdx.x * A.a.heads + h) * entries + e] = 0.f;
        return;
    }
    const int64_t o_row = (int64_t)A.a.heads * A.a.dim;
    load_rows<T, DP>(S.rows[0], A.a.q, H.row, H.rows, h, A.a.q_row, A.a.q_head, A.a.dim);
    load_rows<T, DP>(S.rows[1], A.a.grad_out, H.row, H.rows, h, o_row, A.a.dim, A.a.dim);
    if (A.a.table) {
        load_bias(A, S, h);
        load_pos(S.rpos, A.a.qpos, H.row, H.rows, A.a.axes);
    }
    if (partial)
        for (int e = threadIdx.x; e < entries * 64; e += kThreads) S.hist[e] = 0.f;
    __syncthreads();
    {   // D_i = o . do, two threads per row
        const int r = threadIdx.x >> 1;
        float sum = 0.f;
        if (r < H.rows) {
            const int64_t at = ((H.row + r) * A.a.heads + h) * A.a.dim;
            for (int d = threadIdx.x & 1; d < A.a.dim; d += 2) {
                const float ov = Elem<T>::to(static_cast<const T*>(A.a.out)[at + d]);
                sum = fmaf(ov, S.rows[1][r * Pitch<DP>::v + d], sum);
            }
        }
        sum += __shfl_xor_sync(FULL_MASK, sum, 1);
        if (!(threadIdx.x & 1)) {
            S.delta[r] = sum;
            S.lse2[r] = r < H.rows ? load_lse2(A, H.row + r, h) : INFINITY;
            if (r < H.rows) A.a.delta[(int64_t)h * A.a.q_rows + H.row + r] = sum;
        }
    }
    float dq[8][W];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) dq[i][e] = 0.f;
    const KeySpan span = key_span(A, H.p0, H.p0 + H.rows - 1, H.t.lk, kTR);
    for (int t = 0; t < span.count(); ++t) {
        const int k0 = span.tile(t) * kTR, n = min(kTR, H.t.lk - k0);
        const int64_t kr = (int64_t)H.t.other + k0;
        __syncthreads();
        load_rows<T, DP>(S.rows[2], A.a.k, kr, n, hk, A.a.k_row, A.a.k_head, A.a.dim);
        load_rows<T, DP>(S.rows[3], A.a.v, kr, n, hk, A.a.v_row, A.a.v_head, A.a.dim);
        if (A.a.table) load_pos(S.cpos, A.a.kpos, kr, n, A.a.axes);
        __syncthreads();
        float s[8][4], dp[8][4];
        product_nt<DP>(s, S.rows[0], S.rows[2]);
        finish_scores<false>(A, S, s, H.p0, H.rows, k0, n,
                             n == kTR && H.rows == kTR && all_visible(A, H.p0, H.p0 + kTR - 1, k0, k0 + kTR - 1));
        product_nt<DP>(dp, S.rows[1], S.rows[3]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 8 * ty + i;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                S.w[r * kPS + tx + 16 * c] =
                    s[i][c] == -INFINITY ? 0.f
                                         : exp2_sfu(s[i][c] - S.lse2[r]) * (dp[i][c] - S.delta[r]);
        }
        __syncwarp();
        product_nn<DP>(dq, S.w, S.rows[2]);
        if (partial) {
            __syncthreads();
            // A row per thread and half block, columns in a rotated order (spreads the banks);
            // even axes by the first 64 threads, odd ones by the others, so cell (entry, row)
            // belongs to one thread.  Two columns at a time: where both meet in one cell the
            // second sum carries the first, and is written last.
            const int r = threadIdx.x & 63;
            for (int a = threadIdx.x >> 6; a < A.a.axes; a += 2) {
                float* cells = S.hist + (size_t)a * A.a.buckets * 64 + r;
                const int rp = S.rpos[a * kTR + r];
                const uint8_t* map = A.a.map ? S.map : nullptr;
#pragma unroll 4
                for (int c = 0; c < kTR; c += 2) {
                    const int c0 = (c + r) & 63, c1 = (c + 1 + r) & 63;
                    const int x = bias_bucket(S.cpos[a * kTR + c0], rp, A.a.reach, map) * 64;
                    const int y = bias_bucket(S.cpos[a * kTR + c1], rp, A.a.reach, map) * 64;
                    const float u = cells[x] + S.w[r * kPS + c0];
                    const float v = (x == y ? u : cells[y]) + S.w[r * kPS + c1];
                    cells[x] = u;
                    cells[y] = v;
                }
            }
        }
    }
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 8 * ty + i;
        bool nan = false;
        if (r < H.rows) {
            const int64_t at = ((H.row + r) * A.a.heads + h) * A.a.dim + tx * W;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                nan |= isnan(dq[i][e]);
                if (tx * W + e < A.a.dim)
                    static_cast<T*>(A.a.grad_q)[at + e] = Elem<T>::from(dq[i][e] * A.a.scale);
            }
        }
        const unsigned b = __ballot_sync(FULL_MASK, nan);
        if (b & 0xffffu) bad |= 1u << i;
        if (b >> 16) bad |= 1u << (8 + i);
    }
    __syncthreads();
    for (; bad; bad &= bad - 1) {
        const int r = (threadIdx.x >> 5) * 16 + __ffs(bad) - 1;
        exact_grad_q_row<T>(A, H.row + r, H.p0 + r, H.t.other, H.t.lk, h);
    }
    if (partial)
        for (int e = threadIdx.x; e < entries; e += kThreads) {
            float v = 0.f;
            for (int r = 0; r < 64; ++r) v += S.hist[e * 64 + ((r + e) & 63)];
            partial[((int64_t)blockIdx.x * A.a.heads + h) * entries + e] = v;
        }
}

// ---------------------------------------------------------------- backward: keys and values
// Three blocks per SM up to 32 elements: at two (234 registers) the time was 270 us or,
// in some runs, 457, against 287.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, DP <= 32 ? 3 : 1)
attn_simt_grad_kv_kernel(const __grid_constant__ AttnArgs A, const KeyShares K,
                         float* __restrict__ partial) {
    extern __shared__ __align__(16) unsigned char smem[];
    const SimtSmem S(smem, DP, 4);
    constexpr int W = DP / 16;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, hk = blockIdx.y;
    Half H;  // p0: index of the first key
    const ShareBlock block = share_block(blockIdx.x >> 1, K);
    if (!H.load(A.a.k_tiles, 2 * block.tile + ((int)blockIdx.x & 1))) return;
    // The planned tile decides: both of its halves are shared out or neither is.
    const bool shared = block.divided && H.t.first < K.limit;
    if (!shared && block.share > 0) return;
    const int64_t o_row = (int64_t)A.a.heads * A.a.dim;
    load_rows<T, DP>(S.rows[0], A.a.k, H.row, H.rows, hk, A.a.k_row, A.a.k_head, A.a.dim);
    load_rows<T, DP>(S.rows[1], A.a.v, H.row, H.rows, hk, A.a.v_row, A.a.v_head, A.a.dim);
    if (A.a.table) load_pos(S.rpos, A.a.kpos, H.row, H.rows, A.a.axes);
    float dk[8][W], dv[8][W];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) dk[i][e] = dv[i][e] = 0.f;
    int lo, hi;
    query_span(A, H.p0, H.p0 + H.rows - 1, H.t.lq, H.t.lk, lo, hi);
    // `count` tiles of queries for each query head in turn, of which this block takes its share.
    const int count = hi > lo ? (hi - lo + kTR - 1) / kTR : 0;
    int begin = 0, end = count * A.group;
    if (shared) {
        begin = (int)((int64_t)count * A.group * block.share / K.shares);
        end = (int)((int64_t)count * A.group * (block.share + 1) / K.shares);
    }
    for (int h = hk * A.group; h < (hk + 1) * A.group; ++h, begin -= count, end -= count) {
        if (begin >= count || end <= 0) continue;
        __syncthreads();
        if (A.a.table) load_bias(A, S, h);
        for (int i0 = lo + max(begin, 0) * kTR; i0 < min(hi, lo + end * kTR); i0 += kTR) {
            const int n = min(kTR, hi - i0);
            const int64_t qr = (int64_t)H.t.other + i0;
            __syncthreads();
            load_rows<T, DP>(S.rows[2], A.a.q, qr, n, h, A.a.q_row, A.a.q_head, A.a.dim);
            load_rows<T, DP>(S.rows[3], A.a.grad_out, qr, n, h, o_row, A.a.dim, A.a.dim);
            if (A.a.table) load_pos(S.cpos, A.a.qpos, qr, n, A.a.axes);
            if (threadIdx.x < kTR) {
                const int c = threadIdx.x;
                S.lse2[c] = c < n ? load_lse2(A, qr + c, h) : INFINITY;
                S.delta[c] = c < n ? A.a.delta[(int64_t)h * A.a.q_rows + qr + c] : 0.f;
            }
            __syncthreads();
            float s[8][4];
            product_nt<DP>(s, S.rows[0], S.rows[2]);
            const int q0 = i0 + H.t.lk - H.t.lq;
            finish_scores<true>(A, S, s, H.p0, H.rows, q0, n,
                                n == kTR && H.rows == kTR && all_visible(A, q0, q0 + kTR - 1, H.p0, H.p0 + kTR - 1));
            unsigned seen = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (s[i][c] != -INFINITY) seen |= 1u << (4 * i + c);
                    s[i][c] = exp2_sfu(s[i][c] - S.lse2[tx + 16 * c]);
                    S.w[(8 * ty + i) * kPS + tx + 16 * c] = s[i][c];
                }
            __syncwarp();
            product_nn<DP>(dv, S.w, S.rows[3]);
            float dp[8][4];
            product_nt<DP>(dp, S.rows[1], S.rows[3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    S.w[(8 * ty + i) * kPS + tx + 16 * c] =
                        (seen >> (4 * i + c)) & 1u ? s[i][c] * (dp[i][c] - S.delta[tx + 16 * c]) : 0.f;
            __syncwarp();
            product_nn<DP>(dk, S.w, S.rows[2]);
        }
    }
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 8 * ty + i;
        bool nan = false;
        if (r < H.rows) {
            const int64_t at = ((H.row + r) * A.a.kv_heads + hk) * A.a.dim + tx * W;
            float* sums =
                shared ? share_sums(A, partial, block.tile, H.p0 - H.t.first + r, hk, K.shares, block.share) + tx * W
                       : nullptr;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                nan |= isnan(dk[i][e]) | isnan(dv[i][e]);
                if (tx * W + e >= A.a.dim) continue;
                if (sums) {
                    sums[e] = dk[i][e] * A.a.scale;
                    sums[(int64_t)kAttnTile * A.a.dim + e] = dv[i][e];
                } else {
                    static_cast<T*>(A.a.grad_k)[at + e] = Elem<T>::from(dk[i][e] * A.a.scale);
                    static_cast<T*>(A.a.grad_v)[at + e] = Elem<T>::from(dv[i][e]);
                }
            }
        }
        const unsigned b = __ballot_sync(FULL_MASK, nan);
        if (b & 0xffffu) bad |= 1u << i;
        if (b >> 16) bad |= 1u << (8 + i);
    }
    __syncwarp();
    for (; bad && !shared; bad &= bad - 1) {
        const int r = (threadIdx.x >> 5) * 16 + __ffs(bad) - 1;
        exact_grad_kv_row<T>(A, (int64_t)H.t.base, H.p0 + r, H.t.other, H.t.lq, H.t.lk, hk);
    }
}

// ---------------------------------------------------------------- launches
template <typename T, int DP>
int run_fwd(const AttnArgs& A, cudaStream_t s) {
    const size_t bytes = SimtSmem::bytes(DP, 3, 0);
    const int st = attn_prepare<&attn_simt_fwd_kernel<T, DP>>("attn_simt_fwd_kernel");
    if (st != kOk) return st;
    const dim3 grid((unsigned)(2 * A.a.q_tile_count), (unsigned)A.a.heads);
    attn_simt_fwd_kernel<T, DP><<<grid, kThreads, bytes, s>>>(A);
    return check_launch("attn_simt_fwd_kernel");
}
template <typename T, int DP>
int run_bwd(const AttnArgs& A, cudaStream_t s) {
    const int entries = A.a.axes * A.a.buckets;
    float* sums = static_cast<float*>(A.a.workspace);
    float* partial = A.a.grad_table ? reinterpret_cast<float*>(
                                          static_cast<unsigned char*>(A.a.workspace) + share_bytes(A))
                                    : nullptr;
    const size_t qb = SimtSmem::bytes(DP, 4, partial ? entries : 0);
    const size_t kb = SimtSmem::bytes(DP, 4, 0);
    int st = attn_prepare<&attn_simt_grad_q_kernel<T, DP>>("attn_simt_grad_q_kernel");
    if (st == kOk) st = attn_prepare<&attn_simt_grad_kv_kernel<T, DP>>("attn_simt_grad_kv_kernel");
    if (st != kOk) return st;
    if (A.a.q_tile_count) {
        const dim3 grid((unsigned)(2 * A.a.q_tile_count), (unsigned)A.a.heads);
        attn_simt_grad_q_kernel<T, DP><<<grid, kThreads, qb, s>>>(A, partial);
        st = check_launch("attn_simt_grad_q_kernel");
        if (st != kOk) return st;
    }
    if (A.a.k_tile_count) {
        const KeyShares K = key_shares(A);
        const dim3 grid((unsigned)(2 * key_blocks(A, K)), (unsigned)A.a.kv_heads);
        attn_simt_grad_kv_kernel<T, DP><<<grid, kThreads, kb, s>>>(A, K, sums);
        st = check_launch("attn_simt_grad_kv_kernel");
        if (st == kOk && K.shares > 1) st = join_shares<T>(A, K, sums, s);
    }
    return st;
}
int by_dim(const AttnArgs& A, bool backward, cudaStream_t s) {
    if (A.a.dim <= 16) return backward ? run_bwd<float, 16>(A, s) : run_fwd<float, 16>(A, s);
    if (A.a.dim <= 32) return backward ? run_bwd<float, 32>(A, s) : run_fwd<float, 32>(A, s);
    if (A.a.dim <= 64) return backward ? run_bwd<float, 64>(A, s) : run_fwd<float, 64>(A, s);
    return backward ? run_bwd<float, 128>(A, s) : run_fwd<float, 128>(A, s);
}

}  // namespace

int attn_simt_forward(const AttnArgs& A, cudaStream_t s) { return by_dim(A, false, s); }
int attn_simt_backward(const AttnArgs& A, cudaStream_t s) { return by_dim(A, true, s); }

}  // namespace mpo
