// Attention of few query rows per cloud (single new rows, short chunks) over
// many keys (definitions: attention_common.cuh).
//
// Bound by HBM: each visible key and value is read once per key head, so the
// query heads that share a key head, and up to 16 / group query rows of a
// cloud, sit together as the 16 rows of one product.  16-bit types: a warp takes
// 16 keys at a time as operands of mma.sync m16n8k16, loaded straight from
// global memory in 16-byte pieces.  The sum over a head's elements may run in
// any order, so lane t of a quad loads elements 8 t .. 8 t + 7 of each 32 and
// calls them the four k-slots it owns in two products; the columns of the
// second product may stand for any elements, so lane group g loads elements
// 8 g .. of a value row.  tcgen05 would need the 16 rows padded to 128 and its
// operands in shared memory; at a quarter of an instruction per byte the plain
// tensor instruction leaves the loads as the only limit.  float32: a key per
// group of lanes, multiply-adds.
//
// The keys are split over the blocks of grid.z, then over a block's four warps,
// so that few rows fill the GPU; a second kernel joins the splits' rows by
// their maxima and sums, in split order.  64 streams over up to 8192 cached keys of
// 8 heads of 128: 288 us, 5.6 TB/s, 86 % of a plain copy.  32 streams over 2047 keys of
// 8 heads of 64 with a table, one row of a product's 16 in use: 49 us, 2.2 TB/s; the
// chain from a key's position over its buckets to its weight binds, not the loads.
#include <string>

#include "attention_exact.cuh"

namespace mpo {
namespace {

constexpr int kRowsThreads = 128, kRowsWarps = 4;

// Which query rows, heads and keys a block works on.
struct Unit {
    AttnTile t;
    int row0, rows;   // query rows [row0, row0 + rows) of the tile
    int hk, h0, gc;   // key head; first query head and count of heads per query row
    int s1, lo, hi;   // keys [0, s1) and [lo, hi)
    int c0, c1;       // this split's share of the s1 + hi - lo keys
    __device__ __forceinline__ int key(int c) const { return c < s1 ? c : lo + (c - s1); }
};
__device__ __forceinline__ bool rows_unit(const AttnArgs& A, int per, int units, int heads_per,
                                          int splits, Unit& U) {
    U.t = reinterpret_cast<const AttnTile*>(A.a.q_tiles)[blockIdx.x / units];
    U.row0 = (int)(blockIdx.x % units) * per;
    U.rows = min(per, U.t.rows - U.row0);
    if (U.rows <= 0) return false;
    const int groups = (A.group + heads_per - 1) / heads_per;
    U.hk = blockIdx.y / groups;
    const int g0 = (int)(blockIdx.y % groups) * heads_per;
    U.h0 = U.hk * A.group + g0;
    U.gc = min(heads_per, A.group - g0);
    const int p0 = U.t.first + U.row0, p1 = p0 + U.rows - 1;
    U.hi = max(0, min(U.t.lk, p1 + A.right + 1));
    U.lo = min(max(0, p0 - A.left), U.hi);
    U.s1 = min(A.a.sinks, U.t.lk);
    if (A.a.causal) U.s1 = max(0, min(U.s1, p1 + 1));
    if (U.s1 >= U.lo) {
        U.lo = 0;
        U.hi = max(U.hi, U.s1);
        U.s1 = 0;
    }
    const int64_t n = U.s1 + U.hi - U.lo;
    U.c0 = (int)(n * blockIdx.z / splits);
    U.c1 = (int)(n * (blockIdx.z + 1) / splits);
    return true;
}

// One row's result of a split: maximum (log2 units), sum and unnormalised row.
struct Partial {
    float* base;
    int64_t stride;  // floats of one row
    __device__ __forceinline__ float* at(const AttnArgs& A, int64_t q, int h, int z) const {
        return base + (((int64_t)z * A.a.q_rows + q) * A.a.heads + h) * stride;
    }
};
__host__ __device__ __forceinline__ int64_t partial_stride(int dim) { return dim + 4; }

// Final row: o / l, its log-sum-exp; `nan` rows are formed again pair by pair.
template <typename T>
__device__ __forceinline__ void store_row(const AttnArgs& A, int64_t q, int h, int d, float o, float l,
                                          bool& nan) {
    const float v = l == 0.f ? (isnan(o) ? o : 0.f) : o / l;
    nan |= isnan(v);
    const int64_t at = (q * A.a.heads + h) * A.a.dim + d;
    static_cast<T*>(A.a.out)[at] = Elem<T>::from(v);
}
__device__ __forceinline__ void store_lse(const AttnArgs& A, int64_t q, int h, float m, float l) {
    if (A.a.lse) A.a.lse[(int64_t)h * A.a.q_rows + q] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
}

// A block's rows in shared memory, one slot per warp: [warp][row][maximum, sum,
// 2 unused, dim]; joined by all threads into the result or the split's partial.
template <typename T>
__device__ __forceinline__ void join_warps(const AttnArgs& A, const Unit& U, const float* sh, int pitch,
                                           int slots, int rows, int splits, float* partial) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < rows; r += kRowsWarps) {
        const int64_t q = (int64_t)U.t.row + U.row0 + r / U.gc;
        const int h = U.h0 + r % U.gc;
        float m = -INFINITY;
        for (int w = 0; w < slots; ++w) m = fmaxf(m, sh[(w * 16 + r) * pitch]);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        for (int w = 0; w < slots; ++w)
            l = fmaf(sh[(w * 16 + r) * pitch + 1], exp2_sfu(sh[(w * 16 + r) * pitch] - ref), l);
        float* dst = splits > 1 ? Partial{partial, partial_stride(A.a.dim)}.at(A, q, h, blockIdx.z)
                                : nullptr;
        bool nan = false;
        for (int d = lane; d < A.a.dim; d += 32) {
            float o = 0.f;
            for (int w = 0; w < slots; ++w)
                o = fmaf(sh[(w * 16 + r) * pitch + 4 + d], exp2_sfu(sh[(w * 16 + r) * pitch] - ref), o);
            if (dst) dst[4 + d] = o;
            else store_row<T>(A, q, h, d, o, l, nan);
        }
        if (lane == 0) {
            if (dst) {
                dst[0] = m;
                dst[1] = l;
            } else {
                store_lse(A, q, h, m, l);
            }
        }
        if (__any_sync(FULL_MASK, nan)) {
            __syncwarp();
            exact_forward_row<T>(A, q, U.t.first + U.row0 + r / U.gc, U.t.other, U.t.lk, h);
        }
    }
}

// ---------------------------------------------------------------- 16-bit types
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void* p, bool on) {
    return on ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint32_t low_pair(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_pair(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// DP: 32, 64 or 128 elements (the head size rounded up; what lies past it is not read).
template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(kRowsThreads, DP == 128 ? 2 : 4)
attn_rows_kernel(const __grid_constant__ AttnArgs A, int per, int units, int splits, float* partial) {
    constexpr int NB = DP / 32;                 // 32-element blocks of a dot product
    constexpr int NV = DP / 64 < 1 ? 1 : DP / 64;  // value blocks of 8 (lane groups) x 8 elements
    constexpr int kPitch = DP + 4;
    // The warps' rows at the end; before that the heads' tables ([entry][head], times log2 e)
    // and each warp's bias of 16 rows x 16 keys.
    constexpr int kJoin = kRowsWarps * 16 * kPitch, kBiasWords = kAttnMaxEntries * 16 + kRowsWarps * 256;
    __shared__ float sh[BIAS && kBiasWords > kJoin ? kBiasWords : kJoin];
    Unit U;
    if (!rows_unit(A, per, units, 16, splits, U)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rows = U.rows * U.gc;             // of the 16
    float* tile = sh + (BIAS ? kAttnMaxEntries * 16 + warp * 256 : 0);
    // Bias: lane l forms that of key l % 16 and rows l / 16, l / 16 + 2, ..
    const int kl = lane & 15;
    int kp[kAttnMaxAxes] = {0, 0, 0};
    if (BIAS) {
        for (int e = threadIdx.x; e < A.a.axes * A.a.buckets * U.gc; e += kRowsThreads)
            sh[e / U.gc * 16 + e % U.gc] = table_entry(A.a, e / U.gc, U.h0 + e % U.gc) * kLog2e;
        __syncthreads();
    }
    auto load_key_pos = [&](int c) {
        if (!BIAS || c + kl >= U.c1) return;
        const int64_t k = (int64_t)U.t.other + U.key(c + kl);
#pragma unroll
        for (int a = 0; a < kAttnMaxAxes; ++a)
            if (a < A.a.axes) kp[a] = A.a.kpos[k * A.a.axes + a];
    };
    auto form_bias = [&]() {  // of the keys whose positions are at hand
        if (!BIAS) return;
        __syncwarp();
        int i_old = -1, bucket[kAttnMaxAxes] = {0, 0, 0};
        for (int r = lane >> 4; r < rows; r += 2) {
            const int i = r / U.gc, hh = r - i * U.gc;
            if (i != i_old) {  // the heads of a query row share its buckets
                i_old = i;
                const int64_t q = (int64_t)U.t.row + U.row0 + i;
#pragma unroll
                for (int a = 0; a < kAttnMaxAxes; ++a)
                    if (a < A.a.axes) {
                        int b = bias_bucket(kp[a], A.a.qpos[q * A.a.axes + a], A.a.reach, nullptr);
                        if (A.a.map) b = min(max(__ldg(A.a.map + b), 0), A.a.buckets - 1);
                        bucket[a] = (a * A.a.buckets + b) * 16;
                    }
            }
            float x = 0.f;
#pragma unroll
            for (int a = 0; a < kAttnMaxAxes; ++a)
                if (a < A.a.axes) x += sh[bucket[a] + hh];
            tile[r * 16 + kl] = x;
        }
        __syncwarp();
    };
    // Queries: rows g and g + 8.
    uint32_t qf[2 * NB][4];
    int pos[2], head[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = g + 8 * half;
        const bool on = r < rows;
        const int i = on ? r / U.gc : 0;
        pos[half] = U.t.first + U.row0 + i;
        head[half] = U.h0 + (on ? r % U.gc : 0);
        const int64_t q = (int64_t)U.t.row + U.row0 + i;
        const T* src = attn_row<T>(A.a.q, q, head[half], A.a.q_row, A.a.q_head);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int d = 32 * b + 8 * t;
            const uint4 u = load16(src + d, on && d < A.a.dim);
            qf[2 * b][half] = u.x;
            qf[2 * b][half + 2] = u.y;
            qf[2 * b + 1][half] = u.z;
            qf[2 * b + 1][half + 2] = u.w;
        }
        if (!on) head[half] = -1;
    }
    float o[8 * NV][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 8 * NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    const T* kbase = attn_row<T>(A.a.k, U.t.other, U.hk, A.a.k_row, A.a.k_head);
    const T* vbase = attn_row<T>(A.a.v, U.t.other, U.hk, A.a.v_row, A.a.v_head);
    constexpr int kStep = 16 * kRowsWarps;
    uint4 kf[2][NB];
    auto load_keys = [&](int c) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int cc = c + g + 8 * half;
            const T* src = kbase + (int64_t)U.key(min(cc, U.c1 - 1)) * A.a.k_row + 8 * t;
#pragma unroll
            for (int b = 0; b < NB; ++b)
                kf[half][b] = load16(src + 32 * b, cc < U.c1 && 32 * b + 8 * t < A.a.dim);
        }
    };
    // Values of keys 2t, 2t + 1, 2t + 8, 2t + 9: a step ahead for narrow heads, where there are
    // registers and fewer bytes in flight (53 -> 47 us for 32 streams of 2047 keys, D = 64; at D =
    // 128 the same costs 287 -> 338 us for 64 streams of 8192).
    constexpr bool kValuesAhead = DP <= 64;
    uint4 vf[4][NV];
    auto load_values = [&](int c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int cc = c + 2 * t + (e & 1) + 8 * (e >> 1);
            const T* src = vbase + (int64_t)U.key(min(cc, U.c1 - 1)) * A.a.v_row + 8 * g;
#pragma unroll
            for (int b = 0; b < NV; ++b)
                vf[e][b] = load16(src + 64 * b, cc < U.c1 && 64 * b + 8 * g < A.a.dim);
        }
    };
    int c = U.c0 + 16 * warp;
    if (c < U.c1) {
        load_keys(c);
        if (kValuesAhead) load_values(c);
        load_key_pos(c);
    }
    for (; c < U.c1; c += kStep) {
        form_bias();
        load_key_pos(c + kStep);
        if (!kValuesAhead) load_values(c);
        float s[2][4];  // keys 2t, 2t + 1 of the half: rows g (0, 1) and g + 8 (2, 3)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[half][e] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                mma16816<T>(s[half], qf[2 * b], kf[half][b].x, kf[half][b].y);
                mma16816<T>(s[half], qf[2 * b + 1], kf[half][b].z, kf[half][b].w);
            }
        }
        if (c + kStep < U.c1) load_keys(c + kStep);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = e >> 1, cc = c + 8 * half + 2 * t + (e & 1);
                const int j = U.key(cc);
                float x = -INFINITY;
                if (head[row] >= 0 && cc < U.c1 && attn_visible(A, pos[row], j)) {
                    x = s[half][e] * A.scale_log2;
                    if (BIAS) x += tile[(g + 8 * row) * 16 + 8 * half + 2 * t + (e & 1)];
                }
                s[half][e] = x;
            }
        float f[2];
#pragma unroll
        for (int row = 0; row < 2; ++row) {
            float top = fmaxf(fmaxf(s[0][2 * row], s[0][2 * row + 1]), fmaxf(s[1][2 * row], s[1][2 * row + 1]));
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 1));
            top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 2));
            const float mn = fmaxf(m[row], top), ref = mn == -INFINITY ? 0.f : mn;
            f[row] = exp2_sfu(m[row] - ref);
            const bool same = mn == m[row];
            m[row] = mn;
            float sum = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[half][2 * row + e] = exp2_sfu(s[half][2 * row + e] - ref);
                    sum += s[half][2 * row + e];
                }
            if (same) f[row] = 1.f;
            l[row] = fmaf(l[row], f[row], sum);  // this lane's keys; joined at the end
        }
        if (__any_sync(FULL_MASK, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < 8 * NV; ++j) {
                o[j][0] *= f[0];
                o[j][1] *= f[0];
                o[j][2] *= f[1];
                o[j][3] *= f[1];
            }
        }
        const uint32_t pf[4] = {Elem<T>::two(s[0][0], s[0][1]), Elem<T>::two(s[0][2], s[0][3]),
                                Elem<T>::two(s[1][0], s[1][1]), Elem<T>::two(s[1][2], s[1][3])};
#pragma unroll
        for (int b = 0; b < NV; ++b) {
            const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0][b]);
            const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1][b]);
            const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2][b]);
            const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3][b]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                mma16816<T>(o[8 * b + 2 * w], pf, low_pair(v0[w], v1[w]), low_pair(v2[w], v3[w]));
                mma16816<T>(o[8 * b + 2 * w + 1], pf, high_pair(v0[w], v1[w]), high_pair(v2[w], v3[w]));
            }
        }
        if (kValuesAhead && c + kStep < U.c1) load_values(c + kStep);
    }
    if (BIAS) __syncthreads();  // the tables and tiles have been read
    // Column n of product j of block b is element 64 b + 8 n + j.
#pragma unroll
    for (int row = 0; row < 2; ++row) {
        float sum = l[row];
        sum += __shfl_xor_sync(FULL_MASK, sum, 1);
        sum += __shfl_xor_sync(FULL_MASK, sum, 2);
        float* dst = sh + (warp * 16 + g + 8 * row) * kPitch;
        if (t == 0) {
            dst[0] = m[row];
            dst[1] = sum;
        }
#pragma unroll
        for (int j = 0; j < 8 * NV; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = 64 * (j / 8) + 8 * (2 * t + e) + j % 8;
                if (d < DP) dst[4 + d] = o[j][2 * row + e];
            }
    }
    __syncthreads();
    join_warps<T>(A, U, sh, kPitch, kRowsWarps, rows, splits, partial);
}

// ---------------------------------------------------------------- float32
// One query row and head per block; DP / 4 lanes hold a key's elements, four keys
// per lane group in flight.
template <int DP>
__global__ void __launch_bounds__(kRowsThreads)
attn_rows_f32_kernel(const __grid_constant__ AttnArgs A, int units, int splits, float* partial) {
    constexpr int LK = DP / 4, KW = 32 / LK, kPitch = DP + 4, kFly = 4;
    __shared__ float sh[kRowsWarps * 16 * kPitch];
    Unit U;
    if (!rows_unit(A, 1, units, 1, splits, U)) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e4 = (lane % LK) * 4, sub = lane / LK;
    const int64_t q = (int64_t)U.t.row + U.row0;
    const int p = U.t.first + U.row0, h = U.h0;
    const bool on = e4 < A.a.dim;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 x = on ? *reinterpret_cast<const float4*>(attn_row<float>(A.a.q, q, h, A.a.q_row, A.a.q_head) + e4)
                        : zero;
    const float* kbase = attn_row<float>(A.a.k, U.t.other, U.hk, A.a.k_row, A.a.k_head) + e4;
    const float* vbase = attn_row<float>(A.a.v, U.t.other, U.hk, A.a.v_row, A.a.v_head) + e4;
    float4 o = zero;
    float m = -INFINITY, l = 0.f;
    constexpr int kBatch = KW * kFly;
    for (int c = U.c0 + warp * kBatch; c < U.c1; c += kRowsWarps * kBatch) {
        float4 k[kFly], v[kFly];
        int j[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            const int cc = c + i * KW + sub;
            j[i] = U.key(min(cc, U.c1 - 1));
            const bool take = on && cc < U.c1;
            k[i] = take ? *reinterpret_cast<const float4*>(kbase + (int64_t)j[i] * A.a.k_row) : zero;
            v[i] = take ? *reinterpret_cast<const float4*>(vbase + (int64_t)j[i] * A.a.v_row) : zero;
        }
        float s[kFly], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            s[i] = fmaf(x.x, k[i].x, fmaf(x.y, k[i].y, fmaf(x.z, k[i].z, __fmul_rn(x.w, k[i].w))));
#pragma unroll
            for (int w = LK >> 1; w; w >>= 1) s[i] += __shfl_xor_sync(FULL_MASK, s[i], w);
            const bool seen = c + i * KW + sub < U.c1 && attn_visible(A, p, j[i]);
            s[i] = seen ? fmaf(s[i], A.scale_log2, pair_bias(A, q, (int64_t)U.t.other + j[i], h)) : -INFINITY;
            top = fmaxf(top, s[i]);
        }
        const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_sfu(m - ref);
        m = mn;
        l *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            const float w = exp2_sfu(s[i] - ref);
            l += w;
            o.x = fmaf(w, v[i].x, o.x);
            o.y = fmaf(w, v[i].y, o.y);
            o.z = fmaf(w, v[i].z, o.z);
            o.w = fmaf(w, v[i].w, o.w);
        }
    }
    // The warp's key groups, then (join_warps) the warps.
#pragma unroll
    for (int w = LK; w < 32; w <<= 1) {
        const float om = __shfl_xor_sync(FULL_MASK, m, w), mn = fmaxf(m, om);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_sfu(m - ref), of = exp2_sfu(om - ref);
        m = mn;
        l = fmaf(l, f, __fmul_rn(__shfl_xor_sync(FULL_MASK, l, w), of));
        o.x = fmaf(o.x, f, __fmul_rn(__shfl_xor_sync(FULL_MASK, o.x, w), of));
        o.y = fmaf(o.y, f, __fmul_rn(__shfl_xor_sync(FULL_MASK, o.y, w), of));
        o.z = fmaf(o.z, f, __fmul_rn(__shfl_xor_sync(FULL_MASK, o.z, w), of));
        o.w = fmaf(o.w, f, __fmul_rn(__shfl_xor_sync(FULL_MASK, o.w, w), of));
    }
    float* dst = sh + warp * 16 * kPitch;
    if (sub == 0) {
        if (lane == 0) {
            dst[0] = m;
            dst[1] = l;
        }
        *reinterpret_cast<float4*>(dst + 4 + e4) = o;
    }
    __syncthreads();
    join_warps<float>(A, U, sh, kPitch, kRowsWarps, 1, splits, partial);
}

// ---------------------------------------------------------------- join
// A warp per (query row, head): the splits' rows by their maxima and sums.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads, 4)
attn_rows_join_kernel(const __grid_constant__ AttnArgs A, int splits, const float* __restrict__ partial) {
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.q_tiles)[blockIdx.x];
    const int lane = threadIdx.x & 31, h = blockIdx.y * kRowsWarps + (threadIdx.x >> 5);
    if (h >= A.a.heads) return;
    const int64_t stride = partial_stride(A.a.dim), step = (int64_t)A.a.q_rows * A.a.heads * stride;
    for (int r = blockIdx.z; r < t.rows; r += gridDim.z) {
        const int64_t q = (int64_t)t.row + r;
        const float* src = partial + (q * A.a.heads + h) * stride;
        float m = -INFINITY;
        for (int z = lane; z < splits; z += 32) m = fmaxf(m, src[z * step]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < splits; ++z) {
            const float* s = src + z * step;
            const float w = exp2_sfu(s[0] - ref);
            l = fmaf(w, s[1], l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + 32 * i < A.a.dim) o[i] = fmaf(w, s[4 + lane + 32 * i], o[i]);
        }
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < A.a.dim) store_row<T>(A, q, h, lane + 32 * i, o[i], l, nan);
        if (lane == 0) store_lse(A, q, h, m, l);
        if (__any_sync(FULL_MASK, nan)) {
            __syncwarp();
            exact_forward_row<T>(A, q, t.first + r, t.other, t.lk, h);
        }
    }
}

// ---------------------------------------------------------------- launches
struct RowsPlan {
    int heads_per, per, units, splits;
};
RowsPlan rows_plan(const AttnArgs& A) {
    RowsPlan P;
    P.heads_per = A.a.dtype == MPO_F32 ? 1 : 16;
    const int gc = A.group < P.heads_per ? A.group : P.heads_per;
    P.per = A.a.dtype == MPO_F32 ? 1 : 16 / gc;
    P.units = (int)ceil_div(min64(A.a.max_rows, kAttnTile), P.per);
    const int64_t blocks = A.a.q_tile_count * P.units * A.a.kv_heads * ceil_div(A.group, P.heads_per);
    const int64_t span = min64(A.a.max_keys, (int64_t)A.left + A.right + 1 + A.a.sinks + P.per);
    // Twelve blocks per SM (several rounds of what is resident) even out clouds of
    // different lengths; a split keeps at least 512 keys, eight steps of its warps,
    // beside which its start and its join are short.
    P.splits = (int)max64(1, min64(min64(ceil_div(12 * sm_count(), max64(blocks, 1)), span / 512), 64));
    return P;
}

template <typename T, int DP>
int run16(const AttnArgs& A, const RowsPlan& P, dim3 grid, float* partial, cudaStream_t s) {
    if (A.a.table)
        attn_rows_kernel<T, DP, true><<<grid, kRowsThreads, 0, s>>>(A, P.per, P.units, P.splits, partial);
    else
        attn_rows_kernel<T, DP, false><<<grid, kRowsThreads, 0, s>>>(A, P.per, P.units, P.splits, partial);
    return check_launch("attn_rows_kernel");
}
template <int DP>
int run32(const AttnArgs& A, const RowsPlan& P, dim3 grid, float* partial, cudaStream_t s) {
    attn_rows_f32_kernel<DP><<<grid, kRowsThreads, 0, s>>>(A, P.units, P.splits, partial);
    return check_launch("attn_rows_f32_kernel");
}
template <typename T>
int run(const AttnArgs& A, cudaStream_t s) {
    const RowsPlan P = rows_plan(A);
    float* partial = static_cast<float*>(A.a.workspace);
    const dim3 grid((unsigned)(A.a.q_tile_count * P.units),
                    (unsigned)(A.a.kv_heads * ceil_div(A.group, P.heads_per)), (unsigned)P.splits);
    int st;
    if constexpr (std::is_same<T, float>::value) {
        st = A.a.dim <= 16   ? run32<16>(A, P, grid, partial, s)
             : A.a.dim <= 32 ? run32<32>(A, P, grid, partial, s)
             : A.a.dim <= 64 ? run32<64>(A, P, grid, partial, s)
                             : run32<128>(A, P, grid, partial, s);
    } else {
        st = A.a.dim <= 32   ? run16<T, 32>(A, P, grid, partial, s)
             : A.a.dim <= 64 ? run16<T, 64>(A, P, grid, partial, s)
                             : run16<T, 128>(A, P, grid, partial, s);
    }
    if (st != kOk || P.splits == 1) return st;
    const dim3 join((unsigned)A.a.q_tile_count, (unsigned)ceil_div(A.a.heads, kRowsWarps),
                    (unsigned)min64(A.a.max_rows, kAttnTile));
    attn_rows_join_kernel<T><<<join, kRowsThreads, 0, s>>>(A, P.splits, partial);
    return check_launch("attn_rows_join_kernel");
}

}  // namespace

// At most 16 rows of queries and shared heads per key head and cloud: then a
// key is read by one unit (by group / 16 where more heads share it), where a
// tile kernel would fill 1/8 of its rows or less.  Beyond, this kernel reads the
// keys again for every 16 rows, and the tile kernels read them once but by one
// block per 128 rows and head, so they gain with many rows and many clouds only.
// Kernel times in us over 8192 keys per cloud, this kernel | tile kernel:
//   bf16, 32 heads of 128 over 8   5 rows   16       32        128
//     1 cloud                      21 | 94  34 | 94  59 | 94   164 | 94
//     8 clouds                    118 | 152 194 | 154 299 | 155 975 | 157
//     64 clouds                   581 | 1144 1041 | 1154 1978 | 1183
//   bf16, 8 heads of 64           17 rows   32       64        128
//     1 cloud                      20 | 110 21 | 110 26 | 110  39 | 111
//     8 clouds                     79 | 109 86 | 109 139 | 109 227 | 109
//     64 clouds                   423 | 254 450 | 254 805 | 255
//   float32, 8 heads of 64
//     1 cloud                      85 | 866 151 | 867 267 | 714 520 | 715
//     8 clouds                    619 | 1074 1182 | 1074 2290 | 927
// The limit is right for many clouds without shared heads; with few clouds, or a few
// rows of shared heads, a limit by the count of blocks would gain up to 5 times.
bool attn_rows_eligible(const AttnArgs& A) {
    return (int64_t)A.a.max_rows * min64(A.group, 16) <= 16;
}
size_t attn_rows_workspace(const AttnArgs& A) {
    const RowsPlan P = rows_plan(A);
    if (P.splits == 1) return 0;
    return (size_t)P.splits * A.a.q_rows * A.a.heads * partial_stride(A.a.dim) * sizeof(float);
}
int attn_rows_forward(const AttnArgs& A, cudaStream_t s) {
    if (A.a.dtype == MPO_F32) return run<float>(A, s);
    return A.a.dtype == MPO_F16 ? run<__half>(A, s) : run<__nv_bfloat16>(A, s);
}

}  // namespace mpo
