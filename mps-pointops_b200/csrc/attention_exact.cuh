// One row of the attention at a time, by one warp: the visible pairs and no
// others, in the order of the definition.
//
// The tile kernels multiply whole tiles, in which an invisible pair counts as
// a weight of 0; a NaN or an infinity among values that a row may not see then
// turns its 0 into a NaN.  A tile kernel therefore sends each result row that
// holds a NaN through these functions after it has stored it: the row comes out
// with the contributions of its visible pairs alone.  No cost where no NaN is.
// (The backward sends infinities too: a score gradient may leave float16's range
// although its products with the rows do not.)
#pragma once

#include "attention_common.cuh"

namespace mpo {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

// Four elements of a row per lane: d = lane + 32 i (zero past dim).
template <typename T>
__device__ __forceinline__ void lane_row(const T* p, int dim, float (&x)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lane + 32 * i < dim ? Elem<T>::to(p[lane + 32 * i]) : 0.f;
}
__device__ __forceinline__ float lane_dot(const float (&a)[4], const float (&b)[4]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fmaf(a[i], b[i], s);
    return warp_sum(s);
}
// Bucket and bias (units of log2) of (query row, key row), global.
__device__ __forceinline__ int pair_bucket(const AttnArgs& A, int64_t q, int64_t k, int ax) {
    const int b = bias_bucket(A.a.kpos[k * A.a.axes + ax], A.a.qpos[q * A.a.axes + ax], A.a.reach, nullptr);
    return A.a.map ? min(max(A.a.map[b], 0), A.a.buckets - 1) : b;
}
__device__ __forceinline__ float pair_bias(const AttnArgs& A, int64_t q, int64_t k, int h) {
    if (!A.a.table) return 0.f;
    float s = 0.f;
    for (int ax = 0; ax < A.a.axes; ++ax)
        s += table_entry(A.a, ax * A.a.buckets + pair_bucket(A, q, k, ax), h) * kLog2e;
    return s;
}
// Key ranges of one query at p: [0, s1) and [lo, hi) with s1 <= lo.
__device__ __forceinline__ void row_keys(const AttnArgs& A, int p, int lk, int& s1, int& lo, int& hi) {
    hi = max(0, min(lk, p + A.right + 1));
    lo = min(max(0, p - A.left), hi);
    s1 = min(A.a.sinks, lk);
    if (A.a.causal) s1 = max(0, min(s1, p + 1));
    if (s1 >= lo) {  // one run
        lo = 0;
        hi = max(hi, s1);
        s1 = 0;
    } else if (lo >= hi) {
        lo = hi = s1;
    }
}

// out and lse of query row q (global) at position p, head h.
template <typename T>
__device__ __noinline__ void exact_forward_row(const AttnArgs& A, int64_t q, int p, int64_t k0,
                                               int lk, int h) {
    const int lane = threadIdx.x & 31, hk = h / A.group;
    float x[4], y[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
    float m = -INFINITY, l = 0.f;
    int s1, lo, hi;
    row_keys(A, p, lk, s1, lo, hi);
    for (int j = 0; j < hi; ++j) {
        if (j == s1) j = lo;
        if (j >= hi) break;
        lane_row(attn_row<T>(A.a.k, k0 + j, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k0 + j, h));
        lane_row(attn_row<T>(A.a.v, k0 + j, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_sfu(m - ref), w = exp2_sfu(s - ref);
        m = mn;
        l = fmaf(l, f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, y[i], __fmul_rn(acc[i], f));
    }
    const float r = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = (q * A.a.heads + h) * A.a.dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 32 * i;
        if (d >= A.a.dim) continue;
        const float o = l == 0.f ? 0.f : acc[i] * r;
        static_cast<T*>(A.a.out)[at + d] = Elem<T>::from(o);
    }
    if (A.a.lse && lane == 0)
        A.a.lse[(int64_t)h * A.a.q_rows + q] = l == 0.f ? -INFINITY : fmaf(m, kLn2, logf(l));
}

__device__ __forceinline__ float load_lse2(const AttnArgs& A, int64_t q, int h) {
    const float l = A.a.lse[(int64_t)h * A.a.q_rows + q];
    return l == -INFINITY ? INFINITY : l * kLog2e;
}

// D of query row q as sum P dP.
template <typename T>
__device__ __noinline__ float exact_delta_row(const AttnArgs& A, int64_t q, int p, int64_t k0, int lk,
                                              int h) {
    float x[4], g[4], y[4], sum = 0.f;
    lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
    lane_row(static_cast<const T*>(A.a.grad_out) + (q * A.a.heads + h) * A.a.dim, A.a.dim, g);
    const float lse2 = load_lse2(A, q, h);
    const int hk = h / A.group;
    int s1, lo, hi;
    row_keys(A, p, lk, s1, lo, hi);
    for (int j = 0; j < hi; ++j) {
        if (j == s1) j = lo;
        if (j >= hi) break;
        lane_row(attn_row<T>(A.a.v, k0 + j, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float dp = lane_dot(g, y);
        lane_row(attn_row<T>(A.a.k, k0 + j, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k0 + j, h));
        sum = fmaf(exp2_sfu(s - lse2), dp, sum);
    }
    return sum;
}

// grad_q row; `cells` (nullable): this warp's table cells ([entry][32]), to which
// lane 0 adds the row's score gradients.
template <typename T>
__device__ __noinline__ void exact_grad_q_row(const AttnArgs& A, int64_t q, int p, int64_t k0,
                                              int lk, int h, float* cells = nullptr) {
    const int lane = threadIdx.x & 31, hk = h / A.group;
    float x[4], g[4], y[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
    const int64_t at = (q * A.a.heads + h) * A.a.dim;
    lane_row(static_cast<const T*>(A.a.grad_out) + at, A.a.dim, g);
    const float lse2 = load_lse2(A, q, h), delta = A.a.delta[(int64_t)h * A.a.q_rows + q];
    int s1, lo, hi;
    row_keys(A, p, lk, s1, lo, hi);
    for (int j = 0; j < hi; ++j) {
        if (j == s1) j = lo;
        if (j >= hi) break;
        lane_row(attn_row<T>(A.a.v, k0 + j, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float dp = lane_dot(g, y);
        lane_row(attn_row<T>(A.a.k, k0 + j, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k0 + j, h));
        const float ds = exp2_sfu(s - lse2) * (dp - delta);
        if (cells && lane == 0)
            for (int ax = 0; ax < A.a.axes; ++ax)
                cells[(ax * A.a.buckets + pair_bucket(A, q, k0 + j, ax)) * 32] += ds;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(ds, y[i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < A.a.dim)
            static_cast<T*>(A.a.grad_q)[at + lane + 32 * i] = Elem<T>::from(acc[i] * A.a.scale);
}

// grad_k and grad_v rows of key j of a cloud, key head hk.
template <typename T>
__device__ __noinline__ void exact_grad_kv_row(const AttnArgs& A, int64_t k0, int j, int64_t q0,
                                               int lq, int lk, int hk) {
    const int lane = threadIdx.x & 31;
    float kx[4], vx[4], x[4], g[4];
    float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.k, k0 + j, hk, A.a.k_row, A.a.k_head), A.a.dim, kx);
    lane_row(attn_row<T>(A.a.v, k0 + j, hk, A.a.v_row, A.a.v_head), A.a.dim, vx);
    int lo, hi;
    query_span(A, j, j, lq, lk, lo, hi);
    for (int h = hk * A.group; h < (hk + 1) * A.group; ++h)
        for (int i = lo; i < hi; ++i) {
            if (!attn_visible(A, i + lk - lq, j)) continue;
            lane_row(attn_row<T>(A.a.q, q0 + i, h, A.a.q_row, A.a.q_head), A.a.dim, x);
            lane_row(static_cast<const T*>(A.a.grad_out) + ((q0 + i) * A.a.heads + h) * A.a.dim,
                     A.a.dim, g);
            const float s = fmaf(lane_dot(x, kx), A.scale_log2, pair_bias(A, q0 + i, k0 + j, h));
            const float w = exp2_sfu(s - load_lse2(A, q0 + i, h));
            const float ds = w * (lane_dot(g, vx) - A.a.delta[(int64_t)h * A.a.q_rows + q0 + i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dv[e] = fmaf(w, g[e], dv[e]);
                dk[e] = fmaf(ds, x[e], dk[e]);
            }
        }
    const int64_t at = ((k0 + j) * A.a.kv_heads + hk) * A.a.dim;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d = lane + 32 * e;
        if (d >= A.a.dim) continue;
        static_cast<T*>(A.a.grad_k)[at + d] = Elem<T>::from(dk[e] * A.a.scale);
        static_cast<T*>(A.a.grad_v)[at + d] = Elem<T>::from(dv[e]);
    }
}

}  // namespace
}  // namespace mpo
