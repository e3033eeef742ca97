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
//
// Rows whose own pairs hold such values come here as well, all of them after an
// overflow in the loss.  A row ends as soon as each of its elements in question
// has become a NaN, which nothing can change.  Backward of a cloud of 4096 points, 4
// heads of 64, window 512, bf16 (0.35 ms), with a gradient that is NaN throughout:
// 20 -> 0.23 ms; infinities of both signs: 20 -> 0.31 ms; of one sign, or one in each
// row (no NaN ends dv's sums): 20 -> 5.5 ms; one row with a NaN: 10.7 -> 5.4 ms.  Loading
// several pairs at a time gained nothing (4.1 against 4.2 to 4.4 ms) and cost the tile
// kernels registers.
#pragma once

#include "attention_common.cuh"

namespace mpo {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

// Four elements of a row per lane, d = 4 lane + i, in one load (zero past dim, which is a
// multiple of eight; rows start on 16 bytes).
template <typename T>
__device__ __forceinline__ void lane_row(const T* p, int dim, float (&x)[4]) {
    const int d = 4 * (threadIdx.x & 31);
    x[0] = x[1] = x[2] = x[3] = 0.f;
    if (d >= dim) return;
    if constexpr (sizeof(T) == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p + d);
        Elem<T>::two(u.x, x);
        Elem<T>::two(u.y, x + 2);
    } else {
        Elem<T>::unpack(*reinterpret_cast<const uint4*>(p + d), x);
    }
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
// The keys that a query at p sees, [0, s1) and [lo, hi), by number.
struct RowKeys {
    int s1, lo, count;
    __device__ __forceinline__ RowKeys(const AttnArgs& A, int p, int lk) {
        int hi = max(0, min(lk, p + A.right + 1));
        lo = min(max(0, p - A.left), hi);
        s1 = min(A.a.sinks, lk);
        if (A.a.causal) s1 = max(0, min(s1, p + 1));
        if (s1 >= lo) {  // one run
            lo = 0;
            hi = max(hi, s1);
            s1 = 0;
        }
        count = s1 + hi - lo;
    }
    __device__ __forceinline__ int key(int c) const { return c < s1 ? c : lo + (c - s1); }
};
// The elements of a stored result row that are to be formed: all (`whole`), or those that
// are NaN and (`infinite`) infinite.  A finite one came from finite terms alone and is right.
template <typename T>
__device__ __forceinline__ unsigned row_needs(const T* stored, int dim, bool whole, bool infinite) {
    float x[4];
    lane_row(stored, dim, x);
    unsigned need = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (whole || isnan(x[i]) || (infinite && isinf(x[i]))) need |= 1u << i;
    return 4 * (int)(threadIdx.x & 31) < dim ? need : 0u;
}
// Every element in question is a NaN (warp-uniform).
__device__ __forceinline__ bool row_settled(unsigned need, const float (&x)[4]) {
    bool open = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) open |= ((need >> i) & 1u) && !isnan(x[i]);
    return !__any_sync(FULL_MASK, open);
}
// Stores a row, or (settled early) its NaN.
template <typename T>
__device__ __forceinline__ void store_formed(T* dst, int dim, bool settled, unsigned need, const float (&x)[4]) {
    const int d = 4 * (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d < dim && (!settled || ((need >> i) & 1u))) dst[d + i] = Elem<T>::from(x[i]);
}

// out and lse of query row q (global) at position p, head h.  `whole`: nothing of the
// stored row is right; else its lse and its finite elements are (scores are masked
// before their exponentials, so no invisible value reaches them).
template <typename T>
__device__ __noinline__ void exact_forward_row(const AttnArgs& A, int64_t q, int p, int64_t k0,
                                               int lk, int h, bool whole = false) {
    const int lane = threadIdx.x & 31, hk = h / A.group;
    T* out = static_cast<T*>(A.a.out) + (q * A.a.heads + h) * A.a.dim;
    const unsigned need = row_needs(out, A.a.dim, whole, false);
    float x[4], y[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
    float m = -INFINITY, l = 0.f;
    bool settled = false;
    const RowKeys keys(A, p, lk);
    for (int c = 0; c < keys.count && !settled; ++c) {
        const int64_t k = k0 + keys.key(c);
        lane_row(attn_row<T>(A.a.k, k, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k, h));
        lane_row(attn_row<T>(A.a.v, k, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_sfu(m - ref), w = exp2_sfu(s - ref);
        m = mn;
        l = fmaf(l, f, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(w, y[i], __fmul_rn(acc[i], f));
        settled = isnan(l) || (!whole && row_settled(need, acc));
    }
    const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = l == 0.f ? 0.f : acc[i] * r;
    store_formed(out, A.a.dim, settled, need, acc);
    if (A.a.lse && lane == 0 && (!settled || isnan(l)))
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
    const RowKeys keys(A, p, lk);
    for (int c = 0; c < keys.count && !isnan(sum); ++c) {
        const int64_t k = k0 + keys.key(c);
        lane_row(attn_row<T>(A.a.v, k, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float dp = lane_dot(g, y);
        lane_row(attn_row<T>(A.a.k, k, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k, h));
        sum = fmaf(exp2_sfu(s - lse2), dp, sum);
    }
    return sum;
}

// grad_q row (`whole`: nothing of the stored one is right); `cells` (nullable): this
// warp's table cells ([entry][32]), to which lane 0 adds the row's score gradients.
template <typename T>
__device__ __noinline__ void exact_grad_q_row(const AttnArgs& A, int64_t q, int p, int64_t k0,
                                              int lk, int h, bool whole = false, float* cells = nullptr) {
    const int lane = threadIdx.x & 31, hk = h / A.group;
    float x[4], g[4], y[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
    const int64_t at = (q * A.a.heads + h) * A.a.dim;
    lane_row(static_cast<const T*>(A.a.grad_out) + at, A.a.dim, g);
    const float lse2 = load_lse2(A, q, h), delta = A.a.delta[(int64_t)h * A.a.q_rows + q];
    T* dq = static_cast<T*>(A.a.grad_q) + at;
    const unsigned need = row_needs(dq, A.a.dim, whole, true);
    bool settled = false;
    const RowKeys keys(A, p, lk);
    for (int c = 0; c < keys.count && !settled; ++c) {
        const int64_t k = k0 + keys.key(c);
        lane_row(attn_row<T>(A.a.v, k, hk, A.a.v_row, A.a.v_head), A.a.dim, y);
        const float dp = lane_dot(g, y);
        lane_row(attn_row<T>(A.a.k, k, hk, A.a.k_row, A.a.k_head), A.a.dim, y);
        const float s = fmaf(lane_dot(x, y), A.scale_log2, pair_bias(A, q, k, h));
        const float ds = exp2_sfu(s - lse2) * (dp - delta);
        if (cells && lane == 0)
            for (int ax = 0; ax < A.a.axes; ++ax)
                cells[(ax * A.a.buckets + pair_bucket(A, q, k, ax)) * 32] += ds;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(ds, y[i], acc[i]);
        settled = !cells && row_settled(need, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= A.a.scale;
    store_formed(dq, A.a.dim, settled, need, acc);
}

// grad_k and grad_v rows of key j of a cloud, key head hk.
template <typename T>
__device__ __noinline__ void exact_grad_kv_row(const AttnArgs& A, int64_t k0, int j, int64_t q0,
                                               int lq, int lk, int hk) {
    float kx[4], vx[4], x[4], g[4];
    float dk[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
    lane_row(attn_row<T>(A.a.k, k0 + j, hk, A.a.k_row, A.a.k_head), A.a.dim, kx);
    lane_row(attn_row<T>(A.a.v, k0 + j, hk, A.a.v_row, A.a.v_head), A.a.dim, vx);
    const int64_t at = ((k0 + j) * A.a.kv_heads + hk) * A.a.dim;
    T *out_k = static_cast<T*>(A.a.grad_k) + at, *out_v = static_cast<T*>(A.a.grad_v) + at;
    const unsigned need_k = row_needs(out_k, A.a.dim, false, true),
                   need_v = row_needs(out_v, A.a.dim, false, true);
    int lo, hi;
    query_span(A, j, j, lq, lk, lo, hi);  // of a single key: the queries that see it
    bool settled = false;
    for (int h = hk * A.group; h < (hk + 1) * A.group && !settled; ++h)
        for (int i = lo; i < hi && !settled; ++i) {
            const int64_t q = q0 + i;
            lane_row(attn_row<T>(A.a.q, q, h, A.a.q_row, A.a.q_head), A.a.dim, x);
            lane_row(static_cast<const T*>(A.a.grad_out) + (q * A.a.heads + h) * A.a.dim, A.a.dim, g);
            const float s = fmaf(lane_dot(x, kx), A.scale_log2, pair_bias(A, q, k0 + j, h));
            const float w = exp2_sfu(s - load_lse2(A, q, h));
            const float ds = w * (lane_dot(g, vx) - A.a.delta[(int64_t)h * A.a.q_rows + q]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dv[e] = fmaf(w, g[e], dv[e]);
                dk[e] = fmaf(ds, x[e], dk[e]);
            }
            settled = row_settled(need_k, dk) && row_settled(need_v, dv);
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[e] *= A.a.scale;
    store_formed(out_k, A.a.dim, settled, need_k, dk);
    store_formed(out_v, A.a.dim, settled, need_v, dv);
}

}  // namespace
}  // namespace mpo
