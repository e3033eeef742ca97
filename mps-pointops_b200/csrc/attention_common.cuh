// Attention along the serialised order of a ragged batch of clouds: shapes,
// visibility and the pieces that its kernels share.
//
// Rows are flat.  Cloud b has Lq query rows and Lk key rows (offset arrays);
// query row i of a cloud stands at position p = i + Lk - Lq among its keys, so
// self attention has p = i and a chunk of new rows sits at the end of what is
// cached.  Key j is visible to a query at p when
//   (j < sinks  or  p - left <= j <= p + right)  and  (not causal or j <= p).
// With S = scale q.k + sum_a T[a, bucket(clamp(kpos_a - qpos_a, -R, R) + R), h]
//   P = softmax of S over the visible keys,  o = P v,  lse = log sum exp S
// (no visible key: o = 0, lse = -inf), and backwards, with D_i = o_i . do_i,
//   dS = P (do v^T - D),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T do,
//   dT[a, b, h] = sum of dS over the pairs whose bucket on axis a is b.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <string>
#include <type_traits>

#include "../../include/mpo_b200.h"
#include "mpo_common.cuh"

namespace mpo {

constexpr int kAttnTile = 128;        // rows of one planned tile (query or key side)
constexpr int kAttnMaxDim = 128;
constexpr int kAttnMaxAxes = 3;
constexpr int kAttnMaxEntries = 256;  // axes x buckets of a bias table
constexpr int kAttnMaxMap = 2049;     // 2 R + 1 of a bucket map
constexpr size_t kAttnSmem = 232448;  // shared memory of a block at most

// One planned tile: `rows` consecutive rows of one cloud on the owning side.
struct AttnTile {
    int32_t row;   // first row, global, owning side
    int32_t rows;  // 1 .. kAttnTile
    int32_t first; // query tiles: position p of the first row; key tiles: its index j
    int32_t other; // first row of the cloud on the other side, global
    int32_t lq, lk;
    int32_t base;  // first row of the cloud on the owning side, global
    int32_t cloud;
};
static_assert(sizeof(AttnTile) == 32, "eight 32-bit words per tile");

// The argument block of the C ABI with what the kernels derive from it.
struct AttnArgs {
    mpo_attention a;
    int left, right;  // kUnlimited where there is none; right 0 when causal
    int group;        // query heads per key head
    float scale_log2; // scale * log2(e)
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Rows of queries and keys stay below kFar together, so a position plus or
// minus the distance that stands for "no limit" reaches every key and fits 32 bits.
constexpr int kFar = 1 << 30;
constexpr int kUnlimited = kFar - 2;

__device__ __forceinline__ bool attn_visible(const AttnArgs& A, int p, int j) {
    return ((j < A.a.sinks) | ((j >= p - A.left) & (j <= p + A.right))) & (!A.a.causal | (j <= p));
}

// The key tiles (W keys each, aligned to W within the cloud) that the rows at
// positions [p0, p1] can see: `ns` tiles from key 0 for the sinks, then `nw`
// tiles from tile `w0` for the window (one run from tile 0 where they meet).
struct KeySpan {
    int ns, w0, nw;
    __device__ __forceinline__ int count() const { return ns + nw; }
    __device__ __forceinline__ int tile(int t) const { return t < ns ? t : w0 + (t - ns); }
};
__device__ __forceinline__ KeySpan key_span(const AttnArgs& A, int p0, int p1, int lk, int W) {
    const int hi = min(lk, p1 + A.right + 1), lo = max(0, p0 - A.left);
    int se = min(A.a.sinks, lk);
    if (A.a.causal) se = min(se, p1 + 1);
    const int st = se > 0 ? (se + W - 1) / W : 0;
    KeySpan s;
    s.ns = st;
    s.w0 = s.nw = 0;
    if (hi > lo) {
        s.w0 = lo / W;
        int end = (hi + W - 1) / W;
        if (st >= s.w0) {
            if (st > 0) s.w0 = 0;
            end = max(end, st);
            s.ns = 0;
        }
        s.nw = end - s.w0;
    }
    return s;
}
// Every key of [k0, k1] visible to every row of [p0, p1].
__device__ __forceinline__ bool all_visible(const AttnArgs& A, int p0, int p1, int k0, int k1) {
    return (k1 < A.a.sinks || (k0 >= p1 - A.left && k1 <= p0 + A.right)) &&
           (!A.a.causal || k1 <= p0);
}
// The query rows (local indices [lo, hi)) that can see some key of [k0, k1].
__device__ __forceinline__ void query_span(const AttnArgs& A, int k0, int k1, int lq, int lk,
                                           int& lo, int& hi) {
    const int shift = lk - lq;  // p = i + shift
    if (k0 < A.a.sinks) {
        lo = A.a.causal ? k0 - shift : 0;
        hi = lq;
    } else {
        lo = k0 - A.right - shift;
        hi = k1 + A.left - shift + 1;
    }
    lo = max(0, lo);
    hi = min(lq, hi);
}

// ---------------------------------------------------------------- elements
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kVec = 4;  // elements in 16 bytes
    static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y);
        x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                          __float_as_uint(x[3]));
    }
    static __device__ __forceinline__ float to(float x) { return x; }
    static __device__ __forceinline__ float from(float x) { return x; }
};
template <>
struct Elem<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void two(uint32_t u, float* x) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        x[0] = f.x; x[1] = f.y;
    }
    static __device__ __forceinline__ uint32_t two(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
        two(u.x, x); two(u.y, x + 2); two(u.z, x + 4); two(u.w, x + 6);
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7]));
    }
    static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half from(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void two(uint32_t u, float* x) {
        x[0] = __uint_as_float(u << 16);
        x[1] = __uint_as_float(u & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t two(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
        two(u.x, x); two(u.y, x + 2); two(u.z, x + 4); two(u.w, x + 6);
    }
    static __device__ __forceinline__ uint4 pack(const float* x) {
        return make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7]));
    }
    static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 from(float x) { return __float2bfloat16_rn(x); }
};

// 2^x by the SFU (2 ulp); -inf gives 0.
__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ T* attn_row(void* base, int64_t row, int64_t head, int64_t row_stride,
                                       int64_t head_stride) {
    return static_cast<T*>(base) + row * row_stride + head * head_stride;
}
template <typename T>
__device__ __forceinline__ const T* attn_row(const void* base, int64_t row, int64_t head,
                                             int64_t row_stride, int64_t head_stride) {
    return static_cast<const T*>(base) + row * row_stride + head * head_stride;
}

// ---------------------------------------------------------------- bias
// Bucket of a coordinate difference on one axis: clamped to [0, 2 R], then
// through the map when there is one (staged in shared memory as bytes).  The
// difference fits 32 bits: positions are below 2^30 in magnitude.
__device__ __forceinline__ int bias_bucket(int kpos, int qpos, int reach, const uint8_t* map) {
    const int c = min(max(kpos - qpos, -reach), reach) + reach;
    return map ? (int)map[c] : c;
}

// Table entry (axis, bucket) of head h, as float.
__device__ __forceinline__ float table_entry(const mpo_attention& a, int e, int h) {
    const int64_t at = (int64_t)e * a.heads + h;
    if (a.table_dtype == MPO_F32) return static_cast<const float*>(a.table)[at];
    if (a.table_dtype == MPO_F16) return __half2float(static_cast<const __half*>(a.table)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[at]);
}

// ---------------------------------------------------------------- launchers
// Lets a kernel take all of an SM's shared memory, once per device: a limit of
// each call's own size would be lowered by other host threads before the launch.
template <auto Kernel>
int attn_prepare(const char* what) {
    static std::atomic<uint64_t> prepared{0};
    const uint64_t bit = 1ull << (current_device() & 63);
    if (prepared.load(std::memory_order_acquire) & bit) return kOk;
    if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kAttnSmem) != cudaSuccess)
        return fail(kCudaError, std::string(what) + ": cannot reserve shared memory");
    prepared.fetch_or(bit, std::memory_order_release);
    return kOk;
}

// attention_tc_fwd.cu, attention_tc_bwd.cu: 16-bit types on the tensor cores.
int attn_tc_forward(const AttnArgs& A, cudaStream_t s);
int attn_tc_backward(const AttnArgs& A, cudaStream_t s);
// attention_rows.cu: few query rows per cloud.
bool attn_rows_eligible(const AttnArgs& A);
size_t attn_rows_workspace(const AttnArgs& A);
int attn_rows_forward(const AttnArgs& A, cudaStream_t s);
// attention_simt.cu: 32-bit arithmetic throughout.
int attn_simt_forward(const AttnArgs& A, cudaStream_t s);
int attn_simt_backward(const AttnArgs& A, cudaStream_t s);

}  // namespace mpo
