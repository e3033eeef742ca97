// Norms of queries and keys for each head and the rotation by position in one
// pass, forward and backward (no counterpart in gamzerA/mps-pointops; it feeds
// the attention of serialised clouds, attention_common.cuh).
//
//   r = (mean_d x_d^2 + eps)^-1/2,  y = w x r,  theta_t = sum_a pos_a f[a, t],
//   (u, v)_t -> (u cos - v sin, u sin + v cos).
// Backward: g' = the output gradient turned by -theta, dw = sum g' x r over
// rows and heads, h = g' w, dx = r h - x r^3 mean(h x).
//
// Bound by HBM: the forward reads and writes q and k once, the backward reads
// x and its gradient and writes dx.  A warp owns one row (or, when rows are
// few, a share of one row's heads), so the angles of a row are formed once for
// all of its heads; `lanes` = dim / 8 rounded up to a power of two serve one
// head, each holding the two halves of four pairs as two vectors of four, so
// the rotation needs no exchange and the sums one butterfly.  Angles: position
// x frequency / pi is summed in double and reduced to one turn there (positions
// of 10^5 would cost a float sum 2 decimal digits), then sincospif.
#include <string>

#include "attention_common.cuh"

namespace mpo {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;

template <typename T>
struct Four;  // four consecutive elements as one vector
template <>
struct Four<float> {
    using V = float4;
    static __device__ __forceinline__ void get(V u, float* x) {
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    }
    static __device__ __forceinline__ V put(const float* x) {
        return make_float4(x[0], x[1], x[2], x[3]);
    }
};
template <>
struct Four<__half> {
    using V = uint2;
    static __device__ __forceinline__ void get(V u, float* x) {
        Elem<__half>::two(u.x, x);
        Elem<__half>::two(u.y, x + 2);
    }
    static __device__ __forceinline__ V put(const float* x) {
        return make_uint2(Elem<__half>::two(x[0], x[1]), Elem<__half>::two(x[2], x[3]));
    }
};
template <>
struct Four<__nv_bfloat16> {
    using V = uint2;
    static __device__ __forceinline__ void get(V u, float* x) {
        Elem<__nv_bfloat16>::two(u.x, x);
        Elem<__nv_bfloat16>::two(u.y, x + 2);
    }
    static __device__ __forceinline__ V put(const float* x) {
        return make_uint2(Elem<__nv_bfloat16>::two(x[0], x[1]),
                          Elem<__nv_bfloat16>::two(x[2], x[3]));
    }
};

// How a lane's eight elements sit in a head, and its angles.
struct Lane {
    int lo, hi;    // first element of each vector of four
    bool live;     // chunk inside the head
    bool turns;    // elements that rotate
    float c[4], s[4];
    __device__ __forceinline__ Lane(const mpo_rotate& a, int chunk) {
        live = chunk * 8 < a.dim;
        turns = live && chunk * 4 < a.pairs;
        lo = (turns && !a.interleaved) ? chunk * 4 : chunk * 8;
        hi = (turns && !a.interleaved) ? a.pairs + chunk * 4 : chunk * 8 + 4;
    }
    // Cosine and sine of the lane's four pairs at `row`.
    __device__ __forceinline__ void angles(const mpo_rotate& a, int chunk, int64_t row) {
        if (!turns) return;
        double t[4] = {0., 0., 0., 0.};
        for (int ax = 0; ax < a.axes; ++ax) {
            const int64_t at = row * a.axes + ax;
            const double p = a.position_float ? (double)static_cast<const float*>(a.position)[at]
                                              : (double)static_cast<const int32_t*>(a.position)[at];
            const float4 f = *reinterpret_cast<const float4*>(a.freqs + (int64_t)ax * a.pairs + chunk * 4);
            t[0] = fma(p, (double)f.x, t[0]);
            t[1] = fma(p, (double)f.y, t[1]);
            t[2] = fma(p, (double)f.z, t[2]);
            t[3] = fma(p, (double)f.w, t[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double half_turns = t[i] * 0.31830988618379067154;  // / pi
            const double whole = 2.0 * rint(half_turns * 0.5);
            sincospif((float)(half_turns - whole), &s[i], &c[i]);
        }
    }
    // Turn the lane's pairs by theta (sign 1) or -theta (sign -1).
    __device__ __forceinline__ void turn(float (&x)[8], bool interleaved, float sign) const {
        if (!turns) return;
        if (interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) rotate(x[2 * i], x[2 * i + 1], c[i], sign * s[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) rotate(x[i], x[4 + i], c[i], sign * s[i]);
        }
    }
    static __device__ __forceinline__ void rotate(float& u, float& v, float c, float s) {
        const float a = fmaf(u, c, -__fmul_rn(v, s)), b = fmaf(u, s, __fmul_rn(v, c));
        u = a;
        v = b;
    }
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, const Lane& L, float (&x)[8]) {
    using F = Four<T>;
    F::get(*reinterpret_cast<const typename F::V*>(p + L.lo), x);
    F::get(*reinterpret_cast<const typename F::V*>(p + L.hi), x + 4);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Lane& L, const float (&x)[8]) {
    using F = Four<T>;
    *reinterpret_cast<typename F::V*>(p + L.lo) = F::put(x);
    *reinterpret_cast<typename F::V*>(p + L.hi) = F::put(x + 4);
}
__device__ __forceinline__ void load_weight(const float* w, const Lane& L, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 1.f;
    if (w && L.live) load8<float>(w, L, x);
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

// Units of work: (row, share of the row's q and k heads); a warp takes units
// in grid strides.  A share's heads are consecutive, `step` = 32 / lanes of
// them at a time, U rounds of loads in flight.
template <typename T, int U>
__global__ void __launch_bounds__(kRotThreads)
norm_rotate_kernel(const mpo_rotate a, int lanes, int shares) {
    const int lane = threadIdx.x & 31, chunk = lane & (lanes - 1), sub = lane / lanes;
    const int step = 32 / lanes, total = a.heads + a.kv_heads;
    const int rounds = (total + step - 1) / step;
    Lane L(a, chunk);
    float wq[8], wk[8];
    load_weight(a.q_weight, L, wq);
    load_weight(a.k_weight, L, wk);
    const float inv = 1.f / (float)a.dim;
    const int64_t units = a.rows * shares;
    for (int64_t u = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5); u < units;
         u += (int64_t)gridDim.x * kRotWarps) {
        const int64_t row = u / shares;
        const int share = (int)(u - row * shares);
        const int r0 = (int)((int64_t)rounds * share / shares);
        const int r1 = (int)((int64_t)rounds * (share + 1) / shares);
        float x[U][8];
        auto fetch = [&](int r, float (&v)[8]) {
            const int h = r * step + sub;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            if (L.live && r < r1 && h < total)
                load8<T>(h < a.heads ? attn_row<T>(a.q, row, h, a.q_row, a.q_head)
                                     : attn_row<T>(a.k, row, h - a.heads, a.k_row, a.k_head),
                         L, v);
        };
#pragma unroll
        for (int i = 0; i < U; ++i) fetch(r0 + i, x[i]);
        L.angles(a, chunk, row);  // while the first loads are in flight
        for (int r = r0; r < r1; r += U) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (r + i < r1) {  // uniform over the warp
                    const int h = (r + i) * step + sub;
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss = fmaf(x[i][e], x[i][e], ss);
                    ss = lanes_sum(ss, lanes);
                    const float rs = rsqrtf(fmaf(ss, inv, a.eps));
                    const bool is_q = h < a.heads;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] * rs * (is_q ? wq[e] : wk[e]);
                    L.turn(x[i], a.interleaved, 1.f);
                    if (L.live && h < total)
                        store8<T>(is_q ? attn_row<T>(a.out_q, row, h, (int64_t)a.heads * a.dim, a.dim)
                                       : attn_row<T>(a.out_k, row, h - a.heads,
                                                     (int64_t)a.kv_heads * a.dim, a.dim),
                                  L, x[i]);
                    fetch(r + i + U, x[i]);
                }
            }
        }
    }
}

// Backward.  A lane keeps the weight gradients of its eight elements over all
// of its units; the block's warps and head slots join in shared memory in a
// fixed order and each block writes one partial (2, dim) row.
template <typename T>
__global__ void __launch_bounds__(kRotThreads)
norm_rotate_bwd_kernel(const mpo_rotate a, int lanes, int shares, float* __restrict__ partial) {
    const int lane = threadIdx.x & 31, chunk = lane & (lanes - 1), sub = lane / lanes;
    const int step = 32 / lanes, total = a.heads + a.kv_heads;
    const int rounds = (total + step - 1) / step;
    Lane L(a, chunk);
    float wq[8], wk[8], gq[8], gk[8];
    load_weight(a.q_weight, L, wq);
    load_weight(a.k_weight, L, wk);
#pragma unroll
    for (int e = 0; e < 8; ++e) gq[e] = gk[e] = 0.f;
    const float inv = 1.f / (float)a.dim;
    const int64_t units = a.rows * shares;
    const int64_t q_dense = (int64_t)a.heads * a.dim, k_dense = (int64_t)a.kv_heads * a.dim;
    for (int64_t u = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5); u < units;
         u += (int64_t)gridDim.x * kRotWarps) {
        const int64_t row = u / shares;
        const int share = (int)(u - row * shares);
        const int r0 = (int)((int64_t)rounds * share / shares);
        const int r1 = (int)((int64_t)rounds * (share + 1) / shares);
        float x[8], g[8];
        auto fetch = [&](int r) {
            const int h = r * step + sub;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = g[i] = 0.f;
            if (L.live && r < r1 && h < total) {
                if (h < a.heads) {
                    load8<T>(attn_row<T>(a.q, row, h, a.q_row, a.q_head), L, x);
                    load8<T>(attn_row<T>(a.grad_q, row, h, q_dense, a.dim), L, g);
                } else {
                    load8<T>(attn_row<T>(a.k, row, h - a.heads, a.k_row, a.k_head), L, x);
                    load8<T>(attn_row<T>(a.grad_k, row, h - a.heads, k_dense, a.dim), L, g);
                }
            }
        };
        fetch(r0);
        L.angles(a, chunk, row);
        for (int r = r0; r < r1; ++r) {
            const int h = r * step + sub;
            const bool is_q = h < a.heads;
            float y[8], b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = x[e];
                b[e] = g[e];
            }
            fetch(r + 1);
            L.turn(b, a.interleaved, -1.f);
            float ss = 0.f, hx = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = fmaf(y[e], y[e], ss);
                hx = fmaf(__fmul_rn(b[e], is_q ? wq[e] : wk[e]), y[e], hx);
            }
            ss = lanes_sum(ss, lanes);
            hx = lanes_sum(hx, lanes);
            const float rs = rsqrtf(fmaf(ss, inv, a.eps));
            const float back = hx * inv * rs * rs * rs;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float dw = __fmul_rn(b[e], __fmul_rn(y[e], rs));
                if (h < total) {
                    if (is_q) gq[e] += dw;
                    else gk[e] += dw;
                }
                y[e] = fmaf(-y[e], back, __fmul_rn(rs, __fmul_rn(b[e], is_q ? wq[e] : wk[e])));
            }
            if (L.live && h < total)
                store8<T>(is_q ? attn_row<T>(a.out_q, row, h, q_dense, a.dim)
                               : attn_row<T>(a.out_k, row, h - a.heads, k_dense, a.dim),
                          L, y);
        }
    }
    if (!partial) return;
    __shared__ float sums[kRotWarps][32][17];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        sums[threadIdx.x >> 5][lane][e] = gq[e];
        sums[threadIdx.x >> 5][lane][8 + e] = gk[e];
    }
    __syncthreads();
    // Element e of chunk c: over the warps, then the head slots.
    for (int t = threadIdx.x; t < 16 * lanes; t += kRotThreads) {
        const int c = t >> 4, e = t & 15;
        if (c * 8 >= a.dim) continue;
        float v = 0.f;
        for (int w = 0; w < kRotWarps; ++w)
            for (int sl = 0; sl < step; ++sl) v += sums[w][sl * lanes + c][e];
        const Lane at(a, c);
        const int el = (e & 7) < 4 ? at.lo + (e & 3) : at.hi + (e & 3);
        partial[((int64_t)blockIdx.x * 2 + (e >> 3)) * a.dim + el] = v;
    }
}

// grad_weight[d] = sum of the blocks' partials in block order (8 strided runs,
// then their sum).
__global__ void __launch_bounds__(256)
norm_weight_reduce_kernel(const float* __restrict__ partial, int blocks, int dim,
                          float* __restrict__ gq, float* __restrict__ gk) {
    __shared__ float run[8][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float v = 0.f;
    if (col < 2 * dim)
        for (int b = part; b < blocks; b += 8) v += partial[(int64_t)b * 2 * dim + col];
    run[part][threadIdx.x & 31] = v;
    __syncthreads();
    if (part == 0 && col < 2 * dim) {
        for (int i = 1; i < 8; ++i) v += run[i][threadIdx.x & 31];
        float* out = col < dim ? gq : gk;
        if (out) out[col < dim ? col : col - dim] = v;
    }
}

int rotate_lanes(int dim) {
    int l = 1;
    while (l * 8 < dim) l <<= 1;
    return l;
}
struct RotateGrid {
    int lanes, shares;
    unsigned blocks;
};
// At most 8 blocks of 8 warps per SM (its 64 warps); rows are shared out over
// several warps when there are fewer rows than half of those warps.
RotateGrid rotate_grid(const mpo_rotate& a, int per_sm) {
    RotateGrid g;
    g.lanes = rotate_lanes(a.dim);
    const int64_t rounds = ceil_div(a.heads + a.kv_heads, 32 / g.lanes);
    const int64_t warps = (int64_t)sm_count() * per_sm * kRotWarps;
    g.shares = (int)max64(1, min64(rounds, warps / (2 * max64(a.rows, 1))));
    g.blocks = (unsigned)max64(1, min64(ceil_div(a.rows * g.shares, kRotWarps),
                                        (int64_t)sm_count() * per_sm));
    return g;
}
constexpr int kBwdBlocksPerSm = 4;

bool vec_ok(const void* p, int64_t row, int64_t head, int dtype) {
    const uintptr_t bytes = dtype == MPO_F32 ? 16 : 8;
    return aligned_to(p, bytes) && row % 4 == 0 && head % 4 == 0;
}

int check_rotate(const mpo_rotate* a, bool backward, const char* what) {
    auto bad = [&](const char* m) { return fail(kInvalidArgument, std::string(what) + ": " + m); };
    if (!a) return bad("null arguments");
    if (a->dtype < MPO_F32 || a->dtype > MPO_BF16) return bad("unknown dtype");
    if (a->rows < 0 || a->heads < 1 || a->kv_heads < 1) return bad("bad sizes");
    if ((int64_t)a->heads + a->kv_heads > (1 << 20)) return bad("too many heads");
    if (a->dim < 8 || a->dim > 256 || a->dim % 8) return bad("dim must be a multiple of 8 up to 256");
    if (a->pairs < 0 || a->pairs % 4 || 2 * a->pairs > a->dim)
        return bad("pairs must be a multiple of 4 with 2 * pairs <= dim");
    if (a->pairs && (a->axes < 1 || a->axes > kAttnMaxAxes)) return bad("axes must be in [1, 3]");
    if (a->rows == 0) return kOk;
    if (!a->q || !a->k || !a->out_q || !a->out_k) return bad("null pointer");
    if (a->pairs && (!a->position || !a->freqs)) return bad("null pointer");
    if (a->pairs && !aligned_to(a->freqs, 16)) return bad("freqs must be 16-byte aligned");
    if (!aligned_to(a->q_weight, 16) || !aligned_to(a->k_weight, 16))
        return bad("weights must be 16-byte aligned");
    const int64_t qd = (int64_t)a->heads * a->dim, kd = (int64_t)a->kv_heads * a->dim;
    if (!vec_ok(a->q, a->q_row, a->q_head, a->dtype) || !vec_ok(a->k, a->k_row, a->k_head, a->dtype) ||
        !vec_ok(a->out_q, qd, a->dim, a->dtype) || !vec_ok(a->out_k, kd, a->dim, a->dtype))
        return bad("rows must start on multiples of four elements");
    if (backward) {
        if (!a->grad_q || !a->grad_k) return bad("null pointer");
        if (!vec_ok(a->grad_q, qd, a->dim, a->dtype) || !vec_ok(a->grad_k, kd, a->dim, a->dtype))
            return bad("rows must start on multiples of four elements");
    }
    return kOk;
}

template <typename T>
int run_rotate(const mpo_rotate& a, cudaStream_t s) {
    const RotateGrid g = rotate_grid(a, 8);
    norm_rotate_kernel<T, 2><<<g.blocks, kRotThreads, 0, s>>>(a, g.lanes, g.shares);
    return check_launch("norm_rotate_kernel");
}
template <typename T>
int run_rotate_bwd(const mpo_rotate& a, cudaStream_t s) {
    const RotateGrid g = rotate_grid(a, kBwdBlocksPerSm);
    const bool weights = a.grad_q_weight || a.grad_k_weight;
    float* partial = weights ? static_cast<float*>(a.workspace) : nullptr;
    norm_rotate_bwd_kernel<T><<<g.blocks, kRotThreads, 0, s>>>(a, g.lanes, g.shares, partial);
    int st = check_launch("norm_rotate_bwd_kernel");
    if (st != kOk || !weights) return st;
    norm_weight_reduce_kernel<<<(unsigned)ceil_div(2 * a.dim, 32), 256, 0, s>>>(
        partial, (int)g.blocks, a.dim, a.grad_q_weight, a.grad_k_weight);
    return check_launch("norm_weight_reduce_kernel");
}

}  // namespace
}  // namespace mpo

extern "C" {

int mpo_norm_rotate(const mpo_rotate* args, void* stream) {
    using namespace mpo;
    const int st = check_rotate(args, false, __func__);
    if (st != kOk || args->rows == 0) return st;
    cudaStream_t s = (cudaStream_t)stream;
    switch (args->dtype) {
        case MPO_F32: return run_rotate<float>(*args, s);
        case MPO_F16: return run_rotate<__half>(*args, s);
        default: return run_rotate<__nv_bfloat16>(*args, s);
    }
}

size_t mpo_norm_rotate_workspace_bytes(const mpo_rotate* args) {
    using namespace mpo;
    if (check_rotate(args, false, __func__) != kOk) return 0;
    if (!args->grad_q_weight && !args->grad_k_weight) return 0;
    return (size_t)sm_count() * kBwdBlocksPerSm * 2 * args->dim * sizeof(float);
}

int mpo_norm_rotate_backward(const mpo_rotate* args, void* stream) {
    using namespace mpo;
    const int st = check_rotate(args, true, __func__);
    if (st != kOk) return st;
    cudaStream_t s = (cudaStream_t)stream;
    if (args->rows == 0) {
        for (float* g : {args->grad_q_weight, args->grad_k_weight})
            if (g && cudaMemsetAsync(g, 0, sizeof(float) * args->dim, s) != cudaSuccess)
                return fail(kCudaError, std::string(__func__) + ": memset failed");
        return kOk;
    }
    MPO_REQUIRE_WORKSPACE(args->workspace);
    const bool weights = args->grad_q_weight || args->grad_k_weight;
    if (weights && (!args->workspace ||
                    args->workspace_bytes <
                        (size_t)sm_count() * kBwdBlocksPerSm * 2 * args->dim * sizeof(float)))
        return fail(kWorkspaceTooSmall, std::string(__func__) + ": workspace too small");
    switch (args->dtype) {
        case MPO_F32: return run_rotate_bwd<float>(*args, s);
        case MPO_F16: return run_rotate_bwd<__half>(*args, s);
        default: return run_rotate_bwd<__nv_bfloat16>(*args, s);
    }
}

}  // extern "C"
