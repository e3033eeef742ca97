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
// all of its heads, one pair per lane; `lanes` = dim / 8 rounded up to a power
// of two serve one head, each holding the two halves of four pairs as two
// vectors of four, so the rotation needs no exchange and the sums one butterfly.  Angles are formed in
// the type of the frequencies (float32: as elementary float32 operations give
// them; float64 for positions whose float32 angle would be off by too much),
// reduced to one turn in double with the rest of 1 / pi, then sincospif.
//
// At that size the forward moves 4.6 TB/s and the backward 4.7 TB/s, 70 % of a
// plain copy.  Instructions hold it (68 % of the issue slots in the forward), not
// loads in flight: fetching the next row's heads ahead took 281 and 411 us against
// 246 and 362, and weights read once per row instead of once per round 348 against
// 358 us in the backward.
#include <string>
#include <type_traits>

#include "attention_common.cuh"

namespace mpo {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotWarps = kRotThreads / 32;
// Resident, by registers.  262144 rows of 8 + 8 heads of 64 (bf16, 48 elements turned on
// three axes): forward at 2 / 3 / 4 blocks 266 / 235 / 241 us, backward at 2 / 3 344 / 535 us.
constexpr int kFwdBlocksPerSm = 3, kBwdBlocksPerSm = 2;

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

// How a lane's eight elements sit in a head.
struct Lane {
    int lo, hi;    // first element of each vector of four
    bool live;     // chunk inside the head
    bool turns;    // elements that rotate
    __device__ __forceinline__ Lane(const mpo_rotate& a, int chunk) {
        live = chunk * 8 < a.dim;
        turns = live && chunk * 4 < a.pairs;
        lo = (turns && !a.interleaved) ? chunk * 4 : chunk * 8;
        hi = (turns && !a.interleaved) ? a.pairs + chunk * 4 : chunk * 8 + 4;
    }
};

// Eight elements as packed pairs.  Where they rotate, v[0], v[1] hold the first
// halves of the lane's four pairs and v[2], v[3] the second halves.
struct Eight {
    f32x2 v[4];
};
template <typename T>
struct Raw {  // eight elements as loaded
    typename Four<T>::V lo, hi;
};
template <typename T>
__device__ __forceinline__ Eight unpack(const Raw<T>& r, bool interleaved) {
    float x[8];
    Four<T>::get(r.lo, x);
    Four<T>::get(r.hi, x + 4);
    Eight e;
    if (interleaved) {
        e.v[0] = pack2(x[0], x[2]);
        e.v[1] = pack2(x[4], x[6]);
        e.v[2] = pack2(x[1], x[3]);
        e.v[3] = pack2(x[5], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e.v[i] = pack2(x[2 * i], x[2 * i + 1]);
    }
    return e;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int apart, const Eight& e, bool interleaved) {
    float x[8];
    if (interleaved) {
        unpack2(e.v[0], x[0], x[2]);
        unpack2(e.v[1], x[4], x[6]);
        unpack2(e.v[2], x[1], x[3]);
        unpack2(e.v[3], x[5], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(e.v[i], x[2 * i], x[2 * i + 1]);
    }
    *reinterpret_cast<typename Four<T>::V*>(p) = Four<T>::put(x);
    *reinterpret_cast<typename Four<T>::V*>(p + apart) = Four<T>::put(x + 4);
}
// Weights of q and k in shared memory, by chunk in the order of an Eight (ones
// where none is given).
__device__ __forceinline__ void stage_weights(const mpo_rotate& a, float (&w)[2][32][8], int lanes) {
    for (int t = threadIdx.x; t < 2 * lanes; t += kRotThreads) {
        const int which = t / lanes, chunk = t - which * lanes;
        const Lane L(a, chunk);
        const float* src = which ? a.k_weight : a.q_weight;
        float x[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (src && L.live) {
            Four<float>::get(*reinterpret_cast<const float4*>(src + L.lo), x);
            Four<float>::get(*reinterpret_cast<const float4*>(src + L.hi), x + 4);
        }
        const bool il = a.interleaved && L.turns;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[which][chunk][il ? (i & 1) * 4 + (i >> 1) : i] = x[i];
    }
}
__device__ __forceinline__ Eight read_weight(const float* w) {
    const float4 lo = reinterpret_cast<const float4*>(w)[0], hi = reinterpret_cast<const float4*>(w)[1];
    Eight e;
    e.v[0] = pack2(lo.x, lo.y);
    e.v[1] = pack2(lo.z, lo.w);
    e.v[2] = pack2(hi.x, hi.y);
    e.v[3] = pack2(hi.z, hi.w);
    return e;
}
__device__ __forceinline__ float pair_sum(f32x2 a, f32x2 b) {
    float x, y;
    unpack2(add2(a, b), x, y);
    return x + y;
}
__device__ __forceinline__ float dot8(const Eight& a, const Eight& b) {
    const f32x2 p = fma2(a.v[2], b.v[2], mul2(a.v[0], b.v[0]));
    const f32x2 q = fma2(a.v[3], b.v[3], mul2(a.v[1], b.v[1]));
    return pair_sum(p, q);
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES >> 1; o; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
    return v;
}

// Cosines and sines of the lane's four pairs, and the sines negated.
struct Turn {
    f32x2 c[2], s[2], n[2];
    // (u, v) -> (u c - v s, u s + v c); BACK: by -theta.
    template <bool BACK>
    __device__ __forceinline__ void apply(Eight& e) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 u = e.v[i], v = e.v[2 + i];
            e.v[i] = fma2(u, c[i], mul2(v, BACK ? s[i] : n[i]));
            e.v[2 + i] = fma2(u, BACK ? n[i] : s[i], mul2(v, c[i]));
        }
    }
};
// The angles of a row: each lane forms those of pairs lane, lane + 32, .., and
// the warp shares them through `cs` (cosines, then sines, kMaxPairs each).
constexpr int kMaxPairs = 128;
// P: the positions' type, which goes to the frequencies' type in one rounding.
template <typename P>
__device__ __forceinline__ void load_positions(const mpo_rotate& a, int64_t row, P (&pos)[kAttnMaxAxes]) {
#pragma unroll
    for (int ax = 0; ax < kAttnMaxAxes; ++ax)
        pos[ax] = ax < a.axes ? static_cast<const P*>(a.position)[row * a.axes + ax] : P(0);
}
template <typename P>
__device__ __forceinline__ double pair_angle(const mpo_rotate& a, const P (&pos)[kAttnMaxAxes], int t) {
    if (a.freqs_double) {
        double sum = 0.;
#pragma unroll
        for (int ax = 0; ax < kAttnMaxAxes; ++ax)
            if (ax < a.axes)
                sum = __dadd_rn(sum, __dmul_rn((double)pos[ax], static_cast<const double*>(a.freqs)[ax * a.pairs + t]));
        return sum;
    }
    float sum = 0.f;
#pragma unroll
    for (int ax = 0; ax < kAttnMaxAxes; ++ax)
        if (ax < a.axes)
            sum = __fadd_rn(sum, __fmul_rn((float)pos[ax], static_cast<const float*>(a.freqs)[ax * a.pairs + t]));
    return (double)sum;
}
template <typename P>
__device__ __forceinline__ void angles_of(const mpo_rotate& a, int64_t row, float* cs) {
    P pos[kAttnMaxAxes];
    load_positions(a, row, pos);
    __syncwarp();  // the previous row's angles have been read
    for (int t = threadIdx.x & 31; t < a.pairs; t += 32) {
        // Half turns: theta / pi as a product with 1 / pi, and what that leaves out (the product's
        // rounding, and that of 1 / pi), which counts where theta is large.
        const double theta = pair_angle(a, pos, t), kInvPi = 0.31830988618379067154;
        const double half_turns = theta * kInvPi;
        const double rest = fma(theta, -1.9678676675182486e-17, fma(theta, kInvPi, -half_turns));
        const double whole = 2.0 * rint(half_turns * 0.5);
        sincospif((float)((half_turns - whole) + rest), cs + kMaxPairs + t, cs + t);
    }
    __syncwarp();
}
__device__ __forceinline__ void row_angles(const mpo_rotate& a, int64_t row, float* cs) {
    if (a.position_float == MPO_POSITION_F32) angles_of<float>(a, row, cs);
    else if (a.position_float == MPO_POSITION_I32) angles_of<int32_t>(a, row, cs);
    else angles_of<int64_t>(a, row, cs);
}
__device__ __forceinline__ Turn read_turn(const float* cs, int chunk) {
    const float4 c = *reinterpret_cast<const float4*>(cs + 4 * chunk);
    const float4 s = *reinterpret_cast<const float4*>(cs + kMaxPairs + 4 * chunk);
    Turn t;
    t.c[0] = pack2(c.x, c.y);
    t.c[1] = pack2(c.z, c.w);
    t.s[0] = pack2(s.x, s.y);
    t.s[1] = pack2(s.z, s.w);
    t.n[0] = pack2(-s.x, -s.y);
    t.n[1] = pack2(-s.z, -s.w);
    return t;
}

// Units of work: (row, share of the row's heads); a warp takes units in grid
// strides.  A round serves 32 / LANES heads of q or of k; U rounds of loads of
// each are in flight, as loaded (packed), and the first of them go out before
// the row's angles are formed.  A lane past the last head loads that head again
// and stores nothing.
template <typename T>
__device__ __forceinline__ Raw<T> load_at(const T* base, int head, int stride, int apart) {
    const T* p = base + (int64_t)head * stride;
    Raw<T> r;
    r.lo = *reinterpret_cast<const typename Four<T>::V*>(p);
    r.hi = *reinterpret_cast<const typename Four<T>::V*>(p + apart);
    return r;
}
// Runs f(this lane's head, ring slot) over the rounds of `heads` heads from `first`.
template <int U, typename F>
__device__ __forceinline__ void over_rounds(int sub, int first, int step, int heads, F&& f) {
    for (int h = first; h < heads; h += U * step) {  // uniform over the warp
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (h + i * step < heads) f(h + i * step + sub, i);
    }
}

template <typename T, int U, bool IL, int LANES>
__global__ void __launch_bounds__(kRotThreads, kFwdBlocksPerSm)
norm_rotate_kernel(const __grid_constant__ mpo_rotate a, int shares) {
    constexpr int kHeads = 32 / LANES;
    __shared__ __align__(16) float angles[kRotWarps][2 * kMaxPairs];
    __shared__ __align__(16) float weights[2][32][8];
    float* cs = angles[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31, chunk = lane % LANES, sub = lane / LANES;
    const Lane L(a, chunk);
    const bool il = IL && L.turns;
    const int apart = L.hi - L.lo, lo = L.live ? L.lo : 0, step = kHeads * shares;
    stage_weights(a, weights, LANES);
    __syncthreads();
    const float inv = 1.f / (float)a.dim;
    const int64_t units = a.rows * shares;
    for (int64_t u = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5); u < units;
         u += (int64_t)gridDim.x * kRotWarps) {
        const int64_t row = shares == 1 ? u : u / shares;
        const int first = shares == 1 ? 0 : (int)(u - row * shares) * kHeads;
        const T* q = static_cast<const T*>(a.q) + row * a.q_row + lo;
        const T* k = static_cast<const T*>(a.k) + row * a.k_row + lo;
        Raw<T> rq[U], rk[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            rq[i] = load_at<T>(q, min(first + i * step + sub, a.heads - 1), (int)a.q_head, apart);
            rk[i] = load_at<T>(k, min(first + i * step + sub, a.kv_heads - 1), (int)a.k_head, apart);
        }
        Turn turn;
        if (a.pairs) {
            row_angles(a, row, cs);
            if (L.turns) turn = read_turn(cs, chunk);
        }
        auto all = [&](const T* in, int stride, T* out, int heads, Raw<T>(&raw)[U], const float* weight) {
            const Eight w = read_weight(weight);
            over_rounds<U>(sub, first, step, heads, [&](int h, int i) {
                Eight x = unpack<T>(raw[i], il);
                if (h - sub + U * step < heads) raw[i] = load_at<T>(in, min(h + U * step, heads - 1), stride, apart);
                if (!L.live) x = Eight{};
                const float rs = rsqrtf(fmaf(lanes_sum<LANES>(dot8(x, x)), inv, a.eps));
                const f32x2 rs2 = pack2(rs, rs);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.v[e] = mul2(mul2(x.v[e], rs2), w.v[e]);
                if (L.turns) turn.template apply<false>(x);
                if (L.live && h < heads) store8<T>(out + h * a.dim, apart, x, il);
            });
        };
        all(q, (int)a.q_head, static_cast<T*>(a.out_q) + row * a.heads * a.dim + lo, a.heads, rq, weights[0][chunk]);
        all(k, (int)a.k_head, static_cast<T*>(a.out_k) + row * a.kv_heads * a.dim + lo, a.kv_heads, rk,
            weights[1][chunk]);
    }
}

// Backward.  A lane keeps the weight gradients of its eight elements over all
// of its units; the block's warps and head slots join in shared memory in a
// fixed order and each block writes one partial (2, dim) row.
template <typename T, int U, bool IL, int LANES>
__global__ void __launch_bounds__(kRotThreads, kBwdBlocksPerSm)
norm_rotate_bwd_kernel(const __grid_constant__ mpo_rotate a, int shares, float* __restrict__ partial) {
    constexpr int kHeads = 32 / LANES;
    __shared__ __align__(16) union {
        float angles[kRotWarps][2 * kMaxPairs];
        float sums[kRotWarps][32][17];
    } sh;
    __shared__ __align__(16) float weights[2][32][8];
    float* cs = sh.angles[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31, chunk = lane % LANES, sub = lane / LANES;
    const Lane L(a, chunk);
    const bool il = IL && L.turns;
    const int apart = L.hi - L.lo, lo = L.live ? L.lo : 0, step = kHeads * shares;
    stage_weights(a, weights, LANES);
    __syncthreads();
    Eight gq, gk;
#pragma unroll
    for (int e = 0; e < 4; ++e) gq.v[e] = gk.v[e] = pack2(0.f, 0.f);
    const float inv = 1.f / (float)a.dim;
    const int64_t units = a.rows * shares;
    for (int64_t u = (int64_t)blockIdx.x * kRotWarps + (threadIdx.x >> 5); u < units;
         u += (int64_t)gridDim.x * kRotWarps) {
        const int64_t row = shares == 1 ? u : u / shares;
        const int first = shares == 1 ? 0 : (int)(u - row * shares) * kHeads;
        const T* q = static_cast<const T*>(a.q) + row * a.q_row + lo;
        const T* k = static_cast<const T*>(a.k) + row * a.k_row + lo;
        const int64_t dq = row * a.heads * a.dim + lo, dk = row * a.kv_heads * a.dim + lo;
        const T* gyq = static_cast<const T*>(a.grad_q) + dq;
        const T* gyk = static_cast<const T*>(a.grad_k) + dk;
        Raw<T> rq[U], rk[U], rgq[U], rgk[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int hq = min(first + i * step + sub, a.heads - 1), hk = min(first + i * step + sub, a.kv_heads - 1);
            rq[i] = load_at<T>(q, hq, (int)a.q_head, apart);
            rgq[i] = load_at<T>(gyq, hq, a.dim, apart);
            rk[i] = load_at<T>(k, hk, (int)a.k_head, apart);
            rgk[i] = load_at<T>(gyk, hk, a.dim, apart);
        }
        Turn turn;
        if (a.pairs) {
            row_angles(a, row, cs);
            if (L.turns) turn = read_turn(cs, chunk);
        }
        auto all = [&](const T* in, int stride, const T* gin, T* out, int heads, Raw<T>(&raw)[U], Raw<T>(&rg)[U],
                       const float* weight, Eight& gw) {
            const Eight w = read_weight(weight);
            over_rounds<U>(sub, first, step, heads, [&](int h, int i) {
                Eight y = unpack<T>(raw[i], il), b = unpack<T>(rg[i], il), hw;
                if (h - sub + U * step < heads) {
                    const int next = min(h + U * step, heads - 1);
                    raw[i] = load_at<T>(in, next, stride, apart);
                    rg[i] = load_at<T>(gin, next, a.dim, apart);
                }
                const bool on = L.live && h < heads;
                if (!on) y = b = Eight{};  // adds nothing to the weights' gradients
                if (L.turns) turn.template apply<true>(b);
#pragma unroll
                for (int e = 0; e < 4; ++e) hw.v[e] = mul2(b.v[e], w.v[e]);
                const float ss = lanes_sum<LANES>(dot8(y, y)), hx = lanes_sum<LANES>(dot8(hw, y));
                const float rs = rsqrtf(fmaf(ss, inv, a.eps));
                const float back = -(hx * inv * rs * rs * rs);
                const f32x2 rs2 = pack2(rs, rs), back2 = pack2(back, back);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    gw.v[e] = fma2(b.v[e], mul2(y.v[e], rs2), gw.v[e]);
                    y.v[e] = fma2(y.v[e], back2, mul2(rs2, hw.v[e]));
                }
                if (on) store8<T>(out + h * a.dim, apart, y, il);
            });
        };
        all(q, (int)a.q_head, gyq, static_cast<T*>(a.out_q) + dq, a.heads, rq, rgq, weights[0][chunk], gq);
        all(k, (int)a.k_head, gyk, static_cast<T*>(a.out_k) + dk, a.kv_heads, rk, rgk, weights[1][chunk], gk);
    }
    if (!partial) return;
    __syncthreads();
    // Sums slot e < 8: q, else k; within a weight: lo's four elements, then hi's.
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const Eight& g = which ? gk : gq;
        float* dst = &sh.sums[threadIdx.x >> 5][lane][8 * which];
        if (il) {
            unpack2(g.v[0], dst[0], dst[2]);
            unpack2(g.v[1], dst[4], dst[6]);
            unpack2(g.v[2], dst[1], dst[3]);
            unpack2(g.v[3], dst[5], dst[7]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack2(g.v[e], dst[2 * e], dst[2 * e + 1]);
        }
    }
    __syncthreads();
    // Element e of chunk c: over the warps, then the head slots.
    for (int t = threadIdx.x; t < 16 * LANES; t += kRotThreads) {
        const int c = t >> 4, e = t & 15;
        if (c * 8 >= a.dim) continue;
        float v = 0.f;
        for (int w = 0; w < kRotWarps; ++w)
            for (int sl = 0; sl < kHeads; ++sl) v += sh.sums[w][sl * LANES + c][e];
        const Lane at(a, c);
        const int el = (e & 7) < 4 ? at.lo + (e & 3) : at.hi + (e & 3);
        partial[((int64_t)blockIdx.x * 2 + (e >> 3)) * a.dim + el] = v;
    }
}

// grad_weight[d] = sum of the blocks' partials: 32 strided runs in block order,
// then theirs.
__global__ void __launch_bounds__(1024)
norm_weight_reduce_kernel(const float* __restrict__ partial, int blocks, int dim,
                          float* __restrict__ gq, float* __restrict__ gk) {
    __shared__ float run[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float v = 0.f;
    if (col < 2 * dim) {
#pragma unroll 4
        for (int b = part; b < blocks; b += 32) v += partial[(int64_t)b * 2 * dim + col];
    }
    run[part][threadIdx.x & 31] = v;
    __syncthreads();
    if (part == 0 && col < 2 * dim) {
        for (int i = 1; i < 32; ++i) v += run[i][threadIdx.x & 31];
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
// As many blocks as are resident at once; a row's heads are shared out over
// several warps when there are fewer rows than half of the resident warps.
RotateGrid rotate_grid(const mpo_rotate& a, int per_sm) {
    RotateGrid g;
    g.lanes = rotate_lanes(a.dim);
    const int64_t rounds = ceil_div(a.heads > a.kv_heads ? a.heads : a.kv_heads, 32 / g.lanes);
    const int64_t warps = (int64_t)sm_count() * per_sm * kRotWarps;
    g.shares = (int)max64(1, min64(rounds, warps / (2 * max64(a.rows, 1))));
    g.blocks = (unsigned)max64(1, min64(ceil_div(a.rows * g.shares, kRotWarps),
                                        (int64_t)sm_count() * per_sm));
    return g;
}
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
    if (a->q_head < 0 || a->k_head < 0 || a->q_head > INT32_MAX || a->k_head > INT32_MAX)
        return bad("head strides must be in [0, 2^31)");
    if (a->rows == 0) return kOk;
    if (!a->q || !a->k || !a->out_q || !a->out_k) return bad("null pointer");
    if (a->pairs && (!a->position || !a->freqs)) return bad("null pointer");
    if (a->pairs && !aligned_to(a->freqs, 16)) return bad("freqs must be 16-byte aligned");
    if (a->position_float < MPO_POSITION_I32 || a->position_float > MPO_POSITION_I64)
        return bad("unknown position type");
    if (a->pairs && !aligned_to(a->position, a->position_float == MPO_POSITION_I64 ? 8 : 4))
        return bad("position must be aligned to its type");
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

// Calls f with the lane count as a compile-time constant.
template <typename F>
int with_lanes(int lanes, F&& f) {
    switch (lanes) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 4: return f(std::integral_constant<int, 4>());
        case 8: return f(std::integral_constant<int, 8>());
        case 16: return f(std::integral_constant<int, 16>());
        default: return f(std::integral_constant<int, 32>());
    }
}
template <typename T>
int run_rotate(const mpo_rotate& a, cudaStream_t s) {
    constexpr int kDepth = sizeof(T) == 2 ? 2 : 1;
    const RotateGrid g = rotate_grid(a, kFwdBlocksPerSm);
    return with_lanes(g.lanes, [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        if (a.interleaved) norm_rotate_kernel<T, kDepth, true, L><<<g.blocks, kRotThreads, 0, s>>>(a, g.shares);
        else norm_rotate_kernel<T, kDepth, false, L><<<g.blocks, kRotThreads, 0, s>>>(a, g.shares);
        return check_launch("norm_rotate_kernel");
    });
}
template <typename T>
int run_rotate_bwd(const mpo_rotate& a, cudaStream_t s) {
    constexpr int kDepth = sizeof(T) == 2 ? 2 : 1;
    const RotateGrid g = rotate_grid(a, kBwdBlocksPerSm);
    const bool weights = a.grad_q_weight || a.grad_k_weight;
    float* partial = weights ? static_cast<float*>(a.workspace) : nullptr;
    const int st = with_lanes(g.lanes, [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        if (a.interleaved)
            norm_rotate_bwd_kernel<T, kDepth, true, L><<<g.blocks, kRotThreads, 0, s>>>(a, g.shares, partial);
        else
            norm_rotate_bwd_kernel<T, kDepth, false, L><<<g.blocks, kRotThreads, 0, s>>>(a, g.shares, partial);
        return check_launch("norm_rotate_bwd_kernel");
    });
    if (st != kOk || !weights) return st;
    norm_weight_reduce_kernel<<<(unsigned)ceil_div(2 * a.dim, 32), 1024, 0, s>>>(
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
