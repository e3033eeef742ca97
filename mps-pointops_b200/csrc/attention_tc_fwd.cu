// Forward attention of serialised clouds for 16-bit types on the tensor cores
// (definitions: attention_common.cuh; operands: attention_tc.cuh).
//
// A block owns 128 query rows of one head, one thread per row, and a warp that
// issues copies and products.  It streams the
// visible key tiles (64 keys) through two shared-memory stages.  Per tile the
// tensor core forms S = Q K^T into TMEM; a thread reads its row of scores,
// carries the running maximum and sum of the softmax, writes its weights back
// over S as 16-bit pairs, and the tensor core adds P V to the rows in TMEM,
// followed in the same issue by the next tile's S.  The rows in TMEM are
// rescaled only when a row's maximum grew by more than 2^8 since its last
// rescale: weights then reach 256, which costs a 16-bit float no precision.
//
// Bound by the latency of the softmax between two products, with the
// exponentials behind it (60 % of their unit): 131 us for 8 clouds of 4096
// points, 8 heads of 64, window 1024 (490 TFLOP/s; the products alone 38 us, the
// exponentials 56).  With a table its look-ups bind, 45 % of shared memory and of
// the issue slots at once: 728 us for 8 x 8192.  At 128 elements two buffers of S hide
// more of the latency: 183 us with one, 159 with two (5 ragged clouds of up to 4099
// points, 16 heads over 4, window 1024, causal).
#include <string>

#include "attention_exact.cuh"
#include "attention_tc.cuh"

namespace mpo {
namespace {

constexpr int kFwdThreads = kTcRows + 32;
template <int DP>
struct FwdShape {
    // Rows of 128 elements leave TMEM for a second buffer of S at the same two blocks per SM:
    // S of tile i + 1 is then formed beside the softmax of tile i.
    static constexpr int kBuffers = DP == 128 ? 2 : 1;
    static constexpr int kS = 0, kO = kBuffers * kTcCols;  // TMEM columns
    static constexpr int kCols = kO + DP <= 128 ? 128 : 256;
    static constexpr int kBlocks = 512 / kCols;
    static constexpr uint32_t kQ = 0, kK = TcTile<DP>::bytes(128), kStage = TcTile<DP>::bytes(64),
                              kV = kK + 2 * kStage, kPos = kV + 2 * kStage,
                              kBar = kPos + 3 * 3 * kTcCols * 4, kTable = kBar + 64;
    // Barriers: products (2); stages of keys (2) and values (2), the first keys with Q.
    static constexpr uint32_t kFullK = kBar + 16, kFullV = kBar + 32, kSlot = kBar + 48;
    static size_t bytes(int entries) {
        // At least what keeps more blocks than TMEM serves off an SM (they would wait for it).
        const size_t need = kTable + (size_t)entries * 128 + 1024;
        const size_t least = 233472 / (kBlocks + 1);
        return need > least ? need : least;
    }
};

// One thread per row: two threads of 32 columns each, with S in two buffers at two
// blocks per SM, took 147 against 130 us (8 clouds of 4096 points, 8 heads of 64)
// and 839 against 726 us (8 x 8192 with a table); four blocks per SM at 96
// registers 139 us against three.
template <typename T, int DP, int BIAS>
__global__ void __launch_bounds__(kFwdThreads, (DP <= 64 ? 3 : FwdShape<DP>::kBlocks))
attn_tc_fwd_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TcMaps M) {
    using Shape = FwdShape<DP>;
    constexpr int kBuffers = Shape::kBuffers;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x;
    const int h = blockIdx.y, hk = h / A.group;
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.q_tiles)[blockIdx.x];
    const int p = t.first + tid;
    float* kpos = reinterpret_cast<float*>(smem + Shape::kPos);
    float* table = reinterpret_cast<float*>(smem + Shape::kTable);
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + Shape::kSlot);

    const KeySpan span = key_span(A, t.first, t.first + t.rows - 1, t.lk, kTcCols);
    const int tiles = (int)uniform((uint32_t)span.count());

    if (tid >= kTcRows) {  // the warp that feeds the tensor core
        tmem_alloc(smem_u32(slot), Shape::kCols);
        auto load_keys = [&](int i) {
            if (i >= tiles) return;
            const uint32_t bar = sb + Shape::kFullK + 8 * (i & 1);
            tma_expect(bar, Shape::kStage + (i == 0 ? Shape::kK : 0));
            if (i == 0) tma_rows<DP, 128>(sb + Shape::kQ, &M.q, h, t.row, bar);
            tma_rows<DP, kTcCols>(sb + Shape::kK + (i & 1) * Shape::kStage, &M.k, hk,
                                  t.other + span.tile(i) * kTcCols, bar);
        };
        auto load_values = [&](int i) {
            if (i >= tiles) return;
            const uint32_t bar = sb + Shape::kFullV + 8 * (i & 1);
            tma_expect(bar, Shape::kStage);
            tma_rows<DP, kTcCols>(sb + Shape::kV + (i & 1) * Shape::kStage, &M.v, hk,
                                  t.other + span.tile(i) * kTcCols, bar);
        };
        Patience patience(A.a.status);
        uint32_t tmem = 0;
        auto scores = [&](int i) {
            if (i >= tiles) return;
            patience.wait(sb + Shape::kFullK + 8 * (i & 1), (i >> 1) & 1);
            mma_scores<T, DP, kTcCols>(tmem + Shape::kS + (i & (kBuffers - 1)) * kTcCols, sb + Shape::kQ,
                                       sb + Shape::kK + (i & 1) * Shape::kStage);
        };
        if ((tid & 31) == 0)
            for (int i = 0; i < 6; ++i) mbar_init(sb + Shape::kBar + 8 * i);
        __syncwarp();
        load_keys(0);
        load_values(0);
        load_keys(1);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = uniform(*slot);
        // Step i commits to barrier i mod kBuffers; the prologue stands for the kBuffers steps
        // before step 0.
        scores(0);
        mma_commit(sb + Shape::kBar);
        if (kBuffers == 2) {
            scores(1);
            mma_commit(sb + Shape::kBar + 8);
        }
        patience.wait(sb + Shape::kBar, 0);  // S of tile 0: the first keys' stage is free
        load_keys(2);
        load_values(1);
        for (int i = 0; i < tiles; ++i) {
            __syncthreads();  // the weights of tile i are in TMEM
            tc_fence_after();
            patience.wait(sb + Shape::kFullV + 8 * (i & 1), (i >> 1) & 1);
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kO, tmem + Shape::kS + (i & (kBuffers - 1)) * kTcCols,
                                         sb + Shape::kV + (i & 1) * Shape::kStage, i > 0);
            // Issued after P V and executed in order after it: S may overwrite the weights.
            scores(i + kBuffers);
            mma_commit(sb + Shape::kBar + 8 * (i & (kBuffers - 1)));
            if (kBuffers == 1) {
                // S of tile i + 1 and P V of tile i are done: their operands' stages are free.
                // Copies get until the end of the next step.
                patience.wait(sb + Shape::kBar, (i + 1) & 1);
                load_keys(i + 3);
                load_values(i + 2);
            } else {
                // Those of step i - 1: S of tile i + 1 and P V of tile i - 1.
                patience.wait(sb + Shape::kBar + 8 * ((i - 1) & 1), ((i + 1) >> 1) & 1);
                load_keys(i + 3);
                if (i > 0) load_values(i + 1);
            }
        }
        tc_fence_before();
        __syncthreads();  // the rows have been read
        tc_fence_after();
        tmem_free(tmem, Shape::kCols);
        return;
    }

    BiasRow bias;
    if (BIAS) bias.init(A, A.a.qpos, t.row, tid, t.rows, sb + Shape::kTable, 1);
    auto first_key = [&](int i, int& k0, int& n) {
        k0 = span.tile(i) * kTcCols;
        n = min(kTcCols, t.lk - k0);
    };
    Columns columns;
    auto fetch_columns = [&](int i) {
        if (!BIAS || i >= tiles) return;
        int k0, n;
        first_key(i, k0, n);
        columns.fetch(A.a.kpos, (int64_t)t.other + k0, n, A.a.axes);
    };
    auto store_columns = [&](int i) {
        if (!BIAS || i >= tiles) return;
        int k0, n;
        first_key(i, k0, n);
        columns.store(kpos + (i % 3) * 3 * kTcCols, n, A.a.axes, bias, 1);
    };
    fetch_columns(0);
    if (BIAS) tc_load_table(A, table, h);
    store_columns(0);
    fetch_columns(1);
    store_columns(1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t mine = tmem + ((uint32_t)(tid & ~31) << 16);  // this warp's lanes
    Waiters<kBuffers> done(sb + Shape::kBar, A.a.status);

    // Running maximum in units of s2 = S * mul + bias (log2), as of the last rescale.
    float top = -INFINITY, sum = 0.f;
    const float mul = BIAS ? 1.f : (A.scale_log2 > 0.f ? A.scale_log2 : 1.f);
    for (int i = 0; i < tiles; ++i) {
        done.wait(i);
        fetch_columns(i + 2);
        const uint32_t scored = mine + Shape::kS + (i & (kBuffers - 1)) * kTcCols;
        float s[kTcCols];
#pragma unroll
        for (int c = 0; c < kTcCols; c += 16) tmem_ld16(scored + c, s + c);
        tmem_wait_ld();
        tmem_use(s);
        int k0, n;
        first_key(i, k0, n);
        if (BIAS) {
            const float* cols = kpos + (i % 3) * 3 * kTcCols;
            const f32x2 scale2 = pack2(A.scale_log2, A.scale_log2);
#pragma unroll
            for (int c = 0; c < kTcCols; c += 16) {
                f32x2 b[8];
                bias_of<BIAS == 2, false, 16>(A, bias, cols + c, b, nullptr, h);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    unpack2(fma2(pack2(s[c + 2 * e], s[c + 2 * e + 1]), scale2, b[e]), s[c + 2 * e],
                            s[c + 2 * e + 1]);
            }
        } else if (!(A.scale_log2 > 0.f)) {
#pragma unroll
            for (int c = 0; c < kTcCols; ++c) s[c] *= A.scale_log2;
        }
        if (n < kTcCols || !all_visible(A, t.first, t.first + t.rows - 1, k0, k0 + kTcCols - 1)) {
            const uint64_t seen = seen_keys(A, p, k0, n);
            const uint32_t lo = (uint32_t)seen, hi = (uint32_t)(seen >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                s[c] = (lo >> c) & 1u ? s[c] : -INFINITY;
                s[c + 32] = (hi >> c) & 1u ? s[c + 32] : -INFINITY;
            }
        }
        float m[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < 60; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = fmax3(m[e], s[c + e], s[c + 4 + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = fmaxf(m[e], s[60 + e]);
        const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        // (most - top) is NaN only when both are the same infinity: no growth.
        const bool grow = (most - top) * mul > 8.f;
        if (__any_sync(FULL_MASK, grow)) {
            float f = 1.f;
            if (grow) {
                f = exp2_sfu((top - most) * mul);
                top = most;
                sum *= f;
            }
            if (i > 0) {
                if (kBuffers == 2) {  // P V of tile i - 1 still adds to the rows
                    done.even.patience.wait(sb + Shape::kBar + 8 * ((i - 1) & 1), ((i + 1) >> 1) & 1);
                    tc_fence_after();
                }
#pragma unroll
                for (int c = 0; c < DP; c += 16) {
                    float o[16];
                    tmem_ld16(mine + Shape::kO + c, o);
                    tmem_wait_ld();
                    tmem_use(o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] *= f;
                    tmem_st16(mine + Shape::kO + c, reinterpret_cast<const uint32_t*>(o));
                }
            }
        }
        const float ref = top == -INFINITY ? 0.f : -top * mul;
        f32x2 part[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        const f32x2 mul2v = pack2(mul, mul), ref2 = pack2(ref, ref);
#pragma unroll
        for (int c = 0; c < kTcCols; c += 16) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                float a, b;
                unpack2(fma2(pack2(s[c + e], s[c + e + 1]), mul2v, ref2), a, b);
                a = exp2_sfu(a);
                b = exp2_sfu(b);
                part[(e >> 1) & 1] = add2(part[(e >> 1) & 1], pack2(a, b));
                w[e / 2] = Elem<T>::two(a, b);
            }
            tmem_st8(scored + c, w);
        }
        {
            float a, b;
            unpack2(add2(part[0], part[1]), a, b);
            sum += a + b;
        }
        store_columns(i + 2);
        tmem_wait_st();
        tc_fence_before();
        __syncthreads();
    }
    done.wait(tiles);
    if (kBuffers == 2) done.wait(tiles + 1);
    const bool live = tid < t.rows;
    const bool far = BIAS && live && bias.far;
    bool nan = far;
    const int64_t at = (((int64_t)t.row + tid) * A.a.heads + h) * A.a.dim;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int c = 0; c < DP; c += 16) {
        float o[16];
        if (tiles > 0) {
            tmem_ld16(mine + Shape::kO + c, o);
            tmem_wait_ld();
            tmem_use(o);
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            o[e] = sum == 0.f ? (isnan(o[e]) && tiles > 0 ? o[e] : 0.f) : o[e] * inv;
            nan |= isnan(o[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            if (c + e >= A.a.dim) continue;
            *reinterpret_cast<uint4*>(static_cast<T*>(A.a.out) + at + c + e) = Elem<T>::pack(o + e);
        }
    }
    if (live && A.a.lse)
        A.a.lse[(int64_t)h * A.a.q_rows + t.row + tid] =
            sum == 0.f ? -INFINITY : fmaf(top * mul, kLn2, logf(sum));
    __syncwarp();
    const unsigned apart = __ballot_sync(FULL_MASK, far);
    for (unsigned bad = __ballot_sync(FULL_MASK, nan); bad; bad &= bad - 1) {
        const int b = __ffs(bad) - 1, r = (tid & ~31) + b;
        exact_forward_row<T>(A, (int64_t)t.row + r, t.first + r, t.other, t.lk, h, (apart >> b) & 1u);
    }
    tc_fence_before();
    __syncthreads();
}

template <typename T, int DP, int BIAS>
int run(const AttnArgs& A, cudaStream_t s) {
    const size_t bytes = FwdShape<DP>::bytes(BIAS ? A.a.axes * A.a.buckets : 0);
    const int st = attn_prepare<&attn_tc_fwd_kernel<T, DP, BIAS>>("attn_tc_fwd_kernel");
    if (st != kOk) return st;
    TcMaps maps = {};
    const int mapped = make_maps<DP>(maps, A, false);
    if (mapped != kOk) return mapped;
    const dim3 grid((unsigned)A.a.q_tile_count, (unsigned)A.a.heads);
    attn_tc_fwd_kernel<T, DP, BIAS><<<grid, kFwdThreads, bytes, s>>>(A, maps);
    return check_launch("attn_tc_fwd_kernel");
}
template <typename T, int DP>
int by_bias(const AttnArgs& A, cudaStream_t s) {
    if (!A.a.table) return run<T, DP, 0>(A, s);
    return A.a.map ? run<T, DP, 2>(A, s) : run<T, DP, 1>(A, s);
}
template <typename T>
int by_dim(const AttnArgs& A, cudaStream_t s) {
    if (A.a.dim <= 16) return by_bias<T, 16>(A, s);
    if (A.a.dim <= 32) return by_bias<T, 32>(A, s);
    if (A.a.dim <= 64) return by_bias<T, 64>(A, s);
    return by_bias<T, 128>(A, s);
}

}  // namespace

int attn_tc_forward(const AttnArgs& A, cudaStream_t s) {
    return A.a.dtype == MPO_F16 ? by_dim<__half>(A, s) : by_dim<__nv_bfloat16>(A, s);
}

}  // namespace mpo
