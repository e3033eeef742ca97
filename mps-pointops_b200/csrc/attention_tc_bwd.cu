// Backward attention of serialised clouds for 16-bit types on the tensor cores
// (definitions: attention_common.cuh; operands: attention_tc.cuh).
//
// Two kernels form the scores again from q, k and the saved log-sum-exp: one
// owns 128 query rows and adds up dq (and the table's gradient), one owns 128
// key rows and adds up dk and dv over the query heads that share them.  Every
// sum has one owner and a fixed order, so results repeat and nothing is added
// through memory; the price, against one kernel that scatters dq, is that S and
// dP are formed twice, which the tensor cores have time for beside the
// exponentials.
//
// Per tile of 64 columns the tensor core forms S and dP in TMEM, a thread turns
// its row of them into 16-bit pairs of the score gradient (and of the weight)
// over the same columns, and these are the left operands of the accumulating
// products; those and the next tile's S and dP go out in one issue.
#include <string>

#include "attention_exact.cuh"
#include "attention_tc.cuh"

namespace mpo {
namespace {

// Shared memory that keeps a third block, which TMEM could not serve, off an SM.
constexpr size_t kTcPairBytes = 233472 / 3;

// ---------------------------------------------------------------- queries
// With the table's gradient and DP = 128, the lanes' cells (up to 128 KB) leave
// room for one stage of keys and values and one copy of the table.
template <int DP, bool GRAD_TABLE>
struct GradQShape {
    static constexpr bool kTight = GRAD_TABLE && DP == 128;
    static constexpr int kStages = kTight ? 1 : 2;
    static constexpr int kS = 0, kDP = kTcCols, kDQ = 2 * kTcCols, kCols = 256;
    static constexpr uint32_t kQ = 0, kG = TcTile<DP>::bytes(128), kStage = TcTile<DP>::bytes(64),
                              kK = 2 * kG, kV = kK + kStages * kStage, kPos = kV + kStages * kStage,
                              kBar = kPos + kStages * 3 * kTcCols * 4, kTable = kBar + 16;
    static constexpr int kBlocks = DP == 128 || GRAD_TABLE ? 1 : 2;
    static __host__ __device__ constexpr int table_words(int entries) {
        return kTight ? (entries + 3) / 4 * 4 : entries * 32;
    }
    static size_t bytes(int entries) {
        const size_t need = kTable + (size_t)table_words(entries) * 4 +
                            (GRAD_TABLE ? (size_t)entries * 512 : 0) + 1024;
        return need > kTcPairBytes ? need : kTcPairBytes;
    }
};

// Table gradient: every lane of every warp keeps its own cell of each entry
// ([warp][entry][lane], its own bank: a plain read, add and write, no atomics).
template <typename T, int DP, int BIAS, bool GRAD_TABLE>
__global__ void __launch_bounds__(kTcThreads, (GradQShape<DP, GRAD_TABLE>::kBlocks))
attn_tc_grad_q_kernel(const __grid_constant__ AttnArgs A, float* __restrict__ partial) {
    using Shape = GradQShape<DP, GRAD_TABLE>;
    constexpr int kStages = Shape::kStages;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31;
    const int h = blockIdx.y, hk = h / A.group;
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.q_tiles)[blockIdx.x];
    const int p = t.first + tid, entries = A.a.axes * A.a.buckets;
    int* kpos = reinterpret_cast<int*>(smem + Shape::kPos);
    float* table = reinterpret_cast<float*>(smem + Shape::kTable);
    float* hist = table + Shape::table_words(entries) + (tid >> 5) * entries * 32 + lane;  // this lane's cells
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + Shape::kBar + 8);

    if (tid < 32) tmem_alloc(smem_u32(slot), Shape::kCols);
    if (tid == 0) mbar_init(sb + Shape::kBar);
    const KeySpan span = key_span(A, t.first, t.first + t.rows - 1, t.lk, kTcCols);
    const int tiles = span.count();
    auto load_tile = [&](int i) {
        const int k0 = span.tile(i) * kTcCols, n = min(kTcCols, t.lk - k0);
        const int64_t row = (int64_t)t.other + k0;
        const uint32_t stage = (i % kStages) * Shape::kStage;
        tc_load<T, DP, kTcCols>(sb + Shape::kK + stage, A.a.k, row, n, hk, A.a.k_row, A.a.k_head, A.a.dim);
        tc_load<T, DP, kTcCols>(sb + Shape::kV + stage, A.a.v, row, n, hk, A.a.v_row, A.a.v_head, A.a.dim);
        if (BIAS) tc_load_pos(kpos + (i % kStages) * 3 * kTcCols, A.a.kpos, row, n, A.a.axes);
    };
    tc_load<T, DP, 128>(sb + Shape::kQ, A.a.q, t.row, t.rows, h, A.a.q_row, A.a.q_head, A.a.dim);
    tc_load<T, DP, 128>(sb + Shape::kG, A.a.grad_out, t.row, t.rows, h,
                        (int64_t)A.a.heads * A.a.dim, A.a.dim, A.a.dim);
    if (tiles > 0) load_tile(0);
    const bool live = tid < t.rows;
    const int64_t at = (((int64_t)t.row + tid) * A.a.heads + h) * A.a.dim;
    int qpos[3] = {0, 0, 0};
    if (BIAS) {
        if (Shape::kTight) {
            for (int e = tid; e < entries; e += kTcThreads) table[e] = table_entry(A.a, e, h) * kLog2e;
        } else {
            tc_load_table(A, table, h);
        }
        if (live)
            for (int a = 0; a < A.a.axes; ++a)
                qpos[a] = A.a.qpos[((int64_t)t.row + tid) * A.a.axes + a];
    }
    if (GRAD_TABLE)
        for (int e = 0; e < entries; ++e) hist[e * 32] = 0.f;
    const float lse2 = live ? load_lse2(A, t.row + tid, h) : INFINITY;
    tc_load_done();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t mine = tmem + ((uint32_t)(tid & ~31) << 16);
    Waiter done(sb + Shape::kBar, A.a.status);
    if (tid == 0 && tiles > 0) {
        mma_scores<T, DP, kTcCols>(tmem + Shape::kS, sb + Shape::kQ, sb + Shape::kK);
        mma_scores<T, DP, kTcCols>(tmem + Shape::kDP, sb + Shape::kG, sb + Shape::kV);
        mma_commit(sb + Shape::kBar);
    }
    float delta = 0.f;  // D = o . do
    if (live) {
        for (int c = 0; c * 8 < A.a.dim; ++c) {
            float g[8], o[8];
            Elem<T>::unpack(*reinterpret_cast<const uint4*>(smem + Shape::kG + TcTile<DP>::at(128, tid, c)), g);
            if (A.a.out_f32) {
                const float4* src = reinterpret_cast<const float4*>(A.a.out_f32 + at + c * 8);
                Elem<float>::unpack(reinterpret_cast<const uint4*>(src)[0], o);
                Elem<float>::unpack(reinterpret_cast<const uint4*>(src)[1], o + 4);
            } else {
                Elem<T>::unpack(*reinterpret_cast<const uint4*>(static_cast<const T*>(A.a.out) + at + c * 8), o);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(g[e], o[e], delta);
        }
        A.a.delta[(int64_t)h * A.a.q_rows + t.row + tid] = delta;
    }

    for (int i = 0; i < tiles; ++i) {
        done.wait();
        if (kStages == 2 && i + 1 < tiles) load_tile(i + 1);
        const int k0 = span.tile(i) * kTcCols, n = min(kTcCols, t.lk - k0);
        const bool whole = n == kTcCols && t.rows == 128 &&
                           all_visible(A, t.first, t.first + 127, k0, k0 + kTcCols - 1);
        const uint64_t seen = whole ? ~0ull : live ? seen_keys(A, p, k0, n) : 0ull;
        const int* kp = kpos + (i % kStages) * 3 * kTcCols;
#pragma unroll
        for (int c = 0; c < kTcCols; c += 16) {
            float s[16], dp[16];
            tmem_ld16(mine + Shape::kS + c, s);
            tmem_ld16(mine + Shape::kDP + c, dp);
            tmem_wait_ld();
            tmem_use(s);
            tmem_use(dp);
            int words[3][16];
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], A.scale_log2, -lse2);
            if (BIAS) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < A.a.axes) {
                        const float* tab = Shape::kTight ? table + a * A.a.buckets
                                                         : table + (a * A.a.buckets * 32 + lane);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const int4 k4 = *reinterpret_cast<const int4*>(kp + a * kTcCols + c + e);
                            words[a][e] = bucket_word<BIAS == 2>(A, k4.x - qpos[a]);
                            words[a][e + 1] = bucket_word<BIAS == 2>(A, k4.y - qpos[a]);
                            words[a][e + 2] = bucket_word<BIAS == 2>(A, k4.z - qpos[a]);
                            words[a][e + 3] = bucket_word<BIAS == 2>(A, k4.w - qpos[a]);
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[e] += tab[Shape::kTight ? words[a][e] >> 5 : words[a][e]];
                    }
            }
            const uint32_t bits = (uint32_t)(seen >> c);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float ds = exp2_sfu(s[e]) * (dp[e] - delta);
                s[e] = whole || ((bits >> e) & 1u) ? ds : 0.f;
            }
            if (GRAD_TABLE) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    // Cells of different axes are different: read the three, then write them.
                    float v[3];
#pragma unroll
                    for (int a = 0; a < 3; ++a)
                        if (a < A.a.axes) v[a] = hist[a * A.a.buckets * 32 + words[a][e]];
#pragma unroll
                    for (int a = 0; a < 3; ++a)
                        if (a < A.a.axes) hist[a * A.a.buckets * 32 + words[a][e]] = v[a] + s[e];
                }
            }
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = Elem<T>::two(s[2 * e], s[2 * e + 1]);
            tmem_st8(mine + Shape::kS + c / 2, w);  // over columns already read
        }
        tmem_wait_st();
        tc_load_done();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
            tc_fence_after();
            const uint32_t stage = (i % kStages) * Shape::kStage, next = Shape::kStage - stage;
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kDQ, tmem + Shape::kS, sb + Shape::kK + stage, i > 0);
            if (kStages == 2 && i + 1 < tiles) {
                mma_scores<T, DP, kTcCols>(tmem + Shape::kS, sb + Shape::kQ, sb + Shape::kK + next);
                mma_scores<T, DP, kTcCols>(tmem + Shape::kDP, sb + Shape::kG, sb + Shape::kV + next);
            }
            mma_commit(sb + Shape::kBar);
        }
        if (kStages == 1 && i + 1 < tiles) {
            done.wait();  // the keys are free
            load_tile(i + 1);
            tc_load_done();
            tc_fence_before();
            __syncthreads();
            if (tid == 0) {
                tc_fence_after();
                mma_scores<T, DP, kTcCols>(tmem + Shape::kS, sb + Shape::kQ, sb + Shape::kK);
                mma_scores<T, DP, kTcCols>(tmem + Shape::kDP, sb + Shape::kG, sb + Shape::kV);
                mma_commit(sb + Shape::kBar);
            }
        }
    }
    if (tiles > 0) done.wait();
    bool nan = false;
#pragma unroll
    for (int c = 0; c < DP; c += 16) {
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0.f;
        if (tiles > 0) {
            tmem_ld16(mine + Shape::kDQ + c, o);
            tmem_wait_ld();
            tmem_use(o);
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            o[e] *= A.a.scale;
            nan |= isnan(o[e]);
        }
#pragma unroll
        for (int e = 0; e < 16; e += 8)
            if (c + e < A.a.dim)
                *reinterpret_cast<uint4*>(static_cast<T*>(A.a.grad_q) + at + c + e) = Elem<T>::pack(o + e);
    }
    __syncwarp();
    for (unsigned bad = __ballot_sync(FULL_MASK, nan); bad; bad &= bad - 1) {
        const int r = (tid & ~31) + __ffs(bad) - 1;
        exact_grad_q_row<T>(A, (int64_t)t.row + r, t.first + r, t.other, t.lk, h);
    }
    tc_fence_before();
    __syncthreads();
    if (tid < 32) {
        tc_fence_after();
        tmem_free(tmem, Shape::kCols);
    }
    if (GRAD_TABLE)
        for (int e = tid; e < entries; e += kTcThreads) {
            float v = 0.f;
            const float* cells = table + Shape::table_words(entries);
            for (int w = 0; w < 4; ++w)
                for (int l = 0; l < 32; ++l) v += cells[(w * entries + e) * 32 + ((l + e) & 31)];
            partial[((int64_t)blockIdx.x * A.a.heads + h) * entries + e] = v;
        }
}

// ---------------------------------------------------------------- keys and values
template <int DP>
struct GradKvShape {
    static constexpr int kS = 0, kDP = kTcCols, kDK = 2 * kTcCols, kDV = kDK + DP;
    static constexpr int kCols = kDV + DP <= 256 ? 256 : 512;
    static constexpr int kBlocks = 512 / kCols;
    static constexpr uint32_t kK = 0, kV = TcTile<DP>::bytes(128), kStage = TcTile<DP>::bytes(64),
                              kQ = 2 * kV, kG = kQ + 2 * kStage, kRow = kG + 2 * kStage,
                              kPos = kRow + 2 * 2 * kTcCols * 4, kBar = kPos + 2 * 3 * kTcCols * 4,
                              kTable = kBar + 16;
    static size_t bytes(int entries) {
        const size_t need = kTable + (size_t)entries * 128 + 1024;
        return need > kTcPairBytes ? need : kTcPairBytes;
    }
};

// Key tiles that hold sinks are seen by every later query of their cloud.
// `shares` blocks divide those queries; each leaves its sums in `partial`
// ([cloud * sink tiles + tile][key head][share][dk, dv][128][dim], float32) for
// the join kernel.  shares == 1: no block does.
template <typename T, int DP, int BIAS>
__global__ void __launch_bounds__(kTcThreads, (GradKvShape<DP>::kBlocks))
attn_tc_grad_kv_kernel(const __grid_constant__ AttnArgs A, int shares, float* __restrict__ partial) {
    using Shape = GradKvShape<DP>;
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.k_tiles)[blockIdx.x];
    const bool shared = shares > 1 && t.first < A.a.sinks;
    if (!shared && blockIdx.z > 0) return;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31;
    const int hk = blockIdx.y, h0 = hk * A.group;
    const int j = t.first + tid;
    int* qpos = reinterpret_cast<int*>(smem + Shape::kPos);
    float* rows = reinterpret_cast<float*>(smem + Shape::kRow);  // [stage][lse2, D][64]
    float* table = reinterpret_cast<float*>(smem + Shape::kTable);
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + Shape::kBar + 8);

    if (tid < 32) tmem_alloc(smem_u32(slot), Shape::kCols);
    if (tid == 0) mbar_init(sb + Shape::kBar);
    int lo, hi;
    query_span(A, t.first, t.first + t.rows - 1, t.lq, t.lk, lo, hi);
    int first = 0, per = hi > lo ? (hi - lo + kTcCols - 1) / kTcCols : 0;
    if (shared) {
        first = (int)((int64_t)per * blockIdx.z / shares);
        per = (int)((int64_t)per * (blockIdx.z + 1) / shares) - first;
    }
    const int tiles = per * A.group;
    auto query0 = [&](int i) { return lo + (first + i % per) * kTcCols; };
    auto load_tile = [&](int i) {
        const int i0 = query0(i), n = min(kTcCols, hi - i0), h = h0 + i / per;
        const int64_t row = (int64_t)t.other + i0;
        const uint32_t stage = (i & 1) * Shape::kStage;
        tc_load<T, DP, kTcCols>(sb + Shape::kQ + stage, A.a.q, row, n, h, A.a.q_row, A.a.q_head, A.a.dim);
        tc_load<T, DP, kTcCols>(sb + Shape::kG + stage, A.a.grad_out, row, n, h,
                                (int64_t)A.a.heads * A.a.dim, A.a.dim, A.a.dim);
        float* dst = rows + (i & 1) * 2 * kTcCols;
        if (tid < kTcCols) {
            dst[tid] = tid < n ? load_lse2(A, row + tid, h) : INFINITY;
        } else {
            const int r = tid - kTcCols;
            dst[tid] = r < n ? A.a.delta[(int64_t)h * A.a.q_rows + row + r] : 0.f;
        }
        if (BIAS) tc_load_pos(qpos + (i & 1) * 3 * kTcCols, A.a.qpos, row, n, A.a.axes);
    };
    tc_load<T, DP, 128>(sb + Shape::kK, A.a.k, t.row, t.rows, hk, A.a.k_row, A.a.k_head, A.a.dim);
    tc_load<T, DP, 128>(sb + Shape::kV, A.a.v, t.row, t.rows, hk, A.a.v_row, A.a.v_head, A.a.dim);
    if (tiles > 0) load_tile(0);
    const bool live = tid < t.rows;
    int kpos[3] = {0, 0, 0};
    if (BIAS) {
        tc_load_table(A, table, h0);
        if (live)
            for (int a = 0; a < A.a.axes; ++a)
                kpos[a] = A.a.kpos[((int64_t)t.row + tid) * A.a.axes + a];
    }
    tc_load_done();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t mine = tmem + ((uint32_t)(tid & ~31) << 16);
    Waiter done(sb + Shape::kBar, A.a.status);
    if (tid == 0 && tiles > 0) {
        mma_scores<T, DP, kTcCols>(tmem + Shape::kS, sb + Shape::kK, sb + Shape::kQ);
        mma_scores<T, DP, kTcCols>(tmem + Shape::kDP, sb + Shape::kV, sb + Shape::kG);
        mma_commit(sb + Shape::kBar);
    }
    for (int i = 0; i < tiles; ++i) {
        if (BIAS && i > 0 && i % per == 0) {  // the next query head's table
            tc_load_table(A, table, h0 + i / per);
            __syncthreads();
        }
        done.wait();
        if (i + 1 < tiles) load_tile(i + 1);
        const int i0 = query0(i), n = min(kTcCols, hi - i0), p0 = i0 + t.lk - t.lq;
        const bool whole = n == kTcCols && t.rows == 128 &&
                           all_visible(A, p0, p0 + kTcCols - 1, t.first, t.first + 127);
        const uint64_t seen = whole ? ~0ull : live ? seeing_queries(A, j, p0, n) : 0ull;
        const int* qp = qpos + (i & 1) * 3 * kTcCols;
        const float* row = rows + (i & 1) * 2 * kTcCols;
#pragma unroll
        for (int c = 0; c < kTcCols; c += 16) {
            float s[16], dp[16];
            tmem_ld16(mine + Shape::kS + c, s);
            tmem_ld16(mine + Shape::kDP + c, dp);
            tmem_wait_ld();
            tmem_use(s);
            tmem_use(dp);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4 l = *reinterpret_cast<const float4*>(row + c + e);
                s[e] = fmaf(s[e], A.scale_log2, -l.x);
                s[e + 1] = fmaf(s[e + 1], A.scale_log2, -l.y);
                s[e + 2] = fmaf(s[e + 2], A.scale_log2, -l.z);
                s[e + 3] = fmaf(s[e + 3], A.scale_log2, -l.w);
                const float4 d = *reinterpret_cast<const float4*>(row + kTcCols + c + e);
                dp[e] -= d.x;
                dp[e + 1] -= d.y;
                dp[e + 2] -= d.z;
                dp[e + 3] -= d.w;
            }
            if (BIAS) {
#pragma unroll
                for (int a = 0; a < 3; ++a)
                    if (a < A.a.axes) {
                        const float* tab = table + (a * A.a.buckets * 32 + lane);
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const int4 q4 = *reinterpret_cast<const int4*>(qp + a * kTcCols + c + e);
                            s[e] += tab[bucket_word<BIAS == 2>(A, kpos[a] - q4.x)];
                            s[e + 1] += tab[bucket_word<BIAS == 2>(A, kpos[a] - q4.y)];
                            s[e + 2] += tab[bucket_word<BIAS == 2>(A, kpos[a] - q4.z)];
                            s[e + 3] += tab[bucket_word<BIAS == 2>(A, kpos[a] - q4.w)];
                        }
                    }
            }
            const uint32_t bits = (uint32_t)(seen >> c);
            uint32_t w[8], g[8];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool on = whole || ((bits >> e) & 1u);
                s[e] = on ? exp2_sfu(s[e]) : 0.f;
                dp[e] = on ? s[e] * dp[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = Elem<T>::two(s[2 * e], s[2 * e + 1]);
                g[e] = Elem<T>::two(dp[2 * e], dp[2 * e + 1]);
            }
            tmem_st8(mine + Shape::kS + c / 2, w);
            tmem_st8(mine + Shape::kDP + c / 2, g);
        }
        tmem_wait_st();
        tc_load_done();
        tc_fence_before();
        __syncthreads();
        if (tid == 0) {
            tc_fence_after();
            const uint32_t stage = (i & 1) * Shape::kStage, next = Shape::kStage - stage;
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kDV, tmem + Shape::kS, sb + Shape::kG + stage, i > 0);
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kDK, tmem + Shape::kDP, sb + Shape::kQ + stage, i > 0);
            if (i + 1 < tiles) {
                mma_scores<T, DP, kTcCols>(tmem + Shape::kS, sb + Shape::kK, sb + Shape::kQ + next);
                mma_scores<T, DP, kTcCols>(tmem + Shape::kDP, sb + Shape::kV, sb + Shape::kG + next);
            }
            mma_commit(sb + Shape::kBar);
        }
    }
    if (tiles > 0) done.wait();
    bool nan = false;
    const int64_t at = (((int64_t)t.row + tid) * A.a.kv_heads + hk) * A.a.dim;
    const int sink_tiles = (A.a.sinks + kAttnTile - 1) / kAttnTile;
    float* sums = nullptr;
    if (shared) {
        const int64_t tile = (int64_t)t.cloud * sink_tiles + t.first / kAttnTile;
        sums = partial + (((tile * A.a.kv_heads + hk) * shares + blockIdx.z) * 2 * kAttnTile + tid) * A.a.dim;
    }
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int c = 0; c < DP; c += 16) {
            float o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
            if (tiles > 0) {
                tmem_ld16(mine + (which ? Shape::kDV : Shape::kDK) + c, o);
                tmem_wait_ld();
                tmem_use(o);
            }
            if (!live) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (!which) o[e] *= A.a.scale;
                nan |= isnan(o[e]);
            }
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                if (c + e >= A.a.dim) continue;
                if (sums) {
                    float4* dst = reinterpret_cast<float4*>(sums + (int64_t)which * kAttnTile * A.a.dim + c + e);
                    dst[0] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    dst[1] = make_float4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
                } else {
                    *reinterpret_cast<uint4*>(static_cast<T*>(which ? A.a.grad_v : A.a.grad_k) + at + c + e) =
                        Elem<T>::pack(o + e);
                }
            }
        }
    __syncwarp();
    if (!shared)
        for (unsigned bad = __ballot_sync(FULL_MASK, nan); bad; bad &= bad - 1) {
            const int r = (tid & ~31) + __ffs(bad) - 1;
            exact_grad_kv_row<T>(A, t.base, t.first + r, t.other, t.lq, t.lk, hk);
        }
    tc_fence_before();
    __syncthreads();
    if (tid < 32) {
        tc_fence_after();
        tmem_free(tmem, Shape::kCols);
    }
}

// grad_k and grad_v of the key tiles with sinks: the shares' sums in order.  A
// warp per key row.
template <typename T>
__global__ void __launch_bounds__(256)
attn_tc_join_kv_kernel(const __grid_constant__ AttnArgs A, int shares, const float* __restrict__ partial) {
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.k_tiles)[blockIdx.x];
    if (t.first >= A.a.sinks) return;
    const int r = blockIdx.z * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, hk = blockIdx.y;
    if (r >= t.rows) return;
    const int sink_tiles = (A.a.sinks + kAttnTile - 1) / kAttnTile;
    const int64_t tile = (int64_t)t.cloud * sink_tiles + t.first / kAttnTile;
    const float* src = partial + (((tile * A.a.kv_heads + hk) * shares) * 2 * kAttnTile + r) * A.a.dim;
    const int64_t at = (((int64_t)t.row + r) * A.a.kv_heads + hk) * A.a.dim, half = (int64_t)kAttnTile * A.a.dim;
    bool nan = false;
    for (int d = lane; d < A.a.dim; d += 32) {
        float dk = 0.f, dv = 0.f;
        for (int z = 0; z < shares; ++z) {
            dk += src[z * 2 * half + d];
            dv += src[(z * 2 + 1) * half + d];
        }
        nan |= isnan(dk) | isnan(dv);
        static_cast<T*>(A.a.grad_k)[at + d] = Elem<T>::from(dk);
        static_cast<T*>(A.a.grad_v)[at + d] = Elem<T>::from(dv);
    }
    if (__any_sync(FULL_MASK, nan))
        exact_grad_kv_row<T>(A, t.base, t.first + r, t.other, t.lq, t.lk, hk);
}

// Blocks that share a key tile with sinks: each about as many queries as see
// any other key tile, but no more blocks than fill the GPU (eight per SM).
int sink_shares(const AttnArgs& A) {
    if (A.a.sinks == 0) return 1;
    const int64_t window = (int64_t)A.left + A.right + kAttnTile;
    const int64_t tiles = (int64_t)A.a.clouds * ceil_div(A.a.sinks, kAttnTile) * A.a.kv_heads;
    return (int)max64(1, min64(A.a.max_rows / window, ceil_div(8 * sm_count(), max64(tiles, 1))));
}
size_t sink_bytes(const AttnArgs& A) {
    const int shares = sink_shares(A);
    if (shares == 1) return 0;
    const int64_t tiles = (int64_t)A.a.clouds * ceil_div(A.a.sinks, kAttnTile);
    return (size_t)(tiles * A.a.kv_heads * shares * 2 * kAttnTile * A.a.dim) * sizeof(float);
}

template <typename T, int DP, int BIAS, bool GRAD_TABLE>
int run_q(const AttnArgs& A, float* partial, cudaStream_t s) {
    const size_t bytes = GradQShape<DP, GRAD_TABLE>::bytes(BIAS ? A.a.axes * A.a.buckets : 0);
    const int st = tc_prepare(attn_tc_grad_q_kernel<T, DP, BIAS, GRAD_TABLE>, bytes, "attn_tc_grad_q_kernel");
    if (st != kOk) return st;
    const dim3 grid((unsigned)A.a.q_tile_count, (unsigned)A.a.heads);
    attn_tc_grad_q_kernel<T, DP, BIAS, GRAD_TABLE><<<grid, kTcThreads, bytes, s>>>(A, partial);
    return check_launch("attn_tc_grad_q_kernel");
}
template <typename T, int DP, int BIAS>
int run_kv(const AttnArgs& A, float* partial, cudaStream_t s) {
    const size_t bytes = GradKvShape<DP>::bytes(BIAS ? A.a.axes * A.a.buckets : 0);
    int st = tc_prepare(attn_tc_grad_kv_kernel<T, DP, BIAS>, bytes, "attn_tc_grad_kv_kernel");
    if (st != kOk) return st;
    const int shares = sink_shares(A);
    dim3 grid((unsigned)A.a.k_tile_count, (unsigned)A.a.kv_heads, (unsigned)shares);
    attn_tc_grad_kv_kernel<T, DP, BIAS><<<grid, kTcThreads, bytes, s>>>(A, shares, partial);
    st = check_launch("attn_tc_grad_kv_kernel");
    if (st != kOk || shares == 1) return st;
    grid.z = kAttnTile / 8;
    attn_tc_join_kv_kernel<T><<<grid, 256, 0, s>>>(A, shares, partial);
    return check_launch("attn_tc_join_kv_kernel");
}
template <typename T, int DP, int BIAS>
int run(const AttnArgs& A, cudaStream_t s) {
    float* sums = static_cast<float*>(A.a.workspace);
    int st = kOk;
    if (A.a.q_tile_count) {
        if constexpr (BIAS != 0) {
            float* partial = reinterpret_cast<float*>(static_cast<unsigned char*>(A.a.workspace) + sink_bytes(A));
            st = A.a.grad_table ? run_q<T, DP, BIAS, true>(A, partial, s) : run_q<T, DP, BIAS, false>(A, nullptr, s);
        } else {
            st = run_q<T, DP, BIAS, false>(A, nullptr, s);
        }
    }
    if (st == kOk && A.a.k_tile_count) st = run_kv<T, DP, BIAS>(A, sums, s);
    return st;
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

size_t attn_tc_backward_bytes(const AttnArgs& A) { return sink_bytes(A); }
int attn_tc_backward(const AttnArgs& A, cudaStream_t s) {
    return A.a.dtype == MPO_F16 ? by_dim<__half>(A, s) : by_dim<__nv_bfloat16>(A, s);
}

}  // namespace mpo
