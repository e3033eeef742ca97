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
// Per tile of 64 columns the tensor core forms S and dP in TMEM, the threads of a
// row turn them into 16-bit pairs of the score gradient (and of the weight) over
// the same columns, and these are the left operands of the accumulating products.
//
// 8 clouds of 8192 points, 8 heads of 64, window 1024, a table of 3 x 63 entries:
// keys and values 904 us, D alone 733 us, dq and the table 1607 us (880 of them its
// cells: shared memory at 59 % and the issue slots at 57 % of their peaks bind).
// Without a table, 5 ragged clouds of up to 4099 points, 16 heads of 128 over 4:
// keys and values 287 us, queries 285 us, tensor memory busy for 59 and 44 % of the
// cycles; latency at one block per SM binds.
#include <string>

#include "attention_shares.cuh"
#include "attention_tc.cuh"

namespace mpo {
namespace {

// ---------------------------------------------------------------- queries
// What the query kernel forms.  kGradQ: dq, with D = o . do from the stored
// result.  For the table's gradient, which is kept in float32, D has to be the
// sum over the pairs of the very weights and dP that it is subtracted from:
// stored and tensor-core results are off by 2e-3 and (sums rounded towards zero)
// 3e-6 of it, always the same way for all pairs of a row (in dq and dk, which round each
// score gradient to 16 bits anyway, the stored result's share is 0.0003 to 0.001 of their norm
// beside 0.0024 for bf16).  kDelta forms D = sum
// P dP in float32 first; kGradQTable then forms dq and the table's gradient.
enum QueryMode { kGradQ = 0, kDelta = 1, kGradQTable = 2 };

// Threads: NG groups of 128; thread `row` of each group shares the row and takes
// 64 / NG columns of every tile, so that 16 warps are on an SM (one thread per
// row left 4 to 8, and most of the time went to fixed latencies).  A further warp
// issues the copies and the products: a computing warp that did was held up by
// the tensor core's queue, 2400 of 4300 cycles of a step at D = 128, and the
// others with it at the next barrier.
//
// Where shared memory and TMEM serve two blocks per SM (DP <= 64, no cells), each
// has NG = 2 and one buffer of S and dP, and the blocks fill each other's gaps.
// Else one block has NG = 4 and two buffers: at the end of step i the tensor core
// gets dq += dS_i K_i and then, over the buffer that this frees, S and dP of tile
// i + 2, so those of tile i + 1 are ready when the step's barrier falls.
//
// Table gradient: a thread may only add to cells that no other adds to, so lane
// l of quarter w (rows 32 w ..) has its own cell of each entry ([w][entry][l],
// its own bank: a plain read, add and write, no atomics), and group a keeps
// those of axis a: the groups leave their score gradients in TMEM as float32
// (two buffers), and after the tile's barrier group a adds all 64 columns of
// them to its axis.  A group that keeps cells forms 8 columns of a tile itself, the
// others the rest, so that both take about as long; the pairs then have columns of
// their own in TMEM.  With DP = 128 the cells (up to 128 KB) leave room for one
// stage of keys and values, one buffer of S and dP, and one copy of the table.
template <int DP, int MODE>
struct QueryShape {
    static constexpr bool kCells = MODE == kGradQTable, kTight = kCells && DP == 128;
    static constexpr int kBlocks = kCells || DP == 128 ? 1 : 2, kGroups = 4 / kBlocks;
    static constexpr int kCompute = kGroups * kTcRows, kThreads = kCompute + 32, kPer = kTcCols / kGroups;
    static constexpr int kBuffers = kTight || kBlocks == 2 ? 1 : 2;
    // Keys serve S and dq of their tile, values dP alone.
    static constexpr int kKStages = kTight ? 1 : 2 + kBuffers, kVStages = kTight ? 1 : 2;
    static constexpr int kPosStages = kTight ? 3 : 4;
    static constexpr int kS = 0, kDP = kTcCols, kBuffer = (kBuffers - 1) * 2 * kTcCols;  // TMEM columns
    static constexpr int kDQ = 2 * kTcCols + kBuffer;
    static constexpr int kDS = kDQ + DP, kP = kDS + 2 * kTcCols;  // cells: two buffers each
    static constexpr int kCols = kBlocks == 2 ? 256 : 512;
    static_assert(!kCells || kP + kTcCols <= kCols, "TMEM");
    static constexpr uint32_t kQ = 0, kG = TcTile<DP>::bytes(128), kStage = TcTile<DP>::bytes(64),
                              kK = 2 * kG, kV = kK + kKStages * kStage, kBar = kV + kVStages * kStage,
                              kTable = kBar + 128;
    // Barriers: products (2); stages of keys (4), values (2), Q and dO; then TMEM's address, row flags.
    static constexpr uint32_t kFullK = kBar + 16, kFullV = kBar + 48, kFullQ = kBar + 64, kSlot = kBar + 72,
                              kFlags = kBar + 80;
    static constexpr int kAhead = kTight ? 1 : 2;  // steps from the fetch of a tile's positions to their use
    static constexpr int kTightEntries = 248;  // the table fits beside this many cells (DP = 128)
    static __host__ __device__ constexpr int table_words(int entries, bool one) {
        return !one ? entries * 32 : kTight && entries > kTightEntries ? 0 : (entries + 3) / 4 * 4;
    }
    static __host__ __device__ constexpr int pos_words(int axes) { return kPosStages * axes * kTcCols; }
    static size_t bytes(int axes, int entries, bool one) {
        size_t need = kTable + (size_t)(pos_words(axes) + table_words(entries, one)) * 4 +
                      (kCells ? (size_t)entries * 512 : 0) + 1024;
        if (MODE == kDelta && need < kTable + 4 * kCompute + 1024) need = kTable + 4 * kCompute + 1024;
        const size_t least = 233472 / (kBlocks + 1);  // no more blocks than TMEM serves
        return need > least ? need : least;
    }
    // One copy of the table where a copy per lane does not fit beside the cells.
    static bool one_copy(int axes, int entries) { return kTight || bytes(axes, entries, false) > kAttnSmem; }
};

template <typename T, int DP, int BIAS, int MODE, bool ONE>
__global__ void __launch_bounds__((QueryShape<DP, MODE>::kThreads), (QueryShape<DP, MODE>::kBlocks))
attn_tc_query_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TcMaps M,
                     float* __restrict__ partial) {
    using Shape = QueryShape<DP, MODE>;
    constexpr int kPer = Shape::kPer, kBuffers = Shape::kBuffers;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, r = tid & 127, quarter = r >> 5, group = tid >> 7;
    const int h = blockIdx.y, hk = h / A.group;
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.q_tiles)[blockIdx.x];
    const int p = t.first + r, entries = A.a.axes * A.a.buckets;
    // After the barriers: the table, the cells ([quarter][entry][lane]), the columns' positions.
    float* table = reinterpret_cast<float*>(smem + Shape::kTable);
    float* all_cells = table + Shape::table_words(entries, ONE);
    float* cells = all_cells + quarter * entries * 32;  // this quarter's
    float* kpos = reinterpret_cast<float*>(all_cells + (Shape::kCells ? entries * 128 : 0));
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + Shape::kSlot);
    unsigned* flags = reinterpret_cast<unsigned*>(smem + Shape::kFlags);  // rows to form again
    const KeySpan span = key_span(A, t.first, t.first + t.rows - 1, t.lk, kTcCols);
    const int tiles = (int)uniform((uint32_t)span.count());

    if (tid >= Shape::kCompute) {  // the warp that feeds the tensor core
        tmem_alloc(smem_u32(slot), Shape::kCols);
        auto full_k = [&](int i) { return sb + Shape::kFullK + 8 * (i % Shape::kKStages); };
        auto full_v = [&](int i) { return sb + Shape::kFullV + 8 * (i % Shape::kVStages); };
        auto load_tile = [&](int i) {
            if (i >= tiles) return;
            const int row = t.other + span.tile(i) * kTcCols;
            tma_expect(full_k(i), Shape::kStage);
            tma_rows<DP, kTcCols>(sb + Shape::kK + (i % Shape::kKStages) * Shape::kStage, &M.k, hk, row, full_k(i));
            tma_expect(full_v(i), Shape::kStage);
            tma_rows<DP, kTcCols>(sb + Shape::kV + (i % Shape::kVStages) * Shape::kStage, &M.v, hk, row, full_v(i));
        };
        Patience patience(A.a.status);
        uint32_t tmem = 0;
        auto scores = [&](int i) {  // S and dP of tile i into its buffer
            if (i >= tiles) return;
            const uint32_t buffer = tmem + (i & (kBuffers - 1)) * Shape::kBuffer;
            patience.wait(full_k(i), (i / Shape::kKStages) & 1);
            mma_scores<T, DP, kTcCols>(buffer + Shape::kS, sb + Shape::kQ,
                                       sb + Shape::kK + (i % Shape::kKStages) * Shape::kStage);
            patience.wait(full_v(i), (i / Shape::kVStages) & 1);
            mma_scores<T, DP, kTcCols>(buffer + Shape::kDP, sb + Shape::kG,
                                       sb + Shape::kV + (i % Shape::kVStages) * Shape::kStage);
        };
        if (lane == 0)
            for (int i = 0; i < 9; ++i) mbar_init(sb + Shape::kBar + 8 * i);
        __syncwarp();
        tma_expect(sb + Shape::kFullQ, 2 * Shape::kG);
        tma_rows<DP, 128>(sb + Shape::kQ, &M.q, h, t.row, sb + Shape::kFullQ);
        tma_rows<DP, 128>(sb + Shape::kG, &M.g, h, t.row, sb + Shape::kFullQ);
        load_tile(0);
        if (!Shape::kTight) load_tile(1);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = uniform(*slot);
        patience.wait(sb + Shape::kFullQ, 0);
        // Step i commits to barrier i mod kBuffers; the prologue stands for the kBuffers steps
        // before step 0.
        scores(0);
        mma_commit(sb + Shape::kBar);
        if (kBuffers == 2) {
            scores(1);
            mma_commit(sb + Shape::kBar + 8);
            patience.wait(sb + Shape::kBar, 0);
            load_tile(2);
        }
        for (int i = 0; i < tiles; ++i) {
            __syncthreads();  // the score gradients of tile i are in TMEM
            tc_fence_after();
            const uint32_t keys = sb + Shape::kK + (i % Shape::kKStages) * Shape::kStage;
            if (Shape::kCells)
                mma_weighted<T, DP, kTcCols, 8>(tmem + Shape::kDQ, tmem + Shape::kP + (i & 1) * (kTcCols / 2), keys, i > 0);
            else if (MODE == kGradQ)
                mma_weighted<T, DP, kTcCols>(tmem + Shape::kDQ, tmem + (i & (kBuffers - 1)) * Shape::kBuffer + Shape::kS,
                                             keys, i > 0);
            if (Shape::kTight) {
                // One stage, one buffer: barrier 1 tells that it is free, barrier 0 that S is there.
                mma_commit(sb + Shape::kBar + 8);
                patience.wait(sb + Shape::kBar + 8, i & 1);
                if (i + 1 < tiles) {
                    load_tile(i + 1);
                    scores(i + 1);
                    mma_commit(sb + Shape::kBar);
                }
            } else {
                scores(i + kBuffers);  // executed in order: the buffer may be overwritten
                mma_commit(sb + Shape::kBar + 8 * (i & (kBuffers - 1)));
                // The products of step i - 1 are done (one buffer: the others waited for them):
                // keys i - 1 and values i + kBuffers - 1 are free.
                if (kBuffers == 2) patience.wait(sb + Shape::kBar + 8 * ((i - 1) & 1), ((i + 1) >> 1) & 1);
                load_tile(i + kBuffers + 1);
            }
        }
        tc_fence_before();
        __syncthreads();  // the results have been read
        tc_fence_after();
        tmem_free(tmem, Shape::kCols);
        return;
    }

    if (tid < 4) flags[tid] = 0u;
    const bool live = r < t.rows;
    BiasRow bias;
    if (BIAS) bias.init(A, A.a.qpos, t.row, r, t.rows, sb + Shape::kTable, 1);
    Columns columns;
    auto fetch_columns = [&](int i) {
        if (!BIAS || i >= tiles) return;
        const int k0 = span.tile(i) * kTcCols;
        columns.fetch(A.a.kpos, (int64_t)t.other + k0, min(kTcCols, t.lk - k0), A.a.axes);
    };
    auto store_columns = [&](int i) {
        if (!BIAS || i >= tiles) return;
        columns.store(kpos + (i % Shape::kPosStages) * A.a.axes * kTcCols,
                      min(kTcCols, t.lk - span.tile(i) * kTcCols), A.a.axes, bias, 1);
    };
    fetch_columns(0);
    const int64_t at = (((int64_t)t.row + r) * A.a.heads + h) * A.a.dim;
    float* delta_at = A.a.delta + (int64_t)h * A.a.q_rows + t.row + r;
    if (BIAS) {
        if (!ONE) {
            tc_load_table(A, table, h);
        } else if (!Shape::kTight || entries <= Shape::kTightEntries) {
            for (int e = tid; e < entries; e += Shape::kCompute) table[e] = table_entry(A.a, e, h) * kLog2e;
        }
    }
    if (Shape::kCells)
        for (int e = tid; e < entries * 128; e += Shape::kCompute) all_cells[e] = 0.f;
    const float lse2 = live ? load_lse2(A, t.row + r, h) : INFINITY;
    store_columns(0);
    fetch_columns(1);
    store_columns(1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21);  // 32 quarter ..
    // Columns of a tile that this thread forms, in units.  With cells, a group that keeps those
    // of an axis forms one unit of 8 columns and the others divide the rest.
    constexpr int kUnit = Shape::kCells ? 8 : 16;
    int first_column = 0, last_column = 0;
    if (Shape::kCells) {
        const int axes = A.a.axes, rest = kTcCols / kUnit - axes, others = Shape::kGroups - axes;
        auto begin = [&](int g) { return g <= axes ? g : axes + rest * (g - axes) / others; };
        first_column = kUnit * begin(group);
        last_column = kUnit * begin(group + 1);
    }
    Waiters<kBuffers> done(sb + Shape::kBar, A.a.status);
    float delta = 0.f;  // D; kDelta: this thread's columns of its sum so far
    if constexpr (MODE == kGradQTable) {
        if (live) delta = *delta_at;
    } else if constexpr (MODE == kGradQ) {
        // A row's elements lie across kLanes lanes (a thread that read its whole row, in each
        // group again, fetched a line per lane and load: 348 against 289 us at 128 elements).
        constexpr int kLanes = DP / 8, kRows = 128 / (Shape::kCompute / 32), kSteps = kRows * kLanes / 32;
        static_assert(kSteps * 32 == kRows * kLanes, "a warp's rows in whole steps");
        const int c = lane % kLanes, row0 = (tid >> 5) * kRows + lane / kLanes;
        uint4 own[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int row = row0 + i * (32 / kLanes);
            own[i] = make_uint4(0u, 0u, 0u, 0u);
            if (row < t.rows && c * 8 < A.a.dim)
                own[i] = *reinterpret_cast<const uint4*>(
                    static_cast<const T*>(A.a.out) + (((int64_t)t.row + row) * A.a.heads + h) * A.a.dim + c * 8);
        }
        Patience(A.a.status).wait(sb + Shape::kFullQ, 0);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int row = row0 + i * (32 / kLanes);
            float g[8], o[8], sum = 0.f;
            Elem<T>::unpack(own[i], o);
            Elem<T>::unpack(*reinterpret_cast<const uint4*>(smem + Shape::kG + TcTile<DP>::at(128, row, c)), g);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(g[e], o[e], sum);
#pragma unroll
            for (int x = kLanes / 2; x; x >>= 1) sum += __shfl_xor_sync(FULL_MASK, sum, x);
            if (c == 0 && row < t.rows) A.a.delta[(int64_t)h * A.a.q_rows + t.row + row] = sum;
        }
        compute_sync<Shape::kCompute>();
        if (live) delta = *delta_at;
    }
    const f32x2 scale2 = pack2(A.scale_log2, A.scale_log2), lse22 = pack2(-lse2, -lse2);
    // Group a's cells of axis a: this lane's first.
    const float cell_first =
        __int_as_float((int)smem_u32(cells) + min(group, 2) * A.a.buckets * 128 + lane * 4);

    for (int i = 0; i < tiles; ++i) {
        done.wait(i);
        fetch_columns(i + Shape::kAhead);
        const int k0 = span.tile(i) * kTcCols, n = min(kTcCols, t.lk - k0);
        const bool whole = n == kTcCols && t.rows == 128 &&
                           all_visible(A, t.first, t.first + 127, k0, k0 + kTcCols - 1);
        uint64_t seen = ~0ull;
        if (!whole) seen = live ? seen_keys(A, p, k0, n) : 0ull;
        if (BIAS && bias.far) seen = 0ull;
        const bool all = __all_sync(FULL_MASK, seen == ~0ull);
        const float* cols = kpos + (i % Shape::kPosStages) * A.a.axes * kTcCols;
        // kUnit columns from c0.
        auto unit = [&](int c0) {
            const uint32_t own = lanes + (i & (kBuffers - 1)) * Shape::kBuffer + c0;
            const uint32_t pairs = Shape::kCells ? lanes + Shape::kP + (i & 1) * (kTcCols / 2) + c0 / 2 : own + Shape::kS;
            float s[kUnit], dp[kUnit];
            if constexpr (kUnit == 16) {
                tmem_ld16(own + Shape::kS, s);
                tmem_ld16(own + Shape::kDP, dp);
            } else {
                tmem_ld8(own + Shape::kS, s);
                tmem_ld8(own + Shape::kDP, dp);
            }
            f32x2 b[kUnit / 2];
            if (BIAS)
                bias_of<BIAS == 2, ONE, kUnit>(
                    A, bias, cols + c0, b, !Shape::kTight || entries <= Shape::kTightEntries ? table : nullptr, h);
            tmem_wait_ld();
            tmem_use(s);
            tmem_use(dp);
#pragma unroll
            for (int e = 0; e < kUnit; e += 2) {
                f32x2 x = fma2(pack2(s[e], s[e + 1]), scale2, lse22);
                if (BIAS) x = add2(x, b[e / 2]);
                float u, v;
                unpack2(x, u, v);
                u = exp2_sfu(u);
                v = exp2_sfu(v);
                if (MODE == kDelta) {
                    s[e] = u * dp[e];
                    s[e + 1] = v * dp[e + 1];
                } else {
                    s[e] = u * (dp[e] - delta);
                    s[e + 1] = v * (dp[e + 1] - delta);
                }
            }
            if (!all) {
#pragma unroll
                for (int e = 0; e < kUnit; ++e) s[e] = (uint32_t)(seen >> (c0 + e)) & 1u ? s[e] : 0.f;
            }
            if (MODE == kDelta) {
                f32x2 sum = pack2(s[0], s[1]);
#pragma unroll
                for (int e = 2; e < kUnit; e += 2) sum = add2(sum, pack2(s[e], s[e + 1]));
                float u, v;
                unpack2(sum, u, v);
                delta += u + v;
            } else {
                uint32_t w[kUnit / 2];
#pragma unroll
                for (int e = 0; e < kUnit / 2; ++e) w[e] = Elem<T>::two(s[2 * e], s[2 * e + 1]);
                if constexpr (kUnit == 8) {
                    tmem_st8(lanes + Shape::kDS + (i & 1) * kTcCols + c0, reinterpret_cast<const uint32_t*>(s));
                    tmem_st4(pairs, w);
                } else {
                    tmem_st8(pairs, w);
                }
            }
        };
        if constexpr (Shape::kCells) {
            for (int c0 = first_column; c0 < last_column; c0 += kUnit) unit(c0);
        } else {
#pragma unroll
            for (int c0 = 0; c0 < kPer; c0 += kUnit) unit(kPer * group + c0);
        }
        if (i + Shape::kAhead > 1) store_columns(i + Shape::kAhead);
        if (MODE != kDelta) tmem_wait_st();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (Shape::kCells && group < A.a.axes) {
            const float* axis = cols + group * kTcCols;
            const float part = group == 0 ? bias.part[0] : group == 1 ? bias.part[1] : bias.part[2];
            const uint32_t buffer = lanes + Shape::kDS + (i & 1) * kTcCols;
#pragma unroll
            for (int c = 0; c < kTcCols; c += 16) {
                float ds[16];
                tmem_ld16(buffer + c, ds);
                int at_cell[16];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 c4 = *reinterpret_cast<const float4*>(axis + c + e);
                    const float col[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        at_cell[e + k] = bias.address<BIAS == 2>(A, part, col[k], cell_first);
                }
                tmem_wait_ld();
                tmem_use(ds);
                // Two columns at a time, for half the round trips: where both meet in one cell the
                // second sum carries the first, and is written last.
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    float u, v;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(u) : "r"(at_cell[e]) : "memory");
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at_cell[e + 1]) : "memory");
                    u += ds[e];
                    v = (at_cell[e] == at_cell[e + 1] ? u : v) + ds[e + 1];
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at_cell[e]), "f"(u) : "memory");
                    asm volatile("st.shared.f32 [%0], %1;" ::"r"(at_cell[e + 1]), "f"(v) : "memory");
                }
            }
            tc_fence_before();
        }
    }
    // What was committed last.
    if (!Shape::kTight) {
        done.wait(tiles);
        if (kBuffers == 2) done.wait(tiles + 1);
    } else if (tiles > 0) {
        done.odd.phase = (tiles - 1) & 1;
        done.odd.wait();
    }
    const bool far = BIAS && live && bias.far;
    if (MODE == kDelta) {
        // The groups' shares in order; the table's place is free now.
        float* shares = table;
        compute_sync<Shape::kCompute>();
        shares[tid] = delta;
        compute_sync<Shape::kCompute>();
        if (group == 0) {
            for (int g = 1; g < Shape::kGroups; ++g) delta += shares[g * kTcRows + r];
            for (unsigned bad = __ballot_sync(FULL_MASK, far); bad; bad &= bad - 1) {
                const int row = (r & ~31) + __ffs(bad) - 1;
                const float d = exact_delta_row<T>(A, (int64_t)t.row + row, t.first + row, t.other, t.lk, h);
                if (row == r) delta = d;
            }
            if (live) *delta_at = delta;
        }
    } else {
        bool nan = far;
#pragma unroll
        for (int c = 0; c < DP; c += 16) {
            if ((c / 16) % Shape::kGroups != group) continue;
            float o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
            if (tiles > 0) {
                tmem_ld16(lanes + Shape::kDQ + c, o);
                tmem_wait_ld();
                tmem_use(o);
            }
            if (!live) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                o[e] *= A.a.scale;
                nan |= !isfinite(o[e]);  // a float16 score gradient may have overflowed
            }
#pragma unroll
            for (int e = 0; e < 16; e += 8)
                if (c + e < A.a.dim)
                    *reinterpret_cast<uint4*>(static_cast<T*>(A.a.grad_q) + at + c + e) = Elem<T>::pack(o + e);
        }
        const unsigned bad_here = __ballot_sync(FULL_MASK, nan), apart = __ballot_sync(FULL_MASK, far);
        if (lane == 0 && bad_here) atomicOr(flags + quarter, bad_here);
        compute_sync<Shape::kCompute>();
        // The groups' warps take the quarter's rows in turn; those that add to its cells are the
        // first group's.
        int turn = 0;
        for (unsigned bad = flags[quarter]; bad; bad &= bad - 1, ++turn) {
            const int b = __ffs(bad) - 1, row = (r & ~31) + b;
            const bool whole = (apart >> b) & 1u;
            float* own_cells = Shape::kCells && whole ? cells : nullptr;
            if ((own_cells ? 0 : turn % Shape::kGroups) != group) continue;
            exact_grad_q_row<T>(A, (int64_t)t.row + row, t.first + row, t.other, t.lk, h, whole, own_cells);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (Shape::kCells)
        for (int e = tid; e < entries; e += Shape::kCompute) {
            float v = 0.f;
            for (int w = 0; w < 4; ++w)
                for (int l = 0; l < 32; ++l) v += all_cells[(w * entries + e) * 32 + ((l + e) & 31)];
            partial[((int64_t)blockIdx.x * A.a.heads + h) * entries + e] = v;
        }
}

// ---------------------------------------------------------------- keys and values
// Pipeline and threads as in the query kernel: dv += P^T_i dO_i and dk += dS^T_i Q_i
// are followed by S^T and dP^T of tile i + 2 over the same buffer.
template <int DP>
struct GradKvShape {
    static constexpr int kBlocks = DP == 128 ? 1 : 2, kGroups = 4 / kBlocks, kBuffers = 3 - kBlocks;
    static constexpr int kCompute = kGroups * kTcRows, kThreads = kCompute + 32, kPer = kTcCols / kGroups;
    static constexpr int kStages = 2 + kBuffers, kRowStages = 4;
    static constexpr int kS = 0, kDP = kTcCols, kBuffer = (kBuffers - 1) * 2 * kTcCols;
    static constexpr int kDK = 2 * kTcCols + kBuffer, kDV = kDK + DP, kCols = 512 / kBlocks;
    static constexpr uint32_t kK = 0, kV = TcTile<DP>::bytes(128), kStage = TcTile<DP>::bytes(64),
                              kQ = 2 * kV, kG = kQ + kStages * kStage, kRow = kG + kStages * kStage,
                              kPos = kRow + kRowStages * 2 * kTcCols * 4,
                              kBar = kPos + kRowStages * 3 * kTcCols * 4, kTable = kBar + 128;
    // Barriers: products (2); stages of queries and gradients (4), K and V; then TMEM's address, row flags.
    static constexpr uint32_t kFull = kBar + 16, kFullK = kBar + 48, kSlot = kBar + 56, kFlags = kBar + 64;
    static bool one_copy(int entries) { return kTable + (size_t)entries * 128 + 1024 > kAttnSmem; }
    static size_t bytes(int entries, bool one) {
        const size_t need = kTable + (size_t)entries * (one ? 4 : 128) + 1024;
        const size_t least = 233472 / (kBlocks + 1);  // no more blocks than TMEM serves
        return need > least ? need : least;
    }
};

// Key tiles that hold sinks are shared out: attention_shares.cuh.
template <typename T, int DP, int BIAS, bool ONE>
__global__ void __launch_bounds__((GradKvShape<DP>::kThreads), (GradKvShape<DP>::kBlocks))
attn_tc_grad_kv_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ TcMaps M, const KeyShares K,
                       float* __restrict__ partial) {
    using Shape = GradKvShape<DP>;
    constexpr int kPer = Shape::kPer, kBuffers = Shape::kBuffers;
    const ShareBlock block = share_block(blockIdx.x, K);
    const AttnTile t = reinterpret_cast<const AttnTile*>(A.a.k_tiles)[block.tile];
    const bool shared = block.divided && t.first < K.limit;
    if (!shared && block.share > 0) return;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, r = tid & 127, quarter = r >> 5, group = tid >> 7;
    const int hk = blockIdx.y, h0 = hk * A.group;
    const int j = t.first + r;
    float* qpos = reinterpret_cast<float*>(smem + Shape::kPos);
    float* rows = reinterpret_cast<float*>(smem + Shape::kRow);  // [stage][-lse2, -D][64]
    float* table = reinterpret_cast<float*>(smem + Shape::kTable);
    uint32_t* slot = reinterpret_cast<uint32_t*>(smem + Shape::kSlot);
    unsigned* flags = reinterpret_cast<unsigned*>(smem + Shape::kFlags);  // rows to form again

    int lo, hi;
    query_span(A, t.first, t.first + t.rows - 1, t.lq, t.lk, lo, hi);
    int first = 0, per = hi > lo ? (hi - lo + kTcCols - 1) / kTcCols : 0;
    if (shared) {
        first = (int)((int64_t)per * block.share / K.shares);
        per = (int)((int64_t)per * (block.share + 1) / K.shares) - first;
    }
    const int tiles = (int)uniform((uint32_t)(per * A.group));

    if (tid >= Shape::kCompute) {  // the warp that feeds the tensor core
        tmem_alloc(smem_u32(slot), Shape::kCols);
        auto full = [&](int i) { return sb + Shape::kFull + 8 * (i % Shape::kStages); };
        int next_head = h0, next_query = 0;  // of the tile to be copied next
        auto load_next = [&](int i) {
            if (i >= tiles) return;
            const int row = t.other + lo + (first + next_query) * kTcCols;
            const uint32_t stage = (i % Shape::kStages) * Shape::kStage;
            tma_expect(full(i), 2 * Shape::kStage);
            tma_rows<DP, kTcCols>(sb + Shape::kQ + stage, &M.q, next_head, row, full(i));
            tma_rows<DP, kTcCols>(sb + Shape::kG + stage, &M.g, next_head, row, full(i));
            if (++next_query == per) {
                next_query = 0;
                ++next_head;
            }
        };
        Patience patience(A.a.status);
        uint32_t tmem = 0;
        auto scores = [&](int i) {  // S^T and dP^T of tile i into its buffer
            if (i >= tiles) return;
            const uint32_t buffer = tmem + (i & (kBuffers - 1)) * Shape::kBuffer;
            const uint32_t stage = (i % Shape::kStages) * Shape::kStage;
            patience.wait(full(i), (i / Shape::kStages) & 1);
            mma_scores<T, DP, kTcCols>(buffer + Shape::kS, sb + Shape::kK, sb + Shape::kQ + stage);
            mma_scores<T, DP, kTcCols>(buffer + Shape::kDP, sb + Shape::kV, sb + Shape::kG + stage);
        };
        if (lane == 0)
            for (int i = 0; i < 7; ++i) mbar_init(sb + Shape::kBar + 8 * i);
        __syncwarp();
        tma_expect(sb + Shape::kFullK, 2 * Shape::kV);
        tma_rows<DP, 128>(sb + Shape::kK, &M.k, hk, t.row, sb + Shape::kFullK);
        tma_rows<DP, 128>(sb + Shape::kV, &M.v, hk, t.row, sb + Shape::kFullK);
        for (int i = 0; i <= kBuffers; ++i) load_next(i);
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        tmem = uniform(*slot);
        patience.wait(sb + Shape::kFullK, 0);
        scores(0);
        mma_commit(sb + Shape::kBar);
        if (kBuffers == 2) {
            scores(1);
            mma_commit(sb + Shape::kBar + 8);
        }
        for (int i = 0; i < tiles; ++i) {
            __syncthreads();  // weights and score gradients of tile i are in TMEM
            tc_fence_after();
            const uint32_t stage = (i % Shape::kStages) * Shape::kStage;
            const uint32_t buffer = tmem + (i & (kBuffers - 1)) * Shape::kBuffer;
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kDV, buffer + Shape::kS, sb + Shape::kG + stage, i > 0);
            mma_weighted<T, DP, kTcCols>(tmem + Shape::kDK, buffer + Shape::kDP, sb + Shape::kQ + stage, i > 0);
            scores(i + kBuffers);  // executed in order: the buffer may be overwritten
            mma_commit(sb + Shape::kBar + 8 * (i & (kBuffers - 1)));
            // The products of step i - 1 are done (one buffer: the others waited for them).
            if (kBuffers == 2) patience.wait(sb + Shape::kBar + 8 * ((i - 1) & 1), ((i + 1) >> 1) & 1);
            load_next(i + kBuffers + 1);
        }
        tc_fence_before();
        __syncthreads();  // the results have been read
        tc_fence_after();
        tmem_free(tmem, Shape::kCols);
        return;
    }

    if (tid < 4) flags[tid] = 0u;
    const f32x2 scale2 = pack2(A.scale_log2, A.scale_log2);
    const bool live = r < t.rows;
    BiasRow bias;
    if (BIAS) bias.init(A, A.a.kpos, t.row, r, t.rows, sb + Shape::kTable, -1);
    auto load_table = [&](int h) {
        if (!BIAS) return;
        if (!ONE) tc_load_table(A, table, h);
        else
            for (int e = tid; e < A.a.axes * A.a.buckets; e += Shape::kCompute) table[e] = table_entry(A.a, e, h) * kLog2e;
    };
    // What a thread fetches of a tile and stores (-lse2, -D, the position) past the latency.  The head and the first query of the tile fetched next.
    int next_head = h0, next_query = 0;
    float stat = 0.f;
    Columns columns;
    auto fetch_next = [&](int i) {
        if (i >= tiles) return;
        const int i0 = lo + (first + next_query) * kTcCols, n = min(kTcCols, hi - i0), c = tid & (kTcCols - 1);
        const int64_t row = (int64_t)t.other + i0;
        if (tid < 2 * kTcCols && c < n)
            stat = (tid < kTcCols ? A.a.lse : A.a.delta)[(int64_t)next_head * A.a.q_rows + row + c];
        if (BIAS) columns.fetch(A.a.qpos, row, n, A.a.axes);
    };
    auto store_next = [&](int i) {
        if (i >= tiles) return;
        const int i0 = lo + (first + next_query) * kTcCols;
        if (tid < 2 * kTcCols) {
            const bool on = (tid & (kTcCols - 1)) < hi - i0;
            rows[(i & 3) * 2 * kTcCols + tid] =
                tid < kTcCols ? (on && stat != -INFINITY ? -stat * kLog2e : -INFINITY) : (on ? -stat : 0.f);
        }
        if (BIAS) columns.store(qpos + (i & 3) * 3 * kTcCols, min(kTcCols, hi - i0), A.a.axes, bias, -1);
        if (++next_query == per) {
            next_query = 0;
            ++next_head;
        }
    };
    fetch_next(0);
    load_table(h0);
    store_next(0);
    fetch_next(1);
    store_next(1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const uint32_t mine = tmem + ((uint32_t)quarter << 21);
    Waiters<kBuffers> done(sb + Shape::kBar, A.a.status);
    int head = h0, query = 0;  // of the tile at hand
    for (int i = 0; i < tiles; ++i) {
        if (BIAS && query == 0 && i > 0) {  // the next query head's table
            load_table(head);
            compute_sync<Shape::kCompute>();
        }
        done.wait(i);
        fetch_next(i + 2);
        const int i0 = lo + (first + query) * kTcCols, n = min(kTcCols, hi - i0), p0 = i0 + t.lk - t.lq;
        const bool whole = n == kTcCols && t.rows == 128 &&
                           all_visible(A, p0, p0 + kTcCols - 1, t.first, t.first + 127);
        uint32_t bits = ~0u;  // of this thread's columns
        if (!whole) bits = live ? (uint32_t)(seeing_queries(A, j, p0, n) >> (kPer * group)) : 0u;
        if (BIAS && bias.far) bits = 0u;
        constexpr uint32_t kFull = kPer == 32 ? ~0u : (1u << (kPer & 31)) - 1;
        const bool all = __all_sync(FULL_MASK, (bits & kFull) == kFull);
        const float* cols = qpos + (i & 3) * 3 * kTcCols;
        const float* row = rows + (i & 3) * 2 * kTcCols;
#pragma unroll
        for (int cc = 0; cc < kPer; cc += 16) {
            const int c = kPer * group + cc;
            const uint32_t own = mine + (i & (kBuffers - 1)) * Shape::kBuffer + c;
            float s[16], dp[16];
            tmem_ld16(own + Shape::kS, s);
            tmem_ld16(own + Shape::kDP, dp);
            f32x2 b[8];
            if (BIAS) bias_of<BIAS == 2, ONE, 16>(A, bias, cols + c, b, table, head);
            tmem_wait_ld();
            tmem_use(s);
            tmem_use(dp);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                // Staged negated: -lse2 and -D.
                f32x2 l0, l1, d0, d1;
                lds_pairs<0>(smem_u32(row + c + e), l0, l1);
                lds_pairs<0>(smem_u32(row + kTcCols + c + e), d0, d1);
                f32x2 x = fma2(pack2(s[e], s[e + 1]), scale2, l0);
                f32x2 y = fma2(pack2(s[e + 2], s[e + 3]), scale2, l1);
                if (BIAS) {
                    x = add2(x, b[e / 2]);
                    y = add2(y, b[e / 2 + 1]);
                }
                unpack2(x, s[e], s[e + 1]);
                unpack2(y, s[e + 2], s[e + 3]);
                unpack2(add2(pack2(dp[e], dp[e + 1]), d0), dp[e], dp[e + 1]);
                unpack2(add2(pack2(dp[e + 2], dp[e + 3]), d1), dp[e + 2], dp[e + 3]);
            }
            uint32_t w[8], g[8];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = exp2_sfu(s[e]);
                dp[e] *= s[e];
            }
            if (!all) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool on = (bits >> (cc + e)) & 1u;
                    s[e] = on ? s[e] : 0.f;
                    dp[e] = on ? dp[e] : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[e] = Elem<T>::two(s[2 * e], s[2 * e + 1]);
                g[e] = Elem<T>::two(dp[2 * e], dp[2 * e + 1]);
            }
            tmem_st8(own + Shape::kS, w);
            tmem_st8(own + Shape::kDP, g);
        }
        store_next(i + 2);
        tmem_wait_st();
        tc_fence_before();
        __syncthreads();
        if (++query == per) {
            query = 0;
            ++head;
        }
    }
    done.wait(tiles);
    if (kBuffers == 2) done.wait(tiles + 1);
    bool nan = BIAS && live && bias.far;
    const int64_t at = (((int64_t)t.row + r) * A.a.kv_heads + hk) * A.a.dim;
    float* sums = shared ? share_sums(A, partial, block.tile, r, hk, K.shares, block.share) : nullptr;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int c = 0; c < DP; c += 16) {
            if ((c / 16) % Shape::kGroups != group) continue;
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
                nan |= !isfinite(o[e]);  // a float16 score gradient may have overflowed
                if (BIAS && bias.far) o[e] = __int_as_float(0x7fffffff);  // for the join: form it again
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
    const unsigned bad_here = __ballot_sync(FULL_MASK, nan);
    if (lane == 0 && bad_here) atomicOr(flags + quarter, bad_here);
    compute_sync<Shape::kCompute>();
    int turn = 0;
    for (unsigned bad = shared ? 0u : flags[quarter]; bad; bad &= bad - 1, ++turn)
        if (turn % Shape::kGroups == group) {  // the groups' warps take the quarter's rows in turn
            const int row = (r & ~31) + __ffs(bad) - 1;
            exact_grad_kv_row<T>(A, t.base, t.first + row, t.other, t.lq, t.lk, hk);
        }
    tc_fence_before();
    __syncthreads();
}

template <typename T, int DP, int BIAS, int MODE, bool ONE = QueryShape<DP, MODE>::kTight>
int run_q(const AttnArgs& A, const TcMaps& M, float* partial, cudaStream_t s) {
    using Shape = QueryShape<DP, MODE>;
    const int axes = BIAS ? A.a.axes : 0, entries = axes * A.a.buckets;
    if constexpr (Shape::kCells && !Shape::kTight) {
        if (!ONE && Shape::one_copy(axes, entries)) return run_q<T, DP, BIAS, MODE, true>(A, M, partial, s);
    }
    const size_t bytes = Shape::bytes(axes, entries, ONE);
    const int st = attn_prepare<&attn_tc_query_kernel<T, DP, BIAS, MODE, ONE>>("attn_tc_query_kernel");
    if (st != kOk) return st;
    const dim3 grid((unsigned)A.a.q_tile_count, (unsigned)A.a.heads);
    attn_tc_query_kernel<T, DP, BIAS, MODE, ONE><<<grid, Shape::kThreads, bytes, s>>>(A, M, partial);
    return check_launch("attn_tc_query_kernel");
}
template <typename T, int DP, int BIAS, bool ONE = false>
int run_kv(const AttnArgs& A, const TcMaps& M, float* partial, cudaStream_t s) {
    const int entries = BIAS ? A.a.axes * A.a.buckets : 0;
    if constexpr (BIAS != 0 && DP == 128) {  // narrower rows always leave room
        if (!ONE && GradKvShape<DP>::one_copy(entries)) return run_kv<T, DP, BIAS, true>(A, M, partial, s);
    }
    const size_t bytes = GradKvShape<DP>::bytes(entries, ONE);
    int st = attn_prepare<&attn_tc_grad_kv_kernel<T, DP, BIAS, ONE>>("attn_tc_grad_kv_kernel");
    if (st != kOk) return st;
    const KeyShares K = key_shares(A);
    const dim3 grid((unsigned)key_blocks(A, K), (unsigned)A.a.kv_heads);
    attn_tc_grad_kv_kernel<T, DP, BIAS, ONE><<<grid, GradKvShape<DP>::kThreads, bytes, s>>>(A, M, K, partial);
    st = check_launch("attn_tc_grad_kv_kernel");
    if (st != kOk || K.shares == 1) return st;
    return join_shares<T>(A, K, partial, s);
}
template <typename T, int DP, int BIAS>
int run(const AttnArgs& A, cudaStream_t s) {
    float* sums = static_cast<float*>(A.a.workspace);
    TcMaps M = {};
    int st = make_maps<DP>(M, A, true);
    if (st != kOk) return st;
    if (A.a.q_tile_count) {
        if constexpr (BIAS != 0) {
            float* partial = reinterpret_cast<float*>(static_cast<unsigned char*>(A.a.workspace) + share_bytes(A));
            if (A.a.grad_table) {
                st = run_q<T, DP, BIAS, kDelta>(A, M, nullptr, s);
                if (st == kOk) st = run_q<T, DP, BIAS, kGradQTable>(A, M, partial, s);
            } else {
                st = run_q<T, DP, BIAS, kGradQ>(A, M, nullptr, s);
            }
        } else {
            st = run_q<T, DP, BIAS, kGradQ>(A, M, nullptr, s);
        }
    }
    if (st == kOk && A.a.k_tile_count) st = run_kv<T, DP, BIAS>(A, M, sums, s);
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

int attn_tc_backward(const AttnArgs& A, cudaStream_t s) {
    return A.a.dtype == MPO_F16 ? by_dim<__half>(A, s) : by_dim<__nv_bfloat16>(A, s);
}

}  // namespace mpo
