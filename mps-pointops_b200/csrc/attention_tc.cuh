// Tensor-core (tcgen05) pieces of the attention kernels for 16-bit types.
//
// Operand tiles are rows of DP elements (the head size rounded up to 16, 32,
// 64 or 128, zero-filled) in shared memory with the swizzle of their row
// length: 32, 64 or 128 bytes; DP = 128 is two halves of 64 elements.  One
// tile serves both ways: as a K-major operand (rows = M or N, elements = K)
// for scores, and as an MN-major B operand (rows = K, elements = N) for the
// products with the weights.  Tiles come by tensor-map copies (TMA) of 64 rows of
// one head, which cost the computing warps nothing (as 16-byte cp.async they took
// a third of a step).  A copy runs past a cloud's end into the next cloud's rows:
// their weights are exact zeros, and a result row that a NaN or an infinity among
// them turns into a NaN is formed again pair by pair (attention_exact.cuh).
#pragma once

#include <cuda.h>

#include <string>

#include "attention_common.cuh"

namespace mpo {
namespace {

constexpr int kTcRows = 128;  // rows of a tile: TMEM lanes, one thread (per column group) each
constexpr int kTcCols = 64;   // columns of a score tile
constexpr unsigned long long kTcWaitNs = 2000000000ull;

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}

// A value that is the same in every lane, for the uniform registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(FULL_MASK, v); }

// ---------------------------------------------------------------- barriers
__device__ __forceinline__ void mbar_init(uint32_t bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Waits of at most kTcWaitNs.  A thread whose wait ran out reports it and goes on
// through the same control flow (barriers of the block stay matched, memory
// accesses do not depend on the data that failed to come).
// One thread's waits: `dead` once one of them ran out; later ones are then cut
// short, but still let copies in flight land.
struct Patience {
    int32_t* status;
    bool dead = false;
    __device__ __forceinline__ explicit Patience(int32_t* st) : status(st) {}
    // By a converged warp.
    __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity) {
        poll(bar, parity);
        __syncwarp();
    }
    __device__ __forceinline__ void poll(uint32_t bar, uint32_t parity) {
        if (mbar_try(bar, parity)) return;
        const unsigned long long t0 = globaltimer_ns(), limit = dead ? kTcWaitNs / 1000 : kTcWaitNs;
        while (!mbar_try(bar, parity))
            if (globaltimer_ns() - t0 > limit) {
                dead = true;
                if (status) *status = 1;
                break;
            }
    }
};
struct Waiter {
    uint32_t bar;
    uint32_t phase = 0;
    Patience patience;
    __device__ __forceinline__ Waiter(uint32_t b, int32_t* st) : bar(b), patience(st) {}
    __device__ __forceinline__ void wait() {
        patience.wait(bar, phase);
        phase ^= 1;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    }
};

// B barriers used in turn: step i waits for what step i - B committed.
template <int B>
struct Waiters {
    Waiter even, odd;
    __device__ __forceinline__ Waiters(uint32_t bars, int32_t* st) : even(bars, st), odd(bars + 8, st) {}
    __device__ __forceinline__ void wait(int i) {
        if (B == 2 && (i & 1)) odd.wait();
        else even.wait();
    }
};

// ---------------------------------------------------------------- TMEM
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
                 "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Ties registers that a load fills to the wait before their first use.
template <int N>
__device__ __forceinline__ void tmem_use(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 16 consecutive 32-bit columns of this thread's lane; wait before use.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
        : "memory");
}

// ---------------------------------------------------------------- operands
template <int DP>
struct TcTile {
    static constexpr int kRowBytes = DP * 2 < 128 ? DP * 2 : 128;
    static constexpr int kHalves = DP * 2 / kRowBytes;
    static constexpr int kChunks = DP / 8;                    // 16-byte chunks of a row
    static constexpr int kHalfChunks = kRowBytes / 16;
    // Layout code of the matrix descriptor: 2 = 128-byte, 4 = 64-byte, 6 = 32-byte swizzle.
    static constexpr uint64_t kSwizzle = kRowBytes == 128 ? 2 : kRowBytes == 64 ? 4 : 6;
    static constexpr uint32_t bytes(int rows) { return rows * DP * 2; }
    // Byte offset of chunk c of row r in a tile of `rows` rows.
    static __device__ __forceinline__ uint32_t at(int rows, int r, int c) {
        const int half = c / kHalfChunks, cc = c % kHalfChunks;
        const int turn = kRowBytes == 128 ? (r & 7) : kRowBytes == 64 ? ((r >> 1) & 3) : ((r >> 2) & 1);
        return half * rows * kRowBytes + r * kRowBytes + ((cc ^ turn) << 4);
    }
    // Matrix descriptors: the low word holds the address and the leading offset (in 16-byte
    // units; shared memory ends below 2^18, so neither runs into the other), the high word
    // the stride of eight rows, the version and the swizzle.  The low word of a tile is formed
    // once; a product's operand is a constant away from it.
    static constexpr uint32_t kHigh = (8 * kRowBytes >> 4) | (1u << 14) | ((uint32_t)kSwizzle << 29);
    static __device__ __forceinline__ uint64_t desc(uint32_t low) {
        uint64_t d;
        asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(kHigh));
        return d;
    }
    // K-major operand of `rows` rows, elements 16 k .. 16 k + 15 of every row.
    static __device__ __forceinline__ uint64_t k_major(uint32_t tile, int rows, int k) {
        const int half = k / (kRowBytes / 32), kk = k % (kRowBytes / 32);
        return desc(((tile >> 4) | (1u << 16)) + ((half * rows * kRowBytes + kk * 32) >> 4));
    }
    // MN-major operand, rows 16 k .. 16 k + 15, all DP elements.
    static __device__ __forceinline__ uint64_t mn_major(uint32_t tile, int rows, int k) {
        return desc(((tile >> 4) | ((uint32_t)(rows * kRowBytes >> 4) << 16)) + (k * 16 * kRowBytes >> 4));
    }
};

// The maps of one call: queries, keys, values and the gradient of the result.
struct TcMaps {
    CUtensorMap q, k, v, g;
};
// What follows is called by a whole converged warp and issued by one elected
// lane, the same one every time: the operands then stay in uniform registers
// (under a branch on the lane each product took 90 cycles to issue, twice what
// it takes to run).
#define MPO_ELECTED "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e "
// Announces `bytes` on a barrier whose phase ends when they have come.
__device__ __forceinline__ void tma_expect(uint32_t bar, uint32_t bytes) {
    asm volatile(MPO_ELECTED "mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
                 : "memory");
}
// Rows [row, row + ROWS) of head h into a tile; rows past the tensor and elements
// past dim are zeros.  The box starts at element 0 or 64: a multiple of 16 bytes.
template <int DP, int ROWS>
__device__ __forceinline__ void tma_rows(uint32_t tile, const CUtensorMap* map, int h, int row, uint32_t bar) {
    using L = TcTile<DP>;
#pragma unroll
    for (int half = 0; half < L::kHalves; ++half)
#pragma unroll
        for (int r = 0; r < ROWS; r += 64)
            asm volatile(
                MPO_ELECTED "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
                "[%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(tile + (half * ROWS + r) * L::kRowBytes),
                "l"(map), "r"(half * 64), "r"(h), "r"(row + r), "r"(bar)
                : "memory");
}

// kind::f16 (both operands the same 16-bit type), float accumulators, M = 128.
template <typename T>
__device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool b_mn) {
    return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) |
           (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        MPO_ELECTED "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
// D (128 x NB) = A (128 rows of tile a) . B (NB rows of tile b)^T over DP elements.
template <typename T, int DP, int NB>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
        mma_ss(d, TcTile<DP>::k_major(a, 128, k), TcTile<DP>::k_major(b, NB, k),
               tc_idesc<T>(NB, false), k > 0);
}
// D (128 x DP) += weights (128 x NB) . B (NB rows of tile b).  The weights are 16-bit
// pairs in TMEM, those of columns 16 k .. in 8 columns from a + STRIDE k.  STRIDE
// 16: in the first half of the scores that they come from, so a thread that forms
// 16 columns overwrites nothing but what it has read itself.
template <typename T, int DP, int NB, int STRIDE = 16>
__device__ __forceinline__ void mma_weighted(uint32_t d, uint32_t a, uint32_t b, bool acc) {
#pragma unroll
    for (int k = 0; k < NB / 16; ++k)
        mma_ts(d, a + STRIDE * k, TcTile<DP>::mn_major(b, NB, k), tc_idesc<T>(DP, true), acc || k > 0);
}

// ---------------------------------------------------------------- masks
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Bits [lo, hi) of 64.
__device__ __forceinline__ uint64_t bit_range(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 64);
    return hi > lo ? (~0ull >> (64 - hi)) & (~0ull << lo) : 0ull;
}
// Columns of the key tile [k0, k0 + n) that a query at p sees.
__device__ __forceinline__ uint64_t seen_keys(const AttnArgs& A, int p, int k0, int n) {
    uint64_t m = bit_range(p - A.left - k0, p + A.right + 1 - k0) | bit_range(0, A.a.sinks - k0);
    if (A.a.causal) m &= bit_range(0, p + 1 - k0);
    return m & bit_range(0, n);
}
// Columns of the query tile at positions [p0, p0 + n) that see key j.
__device__ __forceinline__ uint64_t seeing_queries(const AttnArgs& A, int j, int p0, int n) {
    uint64_t m = j < A.a.sinks ? ~0ull : bit_range(j - A.right - p0, j + A.left + 1 - p0);
    if (A.a.causal) m &= bit_range(j - p0, 64);
    return m & bit_range(0, n);
}

// ---------------------------------------------------------------- bias
// The table of a head in shared memory, times log2(e), one copy per lane:
// entry e of lane l at byte 128 e + 4 l.  A lane reads its own bank, so a read
// costs one wavefront whatever the buckets (one shared copy: about three, for
// neighbouring points that differ).
//
// The address of a pair's entry takes two multiply-adds: integer instructions run
// at half their rate and bound the first form of this.  Positions are staged as
// floats relative to the tile's middle row (the first would be the one that differs from
// all others: a summary row at the head of a cloud); with d = key - query, the saturating
//   t = sat(d / 2R + 1/2)         (d split into the column's and the row's part)
// clamps to the axis' 2 R + 1 entries for nothing, and
//   t * (2R * 128) + first entry  in units of 2^-149, the spacing of denormals,
// is a float whose bits are the address.  Rounding: the row's part is below
// 2^15 / 2R + 1 and off by 2^-25 of its power of two, t by 2^-25, so the address
// before its rounding to an integer is off by at most 0.26 (R = 1; every R was
// gone through) and comes out exact.  Columns beyond +-2^16 of the middle row are
// clamped there (t saturates all the same); a row beyond +-2^15 of it (`far`) is
// left out of the tile and formed pair by pair (attention_exact.cuh).  A cloud of 4096
// points, 4 heads of 64, window 512, with one summary row 2^29 away: forward 0.33, backward
// 4.7 ms (9.8 and 26 relative to the first row; 0.10 and 0.25 without such a row).
constexpr int kNear = 1 << 15;
// By the block's row threads (a multiple of 128).
__device__ __forceinline__ void tc_load_table(const AttnArgs& A, float* table, int h) {
    for (int e = threadIdx.x; e < A.a.axes * A.a.buckets * 32; e += (blockDim.x & ~127u))
        table[e] = table_entry(A.a, e >> 5, h) * kLog2e;
}
struct BiasRow {
    float part[kAttnMaxAxes];  // 1/2 - row / 2R (or + row / 2R)
    float first[kAttnMaxAxes]; // address of this lane's first entry, as bits
    float inv, span;           // 1 / 2R; 256 R as bits
    int ref[kAttnMaxAxes];
    bool far = false;
    // sign 1: rows are queries, columns keys (key - query = column - row); -1: the reverse.
    // `row` of the `rows` from `base` on.
    __device__ __forceinline__ void init(const AttnArgs& A, const int32_t* pos, int64_t base, int row,
                                         int rows, uint32_t table, int sign) {
        inv = A.a.reach ? 1.f / (float)(2 * A.a.reach) : 0.f;
        span = __int_as_float(256 * A.a.reach);
#pragma unroll
        for (int a = 0; a < kAttnMaxAxes; ++a) {
            part[a] = first[a] = 0.f;
            ref[a] = 0;
            if (a >= A.a.axes) continue;
            ref[a] = pos[(base + rows / 2) * A.a.axes + a];
            const int d = row < rows ? pos[(base + row) * A.a.axes + a] - ref[a] : 0;
            const bool beyond = d > kNear || d < -kNear;
            far |= beyond;
            part[a] = (float)(0.5 - (double)(beyond ? 0 : sign * d) * (double)inv);
            first[a] = __int_as_float((int)table + a * A.a.buckets * 128 + (threadIdx.x & 31) * 4);
        }
    }
    // Staged value of a column.
    static __device__ __forceinline__ float column(int pos, int ref, int sign) {
        return (float)(sign * max(min(pos - ref, 2 * kNear), -2 * kNear));
    }
    // Address of the entry (or of the cell, with `from` the first) of a column, `row` being
    // the row's part.
    template <bool MAPPED>
    __device__ __forceinline__ int address(const AttnArgs& A, float row, float col, float from) const {
        const float t = __saturatef(fmaf(col, inv, row));
        int at = __float_as_int(fmaf(t, span, from));
        if (MAPPED) {
            const int lo = __float_as_int(from);
            at = lo + 128 * min(max(__ldg(A.a.map + ((at - lo) >> 7)), 0), A.a.buckets - 1);
        }
        return at;
    }
};
// Positions of columns [r0, r0 + n) by axis, dst[axis * 64 + column]: fetched into
// registers by the first 64 threads and stored later, past the latency.
struct Columns {
    int v[kAttnMaxAxes];
    __device__ __forceinline__ void fetch(const int32_t* pos, int64_t r0, int n, int axes) {
#pragma unroll
        for (int a = 0; a < kAttnMaxAxes; ++a)
            if (a < axes && (int)threadIdx.x < n) v[a] = pos[(r0 + threadIdx.x) * axes + a];
    }
    __device__ __forceinline__ void store(float* dst, int n, int axes, const BiasRow& row, int sign) const {
        if (threadIdx.x < kTcCols) {
#pragma unroll
            for (int a = 0; a < kAttnMaxAxes; ++a)
                if (a < axes)
                    dst[a * kTcCols + threadIdx.x] =
                        (int)threadIdx.x < n ? BiasRow::column(v[a], row.ref[a], sign) : 0.f;
        }
    }
};
// The table does not change while columns are read: free to move.
__device__ __forceinline__ float lds_table(int addr) {
    float v;
    asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
// Bias of N columns as pairs; cols: the staged columns of axis 0 at column c.
// ONE: the table has one copy, at `one` (null: read it from global memory, for
// head h); addresses are then used as entry numbers.
template <bool MAPPED, bool ONE, int N>
__device__ __forceinline__ void bias_of(const AttnArgs& A, const BiasRow& row, const float* cols, f32x2 (&t)[N / 2],
                                       const float* one, int h) {
    auto entry = [&](int a, float col) {
        const int at = row.template address<MAPPED>(A, row.part[a], col, row.first[a]);
        if (!ONE) return lds_table(at);
        const int e = a * A.a.buckets + ((at - __float_as_int(row.first[a])) >> 7);
        return one ? one[e] : table_entry(A.a, e, h) * kLog2e;
    };
#pragma unroll
    for (int a = 0; a < kAttnMaxAxes; ++a)
        if (a < A.a.axes) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 c4 = *reinterpret_cast<const float4*>(cols + a * kTcCols + e);
                const f32x2 x = pack2(entry(a, c4.x), entry(a, c4.y));
                const f32x2 y = pack2(entry(a, c4.z), entry(a, c4.w));
                t[e / 2] = a ? add2(t[e / 2], x) : x;
                t[e / 2 + 1] = a ? add2(t[e / 2 + 1], y) : y;
            }
        }
}

// Host: a map of (rows, heads, dim) for boxes of 64 rows of one head.
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}
template <int DP>
int make_map(CUtensorMap* map, const AttnArgs& A, const void* base, int64_t rows, int heads, int64_t row_stride,
             int64_t head_stride) {
    if (rows == 0) return kOk;  // no tile reads it
    const EncodeTiled encode = encode_tiled();
    if (!encode) return fail(kCudaError, "window attention: cuTensorMapEncodeTiled is not available");
    constexpr int kInner = DP < 64 ? DP : 64;
    const cuuint64_t dims[3] = {(cuuint64_t)A.a.dim, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
    const cuuint32_t box[3] = {kInner, 1, 64}, steps[3] = {1, 1, 1};
    const CUtensorMapSwizzle swizzle = kInner == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                       : kInner == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                      : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUresult r =
        encode(map, A.a.dtype == MPO_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
               const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(kCudaError, "window attention: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return kOk;
}
template <int DP>
int make_maps(TcMaps& M, const AttnArgs& A, bool backward) {
    int st = make_map<DP>(&M.q, A, A.a.q, A.a.q_rows, A.a.heads, A.a.q_row, A.a.q_head);
    if (st == kOk) st = make_map<DP>(&M.k, A, A.a.k, A.a.k_rows, A.a.kv_heads, A.a.k_row, A.a.k_head);
    if (st == kOk) st = make_map<DP>(&M.v, A, A.a.v, A.a.k_rows, A.a.kv_heads, A.a.v_row, A.a.v_head);
    if (st == kOk && backward)
        st = make_map<DP>(&M.g, A, A.a.grad_out, A.a.q_rows, A.a.heads, (int64_t)A.a.heads * A.a.dim, A.a.dim);
    return st;
}

// Barrier of THREADS computing threads.
template <int THREADS>
__device__ __forceinline__ void compute_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

}  // namespace
}  // namespace mpo
