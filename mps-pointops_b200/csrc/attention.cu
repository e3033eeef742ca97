// C entry points of the attention of serialised clouds: the tiles of a ragged
// batch, the checks of arguments, the choice of kernels and the reduction of
// the table's gradient (definitions: attention_common.cuh).
#include <algorithm>
#include <cmath>
#include <string>

#include "attention_shares.cuh"

namespace mpo {
namespace {

// grad_table[entry, head] = sum over the blocks of the query kernel of their
// partials (blocks, heads, entries), in block order: eight strided runs, then
// their sum.
__global__ void __launch_bounds__(256)
attn_table_reduce_kernel(const float* __restrict__ partial, int64_t blocks, int heads, int entries,
                         float* __restrict__ grad) {
    __shared__ float run[8][33];
    const int e = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5, h = blockIdx.y;
    float v = 0.f;
    if (e < entries)
        for (int64_t b = part; b < blocks; b += 8) v += partial[(b * heads + h) * entries + e];
    run[part][threadIdx.x & 31] = v;
    __syncthreads();
    if (part == 0 && e < entries) {
        for (int i = 1; i < 8; ++i) v += run[i][threadIdx.x & 31];
        grad[(int64_t)e * heads + h] = v;
    }
}

// Blocks of the query kernel for one planned tile: the 32-bit kernel takes 64 rows.
int partial_blocks_per_tile(const mpo_attention& a) { return a.dtype == MPO_F32 ? 2 : 1; }

size_t table_partial_bytes(const mpo_attention& a) {
    if (!a.grad_table) return 0;
    return (size_t)a.q_tile_count * partial_blocks_per_tile(a) * a.heads * a.axes * a.buckets *
           sizeof(float);
}

bool rows_ok(const void* p, int64_t row, int64_t head, int dtype) {
    const int64_t vec = dtype == MPO_F32 ? 4 : 8;
    return aligned_to(p, 16) && row % vec == 0 && head % vec == 0;
}

int check_attention(const mpo_attention* a, bool backward, const char* what) {
    auto bad = [&](const char* m) { return fail(kInvalidArgument, std::string(what) + ": " + m); };
    if (!a) return bad("null arguments");
    if (a->dtype < MPO_F32 || a->dtype > MPO_BF16) return bad("unknown dtype");
    if (a->q_rows < 0 || a->k_rows < 0 || a->q_rows + a->k_rows >= kFar)
        return bad("rows of queries and keys must be below 2^30 together");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
        return bad("heads must be a multiple of kv_heads");
    if (a->heads > 65535) return bad("too many heads");
    if (a->dim < 8 || a->dim > kAttnMaxDim || a->dim % 8)
        return bad("dim must be a multiple of 8 up to 128");
    if (a->sinks < 0) return bad("sinks must not be negative");
    if (a->q_tile_count < 0 || a->k_tile_count < 0 || a->q_tile_count >= kFar ||
        a->k_tile_count >= kFar)
        return bad("bad tile counts");
    if (a->max_rows < 0 || a->max_keys < 0 || a->clouds < 0) return bad("bad cloud sizes");
    if (!std::isfinite(a->scale)) return bad("scale must be finite");
    if (a->table) {
        if (a->table_dtype < MPO_F32 || a->table_dtype > MPO_BF16) return bad("unknown table dtype");
        if (a->axes < 1 || a->axes > kAttnMaxAxes) return bad("axes must be in [1, 3]");
        if (a->buckets < 1 || a->axes * (int64_t)a->buckets > kAttnMaxEntries)
            return bad("axes * buckets must be at most 256");
        if (a->reach < 0 || 2 * (int64_t)a->reach + 1 > kAttnMaxMap)
            return bad("reach must be in [0, 1024]");
        if (!a->map && a->buckets != 2 * a->reach + 1)
            return bad("buckets must be 2 * reach + 1 without a map");
        if ((a->q_rows && !a->qpos) || (a->k_rows && !a->kpos)) return bad("null position");
    } else if (a->grad_table) {
        return bad("grad_table needs a table");
    }
    if (a->q_tile_count > 0) {
        if (!a->q || !a->out || !a->q_tiles) return bad("null pointer");
        if (a->k_rows > 0 && (!a->k || !a->v)) return bad("null pointer");
        if (!rows_ok(a->q, a->q_row, a->q_head, a->dtype) ||
            !rows_ok(a->k, a->k_row, a->k_head, a->dtype) ||
            !rows_ok(a->v, a->v_row, a->v_head, a->dtype) || !aligned_to(a->out, 16))
            return bad("rows must start on 16-byte boundaries");
    }
    if (backward) {
        if (a->q_tile_count > 0 && (!a->grad_out || !a->grad_q || !a->lse || !a->delta))
            return bad("null pointer");
        if (a->k_tile_count > 0 && (!a->grad_k || !a->grad_v || !a->k_tiles || !a->k || !a->v))
            return bad("null pointer");
        if (!aligned_to(a->grad_out, 16) || !aligned_to(a->grad_q, 16) ||
            !aligned_to(a->grad_k, 16) || !aligned_to(a->grad_v, 16))
            return bad("rows must start on 16-byte boundaries");
    }
    return kOk;
}

AttnArgs derive(const mpo_attention& a) {
    AttnArgs A;
    A.a = a;
    if (!a.table) A.a.axes = A.a.buckets = 0;
    A.left = a.left < 0 || a.left > kUnlimited ? kUnlimited : a.left;
    A.right = a.right < 0 || a.right > kUnlimited ? kUnlimited : a.right;
    if (a.causal) A.right = 0;
    A.a.sinks = (int)min64(a.sinks, a.max_keys);
    A.group = a.heads / a.kv_heads;
    A.scale_log2 = a.scale * kLog2e;
    return A;
}

// Backward workspace: the shares' sums, then the table's partials.
size_t workspace_bytes(const AttnArgs& A, bool backward) {
    if (backward) return share_bytes(A) + table_partial_bytes(A.a);
    return A.a.q_tile_count && attn_rows_eligible(A) ? attn_rows_workspace(A) : 0;
}

}  // namespace
}  // namespace mpo

extern "C" {

int64_t mpo_attention_plan(const int64_t* ends, const int64_t* other_ends, int64_t segs, int keys,
                           int32_t* tiles, int64_t capacity) {
    using namespace mpo;
    auto bad = [&](const char* m) {
        fail(kInvalidArgument, std::string("mpo_attention_plan: ") + m);
        return (int64_t)-1;
    };
    if (segs < 0 || (segs > 0 && (!ends || !other_ends))) return bad("bad offsets");
    int64_t count = 0, base = 0, other = 0;
    for (int64_t b = 0; b < segs; ++b) {
        const int64_t n = ends[b] - base, m = other_ends[b] - other;
        if (ends[b] < base || other_ends[b] < other)
            return bad("offsets must be nondecreasing and nonnegative");
        if (ends[b] >= kFar || other_ends[b] >= kFar) return bad("offsets must be below 2^30");
        const int64_t lq = keys ? m : n, lk = keys ? n : m;
        for (int64_t i = 0; i < n; i += kAttnTile, ++count) {
            if (!tiles || count >= capacity) continue;
            int32_t* t = tiles + count * 8;
            t[0] = (int32_t)(base + i);
            t[1] = (int32_t)min64(kAttnTile, n - i);
            t[2] = (int32_t)(keys ? i : i + lk - lq);
            t[3] = (int32_t)other;
            t[4] = (int32_t)lq;
            t[5] = (int32_t)lk;
            t[6] = (int32_t)base;
            t[7] = (int32_t)b;
        }
        base = ends[b];
        other = other_ends[b];
    }
    if (keys && tiles) {  // the tiles that may hold sinks to the head of the list
        AttnTile* list = reinterpret_cast<AttnTile*>(tiles);
        std::sort(list, list + max64(0, min64(count, capacity)), [](const AttnTile& x, const AttnTile& y) {
            return x.first != y.first ? x.first < y.first : x.cloud < y.cloud;
        });
    }
    return count;
}

size_t mpo_window_attention_workspace_bytes(const mpo_attention* args) {
    using namespace mpo;
    if (check_attention(args, false, __func__) != kOk) return 0;
    return workspace_bytes(derive(*args), args->backward != 0);
}

int mpo_window_attention(const mpo_attention* args, void* stream) {
    using namespace mpo;
    const int st = check_attention(args, false, __func__);
    if (st != kOk || args->q_tile_count == 0) return st;
    const AttnArgs A = derive(*args);
    cudaStream_t s = (cudaStream_t)stream;
    if (attn_rows_eligible(A)) {
        MPO_REQUIRE_WORKSPACE(args->workspace);
        const size_t need = attn_rows_workspace(A);
        if (need && (!args->workspace || args->workspace_bytes < need))
            return fail(kWorkspaceTooSmall, std::string(__func__) + ": workspace too small");
        return attn_rows_forward(A, s);
    }
    return A.a.dtype == MPO_F32 ? attn_simt_forward(A, s) : attn_tc_forward(A, s);
}

int mpo_window_attention_backward(const mpo_attention* args, void* stream) {
    using namespace mpo;
    int st = check_attention(args, true, __func__);
    if (st != kOk) return st;
    MPO_REQUIRE_WORKSPACE(args->workspace);
    cudaStream_t s = (cudaStream_t)stream;
    const AttnArgs A = derive(*args);
    const size_t need = workspace_bytes(A, true);
    if (need && (!args->workspace || args->workspace_bytes < need))
        return fail(kWorkspaceTooSmall, std::string(__func__) + ": workspace too small");
    st = A.a.dtype == MPO_F32 ? attn_simt_backward(A, s) : attn_tc_backward(A, s);
    if (st != kOk || !A.a.grad_table) return st;
    const int entries = A.a.axes * A.a.buckets;
    attn_table_reduce_kernel<<<dim3((unsigned)ceil_div(entries, 32), (unsigned)A.a.heads), 256, 0, s>>>(
        reinterpret_cast<const float*>(static_cast<const unsigned char*>(A.a.workspace) + share_bytes(A)),
        A.a.q_tile_count * partial_blocks_per_tile(A.a), A.a.heads, entries, A.a.grad_table);
    return check_launch("attn_table_reduce_kernel");
}

}  // extern "C"
