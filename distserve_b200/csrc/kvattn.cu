// Causal attention of new tokens over the paged cache, and of whole packed prompts.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - m),   m = max_j (scale q . k_j)
//
// in one pass over the keys: when the running maximum grows from m to m', what has been summed so far is multiplied
// by exp(m - m').
#include "kvattn_few.cuh"
#include "kvattn_tile.cuh"
#include "kvmig_common.h"

#include <algorithm>
#include <cmath>

namespace kvmig {
namespace {

// Blocks that the device holds at once when two share an SM (B200: 148 SMs).
constexpr int64_t kResident = 2 * 148;

// Up to 16 rows of a sequence share a KV head: the kernel for few rows.
bool few_rows(int64_t max_rows, int64_t group) { return max_rows * group <= kFewRows; }

// Parts that a sequence's keys are cut into: as many as fill the device, but none shorter than 256 keys of what the
// block tables have room for.
int64_t splits_for(int64_t tiles, int64_t capacity) {
    const int64_t fill = kResident / std::max<int64_t>(tiles, 1), longest = std::max<int64_t>(capacity / 256, 1);
    return std::max<int64_t>(1, std::min(std::min(fill, longest), (int64_t)256));
}

struct PagedPlan {
    bool few;
    int64_t splits, workspace;
};

PagedPlan plan_paged(const kvmig_pool_shape* shape, int64_t heads, const kvmig_batch* b) {
    PagedPlan plan = {};
    plan.few = few_rows(b->max_rows, heads / shape->num_heads);
    const int64_t capacity = std::min<int64_t>(b->max_blocks * shape->block_size, INT32_MAX);
    if (plan.few) {
        plan.splits = splits_for(b->num_seqs * shape->num_heads, capacity);
    } else {
        const int64_t tiles = (b->num_rows * (heads / shape->num_heads) / kBlockRows + b->num_seqs) * shape->num_heads;
        plan.splits = splits_for(2 * tiles, capacity);        // a block has an SM to itself
    }
    const int64_t head_dim = shape->head_dim - (shape->elem_size == 1 ? KVMIG_SCALE_BYTES : 0);
    if (plan.splits > 1) plan.workspace = b->num_rows * heads * plan.splits * (head_dim * 4 + (int64_t)sizeof(float2));
    return plan;
}

BatchView batch_view(const kvmig_batch* batch) {
    return BatchView{batch->starts, batch->seq_lens, batch->block_tables, batch->table_stride, (int32_t)batch->num_seqs,
                     (int32_t)batch->num_rows, (int32_t)batch->max_rows, (int32_t)batch->max_blocks};
}

template <int HD, bool BF16, bool E4M3>
int launch_few(const AttnParams& p, unsigned grid, cudaStream_t stream) {
    constexpr int smem = FewShape<HD, E4M3>::kShared;
    CU_TRY(cudaFuncSetAttribute(attend_few<HD, BF16, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attend_few<HD, BF16, E4M3><<<dim3(grid, p.splits), kFewWarps * 32, smem, stream>>>(p);
    CU_TRY(cudaGetLastError());
    g_attention_launches++;
    return 0;
}

template <int HD, bool BF16, bool PAGED, bool E4M3>
int launch_tiles(const AttnParams& p, cudaStream_t stream, const char* what) {
    constexpr int smem = TileShape<HD, E4M3>::kShared;
    const int64_t tiles = ((int64_t)std::min(p.batch.max_rows, p.batch.num_rows) * p.group + kBlockRows - 1) / kBlockRows;
    const int64_t grid = std::max<int64_t>(tiles, 1) * (p.heads / p.group) * p.batch.num_seqs;
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many rows for one call", what);
    CU_TRY(cudaFuncSetAttribute(attend_tiles<HD, BF16, PAGED, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attend_tiles<HD, BF16, PAGED, E4M3><<<dim3((unsigned)grid, p.splits), kTileThreads, smem, stream>>>(p);
    CU_TRY(cudaGetLastError());
    g_attention_launches++;
    return 0;
}

template <int HD, bool BF16>
int launch(const AttnParams& p, bool paged, bool e4m3, bool few, cudaStream_t stream, const char* what) {
    int rc;
    if (few) {
        const int64_t grid = (int64_t)p.batch.num_seqs * (p.heads / p.group);
        if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many sequences for one call", what);
        rc = e4m3 ? launch_few<HD, BF16, true>(p, (unsigned)grid, stream) : launch_few<HD, BF16, false>(p, (unsigned)grid, stream);
    } else if (!paged) {
        rc = launch_tiles<HD, BF16, false, false>(p, stream, what);
    } else {
        rc = e4m3 ? launch_tiles<HD, BF16, true, true>(p, stream, what) : launch_tiles<HD, BF16, true, false>(p, stream, what);
    }
    if (rc || p.splits == 1) return rc;
    const int64_t grid = ((int64_t)p.batch.num_rows * p.heads + 3) / 4;
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many rows for one call", what);
    attend_join<HD, BF16><<<(unsigned)grid, 128, 0, stream>>>(p);
    CU_TRY(cudaGetLastError());
    g_attention_launches++;
    return 0;
}

int attend(AttnParams& p, bool paged, bool e4m3, bool few, int64_t head_dim, int dtype, const kvmig_batch* batch, cudaStream_t stream,
           const char* what) {
    p.batch = batch_view(batch);
    int dev;
    CU_TRY(cudaGetDevice(&dev));
    if (batch->num_rows == 0 || batch->num_seqs == 0) return 0;
    if (head_dim == 64)
        return dtype == KVMIG_F16 ? launch<64, false>(p, paged, e4m3, few, stream, what) : launch<64, true>(p, paged, e4m3, few, stream, what);
    return dtype == KVMIG_F16 ? launch<128, false>(p, paged, e4m3, few, stream, what) : launch<128, true>(p, paged, e4m3, few, stream, what);
}

AttnRows view(const kvmig_rows* r) { return AttnRows{static_cast<char*>(r->data), r->row_stride * 2, r->head_stride * 2}; }

// Checks that the two attention entry points share.
int check_attention(const kvmig_rows* q, const kvmig_rows* out, int64_t head_dim, int64_t kv_heads, const kvmig_batch* batch,
                    double scale, const char* what) {
    if (head_dim != 64 && head_dim != 128) return fail(KVMIG_EINVAL, "%s: head_dim %lld is neither 64 nor 128", what, (long long)head_dim);
    int rc = check_rows(q, head_dim, batch->num_rows, what);
    if (!rc) rc = check_rows(out, head_dim, batch->num_rows, what);
    if (rc) return rc;
    if (q->num_heads != out->num_heads) return fail(KVMIG_EINVAL, "%s: q has %lld heads, out %lld", what, (long long)q->num_heads, (long long)out->num_heads);
    if (q->num_heads % kv_heads)
        return fail(KVMIG_EINVAL, "%s: %lld query heads do not split over %lld KV heads", what, (long long)q->num_heads, (long long)kv_heads);
    if (!std::isfinite((float)scale * 1.4426950408889634f)) return fail(KVMIG_EINVAL, "%s: scale is not finite", what);
    return 0;
}

}  // namespace

int64_t attention_timeouts() {
    unsigned n = 0;
    return cudaMemcpyFromSymbol(&n, g_attention_timeouts, sizeof n) == cudaSuccess ? (int64_t)n : -1;
}

}  // namespace kvmig

using namespace kvmig;

extern "C" {

int64_t kvmig_paged_attention_workspace(const kvmig_pool_shape* shape, int64_t num_q_heads, const kvmig_batch* batch) {
    clear_error();
    int rc = check_shape(shape, "paged_attention_workspace");
    if (!rc) rc = check_batch(batch, false, false, "paged_attention_workspace");
    if (rc) return rc;
    if (batch->max_blocks < 0 || batch->max_blocks > INT32_MAX || shape->block_size > (1 << 16) || shape->num_heads > (1 << 16) ||
        num_q_heads > (1 << 16))
        return fail(KVMIG_ELIMIT, "paged_attention_workspace: max_blocks, block_size or heads out of range");
    if (num_q_heads <= 0 || num_q_heads % shape->num_heads)
        return fail(KVMIG_EINVAL, "paged_attention_workspace: %lld query heads do not split over %lld KV heads", (long long)num_q_heads,
                    (long long)shape->num_heads);
    return plan_paged(shape, num_q_heads, batch).workspace;
}

int kvmig_paged_attention(const kvmig_rows* q, const kvmig_rows* out, int dtype, void* k_cache, void* v_cache,
                          const kvmig_pool_shape* shape, int64_t layer, const kvmig_batch* batch, double scale, void* workspace,
                          int64_t workspace_bytes, void* stream) {
    clear_error();
    const char* what = "paged_attention";
    int rc = check_pools(k_cache, v_cache, shape, layer, dtype, what);
    if (!rc) rc = check_batch(batch, true, true, what);
    if (rc) return rc;
    const bool e4m3 = shape->elem_size == 1;
    const int64_t head_dim = shape->head_dim - (e4m3 ? KVMIG_SCALE_BYTES : 0);
    rc = check_attention(q, out, head_dim, shape->num_heads, batch, scale, what);
    if (rc) return rc;
    const int64_t need = kvmig_paged_attention_workspace(shape, q->num_heads, batch);
    if (need < 0) return (int)need;
    if (workspace_bytes < need || (need > 0 && (!workspace || (uintptr_t)workspace % 16)))
        return fail(KVMIG_EINVAL, "%s: needs a workspace of %lld bytes at a multiple of 16", what, (long long)need);
    AttnParams p = {};
    p.q = view(q);
    p.out = view(out);
    const int64_t tile = shape->block_size * shape->head_dim * shape->elem_size, at_layer = layer * shape->num_heads * tile;
    p.cache = CacheView{static_cast<char*>(k_cache) + at_layer, static_cast<char*>(v_cache) + at_layer,
                        shape->num_layers * shape->num_heads * tile, (int32_t)tile, (int32_t)shape->num_blocks,
                        (int32_t)shape->block_size};
    p.heads = (int32_t)q->num_heads;
    p.group = (int32_t)(q->num_heads / shape->num_heads);
    p.scale_log2 = (float)(scale * 1.4426950408889634);
    const PagedPlan plan = plan_paged(shape, q->num_heads, batch);
    p.splits = (int32_t)plan.splits;
    p.part_out = static_cast<float*>(workspace);
    p.part_stat = reinterpret_cast<float2*>(p.part_out + batch->num_rows * q->num_heads * plan.splits * head_dim);
    return attend(p, true, e4m3, plan.few, head_dim, dtype, batch, static_cast<cudaStream_t>(stream), what);
}

int kvmig_prompt_attention(const kvmig_rows* q, const kvmig_rows* k, const kvmig_rows* v, const kvmig_rows* out, int dtype,
                           int64_t head_dim, const kvmig_batch* batch, double scale, void* stream) {
    clear_error();
    const char* what = "prompt_attention";
    int rc = check_batch(batch, false, false, what);
    if (rc) return rc;
    if (dtype != KVMIG_F16 && dtype != KVMIG_BF16) return fail(KVMIG_EINVAL, "%s: unknown dtype %d", what, dtype);
    if (!(rc = check_rows(k, head_dim, batch->num_rows, what))) rc = check_rows(v, head_dim, batch->num_rows, what);
    if (rc) return rc;
    if (k->num_heads != v->num_heads)
        return fail(KVMIG_EINVAL, "%s: k has %lld heads, v %lld", what, (long long)k->num_heads, (long long)v->num_heads);
    rc = check_attention(q, out, head_dim, k->num_heads, batch, scale, what);
    if (rc) return rc;
    AttnParams p = {};
    p.q = view(q);
    p.out = view(out);
    p.k = view(k);
    p.v = view(v);
    p.heads = (int32_t)q->num_heads;
    p.group = (int32_t)(q->num_heads / k->num_heads);
    p.scale_log2 = (float)(scale * 1.4426950408889634);
    p.splits = 1;
    return attend(p, false, false, false, head_dim, dtype, batch, static_cast<cudaStream_t>(stream), what);
}

}  // extern "C"
