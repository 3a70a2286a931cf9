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

// The driver's call that makes a map for the copy engine; the library links only the runtime.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* at = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            at = nullptr;
        return reinterpret_cast<EncodeTiled>(at);
    }();
    return f;
}

// Rows of 16-bit values in boxes of 64 values by [`heads` by] `box` rows, 128-byte swizzle.  dims: values, [heads,] rows.
bool encode_map(CUtensorMap* map, const void* data, int rank, const cuuint64_t* dims, const cuuint64_t* strides, int box, bool bf16, int heads = 1) {
    const cuuint32_t boxes[3] = {64, rank == 3 ? (cuuint32_t)heads : (cuuint32_t)box, (cuuint32_t)box}, steps[3] = {1, 1, 1};
    return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(data), dims,
                          strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Maps for this call, or p.box = 0 where the copy engine cannot follow the layout: blocks must tile 128 keys in
// pieces of whole 1024-byte swizzle groups (8 rows).
void make_maps(AttnParams& p, AttnMaps& maps, bool paged, bool e4m3, int64_t head_dim, bool bf16) {
    p.box = p.q_box = 0;
    const cuuint64_t num_rows = p.batch.num_rows;
    auto strides = [&](const AttnRows& r, int64_t heads, cuuint64_t (&s)[2]) {       // the stride of a dimension of one says nothing
        s[0] = heads > 1 ? r.head_stride : head_dim * 2;
        s[1] = num_rows > 1 ? r.row_stride : head_dim * 2;
    };
    if (encode_tiled() && kTileRows % p.group == 0) {
        const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)p.heads, num_rows};
        cuuint64_t qs[2];
        strides(p.q, p.heads, qs);
        p.q_box = encode_map(&maps.q, p.q.data, 3, dims, qs, kTileRows / p.group, bf16, p.group);
    }
    if (!paged) {
        if (!encode_tiled()) return;
        const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)(p.heads / p.group), num_rows};
        cuuint64_t ks[2], vs[2];
        strides(p.k, p.heads / p.group, ks);
        strides(p.v, p.heads / p.group, vs);
        if (encode_map(&maps.k, p.k.data, 3, dims, ks, kTileKeys, bf16) && encode_map(&maps.v, p.v.data, 3, dims, vs, kTileKeys, bf16)) p.box = kTileKeys;
        return;
    }
    const int bs = p.cache.block_size;
    const int box = bs >= kTileKeys ? (bs % kTileKeys == 0 ? kTileKeys : 0) : (bs % 8 == 0 && kTileKeys % bs == 0 ? bs : 0);
    if (!box || e4m3) {
        p.box = box;
        return;
    }
    const int kv_heads = p.heads / p.group;
    const int64_t rows = (int64_t)p.cache.num_blocks * p.layers * kv_heads * bs;
    if (!encode_tiled() || rows > INT32_MAX) return;
    const int64_t back = (int64_t)p.layer * kv_heads * p.cache.head_stride;          // from this layer to the pool's start
    const cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows}, pitch[1] = {(cuuint64_t)head_dim * 2};
    if (encode_map(&maps.k, p.cache.k - back, 2, dims, pitch, box, bf16) && encode_map(&maps.v, p.cache.v - back, 2, dims, pitch, box, bf16)) p.box = box;
}

template <int HD, bool BF16, bool PAGED, bool E4M3>
int launch_tiles(const AttnParams& params, cudaStream_t stream, const char* what) {
    AttnParams p = params;
    AttnMaps maps = {};
    make_maps(p, maps, PAGED, E4M3, HD, BF16);
    constexpr int smem = TileShape<HD, E4M3>::kShared;
    const int64_t tiles = ((int64_t)std::min(p.batch.max_rows, p.batch.num_rows) * p.group + kBlockRows - 1) / kBlockRows;
    const int64_t grid = std::max<int64_t>(tiles, 1) * (p.heads / p.group) * p.batch.num_seqs;
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many rows for one call", what);
    CU_TRY(cudaFuncSetAttribute(attend_tiles<HD, BF16, PAGED, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attend_tiles<HD, BF16, PAGED, E4M3><<<dim3((unsigned)grid, p.splits), TileShape<HD, E4M3>::kThreads, smem, stream>>>(p, maps);
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
    p.layers = (int32_t)shape->num_layers;
    p.layer = (int32_t)layer;
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
