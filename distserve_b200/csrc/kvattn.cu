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

constexpr int64_t kSms = 148;      // of a B200

// How a paged call is run.  Sequences with up to few_most() rows per KV head go to the kernel for few rows (all of them if
// none can have more), the others to the tile kernel; one of the two is launched if the batch can be seen to need only
// that one.
struct PagedPlan {
    bool few, tiles, wide;             // wide: blocks of 8 warps instead of 4 for few rows
    int64_t few_rows, few_tile, parts, workspace;
    SplitRule few_rule, tile_rule;
};

// Row tiles of the tile kernel, of one KV head, that the batch can have.
int64_t most_tiles(int64_t num_rows, int64_t num_seqs, int64_t max_rows, int64_t group) {
    return std::min(num_rows * group / kBlockRows + num_seqs, num_seqs * ((std::min(max_rows, num_rows) * group + kBlockRows - 1) / kBlockRows));
}

PagedPlan plan_paged(const kvmig_pool_shape* shape, int64_t heads, const kvmig_batch* b) {
    PagedPlan plan = {};
    const int64_t group = heads / shape->num_heads, most = std::min(b->max_rows, b->num_rows) * group;
    const int64_t capacity = std::min<int64_t>(b->max_blocks * shape->block_size, INT32_MAX), units = (capacity + kSplitKeys - 1) / kSplitKeys;
    const int64_t bound = few_most(shape->elem_size == 1);
    plan.tiles = most > bound;
    // rows for every sequence to have its most: as good as certain that all have many
    plan.few = !plan.tiles || b->num_rows < b->num_seqs * b->max_rows;
    plan.few_rows = !plan.tiles ? INT64_MAX : plan.few ? bound : 0;
    plan.few_tile = most <= 16 ? 16 : 32;
    const int64_t kv_heads = shape->num_heads, head_dim = shape->head_dim - (shape->elem_size == 1 ? KVMIG_SCALE_BYTES : 0);
    // A part is about the call's work over the blocks that the device holds at once (part_units): the device adds the
    // work up, the host sees to room for the parts of the longest sequence if the others are a quarter as long, with
    // partial results below 256 MB.
    const int64_t room = std::max<int64_t>((256 << 20) / std::max<int64_t>(b->num_rows * heads * (head_dim * 4 + 8), 1), 1);
    auto rule = [&](int64_t blocks, int64_t least, int64_t row_tiles) {
        const double n = std::max<int64_t>(b->num_seqs, 1), work = (double)row_tiles * kv_heads * units * (n + 3) / (4 * n);
        const int64_t part = std::max(least, (int64_t)std::min(work / blocks, (double)units) + 1);
        // joining takes a launch of its own, which two parts of a short sequence are not worth
        const int64_t parts = units <= 2 * least ? 1 : std::min((units + part - 1) / part, room);
        return SplitRule{(int32_t)std::max<int64_t>(parts, 1), (int32_t)least, (int32_t)blocks, 0};
    };
    plan.few_rule = plan.tile_rule = SplitRule{1, 1, 1, 0};
    if (plan.few) {
        const int64_t tiles = b->num_seqs * ((std::min(most, bound) + plan.few_tile - 1) / plan.few_tile);
        // beside sequences of the tile kernel there are fewer of this one's than the batch has: as if it were one
        plan.few_rule = rule(2 * kSms, 2, plan.tiles ? 1 : tiles);
        // More row tiles than half of what runs at once: cut so that the last of the waves is full, two extra units being what
        // a part costs, if that saves a tenth.
        const int64_t slots = plan.few_rule.blocks, all = tiles * kv_heads;
        if (!plan.tiles && 2 * all >= slots) {
            auto cost = [&](int64_t k) { return (double)((all * k + slots - 1) / slots) * ((double)units / k + 2); };
            int64_t best = 1;
            for (int64_t k = 2; k <= 8 && units / k >= 4 && 2 * k <= room; ++k)
                if (cost(k) < 0.9 * cost(1) && cost(k) < cost(best)) best = k;
            plan.few_rule = SplitRule{best > 1 ? (int32_t)(2 * best) : 1, 4, (int32_t)slots, best > 1 ? (int32_t)best : 0};
        }
        // short sequences that nobody shares: more warps for each
        plan.wide = plan.few_rule.parts == 1 && tiles * kv_heads <= kSms;
    }
    // A block of the tile kernel has an SM to itself; the device chooses how to cut (tile_units).  Up to 2048 keys that is not
    // worth the choice and the join where the rows fill the SMs anyway (32 sequences of 1032 tokens, 32 of them new, 64/8
    // heads: 60.7 us, 72.8 with them).
    if (plan.tiles && (units > 16 || b->num_rows * group / kBlockRows * kv_heads < kSms))
        plan.tile_rule = rule(2 * kSms, 4, most_tiles(b->num_rows, b->num_seqs, b->max_rows, group));
    plan.parts = std::max(plan.few_rule.parts, plan.tile_rule.parts);
    if (plan.parts > 1) plan.workspace = b->num_rows * heads * plan.parts * (head_dim * 4 + (int64_t)sizeof(float2)) + 2 * (int64_t)sizeof(int32_t);
    return plan;
}

BatchView batch_view(const kvmig_batch* batch) {
    return BatchView{batch->starts, batch->seq_lens, batch->block_tables, batch->table_stride, (int32_t)batch->num_seqs,
                     (int32_t)batch->num_rows, (int32_t)batch->max_rows, (int32_t)batch->max_blocks};
}

// Launches a grid that may begin, if `early`, once every block of the stream's previous grid has begun.
template <typename... Args>
cudaError_t launch_early(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, bool early, cudaStream_t stream, const Args&... args) {
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// Blocks for all the parts that up to `tiles` row tiles can be cut into (see part_units), a multiple of the KV heads.
int64_t blocks_for(SplitRule rule, int64_t tiles, int64_t kv_heads) {
    if (rule.parts == 1) return tiles;
    if (rule.cuts > 0) return std::min<int64_t>(rule.cuts + 1, rule.parts) * tiles;
    const int64_t cut = std::max<int64_t>(rule.blocks, rule.blocks / 2 + tiles);
    return (std::min(cut, tiles * rule.parts) + kv_heads - 1) / kv_heads * kv_heads;
}

template <int HD, bool BF16, bool E4M3, int MT, int WARPS>
int launch_few(const AttnParams& p, cudaStream_t stream, const char* what) {
    constexpr int smem = FewShape<HD, E4M3, MT, WARPS>::kShared, rows = FewShape<HD, E4M3, MT, WARPS>::kRows;
    const int64_t most = std::min((int64_t)std::min(p.batch.max_rows, p.batch.num_rows) * p.group, p.few_rows);
    const int64_t kv_heads = p.heads / p.group, tiles = (int64_t)p.batch.num_seqs * kv_heads * std::max<int64_t>((most + rows - 1) / rows, 1);
    const int64_t grid = blocks_for(p.few, tiles, kv_heads);
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many sequences for one call", what);
    CU_TRY(cudaFuncSetAttribute(attend_few<HD, BF16, E4M3, MT, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attend_few<HD, BF16, E4M3, MT, WARPS><<<(unsigned)grid, WARPS * 32, smem, stream>>>(p);
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
// Rows that overlap (a stride of 0, one row standing for all) are not the copy engine's.
bool encode_map(CUtensorMap* map, const void* data, int rank, const cuuint64_t* dims, const cuuint64_t* strides, int box, bool bf16, int heads = 1) {
    for (int i = 0; i < rank - 1; ++i)
        if (strides[i] < dims[0] * 2) return false;
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
int launch_tiles(const AttnParams& params, bool after_few, cudaStream_t stream, const char* what) {
    AttnParams p = params;
    AttnMaps maps = {};
    make_maps(p, maps, PAGED, E4M3, HD, BF16);
    constexpr int smem = TileShape<HD, E4M3>::kShared;
    const int64_t kv_heads = p.heads / p.group, tiles = std::max<int64_t>(most_tiles(p.batch.num_rows, p.batch.num_seqs, p.batch.max_rows, p.group), p.batch.num_seqs) * kv_heads;
    const int64_t some = (p.tiles.blocks + kv_heads - 1) / kv_heads * kv_heads;                     // tile_units: no more pieces than this, or tiles
    const int64_t grid = p.batch.num_seqs > 32 ? blocks_for(p.tiles, tiles, kv_heads) : std::max(tiles, std::min(some, tiles * p.tiles.parts));
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many rows for one call", what);
    CU_TRY(cudaFuncSetAttribute(attend_tiles<HD, BF16, PAGED, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    // After the kernel for few rows, which has other rows to do: begins when that one's blocks leave room.
    CU_TRY(launch_early(attend_tiles<HD, BF16, PAGED, E4M3>, dim3((unsigned)grid), TileShape<HD, E4M3>::kThreads, smem, after_few,
                        stream, p, maps));
    g_attention_launches++;
    return 0;
}

template <int HD, bool BF16, bool E4M3>
int launch_paged(const AttnParams& p, const PagedPlan& plan, cudaStream_t stream, const char* what) {
    int rc = 0;
    if (plan.few) {
        if (plan.wide) rc = p.few_tile == 16 ? launch_few<HD, BF16, E4M3, 1, 8>(p, stream, what) : launch_few<HD, BF16, E4M3, 2, 8>(p, stream, what);
        else rc = p.few_tile == 16 ? launch_few<HD, BF16, E4M3, 1, 4>(p, stream, what) : launch_few<HD, BF16, E4M3, 2, 4>(p, stream, what);
    }
    if (!rc && plan.tiles) rc = launch_tiles<HD, BF16, true, E4M3>(p, plan.few, stream, what);
    if (rc || p.parts == 1) return rc;
    // A block for each result while they fit the device at once, else a warp for each.
    const int64_t items = (int64_t)p.batch.num_rows * p.heads, most = 8 * kSms;
    const bool wide = items <= most;
    CU_TRY(launch_early(wide ? attend_join<HD, BF16, true> : attend_join<HD, BF16, false>,
                        dim3((unsigned)std::min(wide ? items : (items + kJoinWarps - 1) / kJoinWarps, most)), kJoinThreads, 0, true, stream, p));
    g_attention_launches++;
    return 0;
}

template <int HD, bool BF16>
int launch(const AttnParams& p, const PagedPlan* plan, bool e4m3, cudaStream_t stream, const char* what) {
    if (!plan) return launch_tiles<HD, BF16, false, false>(p, false, stream, what);
    return e4m3 ? launch_paged<HD, BF16, true>(p, *plan, stream, what) : launch_paged<HD, BF16, false>(p, *plan, stream, what);
}

int attend(AttnParams& p, const PagedPlan* plan, bool e4m3, int64_t head_dim, int dtype, const kvmig_batch* batch, cudaStream_t stream,
           const char* what) {
    p.batch = batch_view(batch);
    int dev;
    CU_TRY(cudaGetDevice(&dev));
    if (batch->num_rows == 0 || batch->num_seqs == 0) return 0;
    if (head_dim == 64)
        return dtype == KVMIG_F16 ? launch<64, false>(p, plan, e4m3, stream, what) : launch<64, true>(p, plan, e4m3, stream, what);
    return dtype == KVMIG_F16 ? launch<128, false>(p, plan, e4m3, stream, what) : launch<128, true>(p, plan, e4m3, stream, what);
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
    p.few_rows = plan.few_rows;
    p.few = plan.few_rule;
    p.tiles = plan.tile_rule;
    p.few_tile = (int32_t)plan.few_tile;
    p.parts = (int32_t)plan.parts;
    p.few_followed = plan.tiles || plan.parts > 1;
    p.tiles_followed = plan.parts > 1;
    p.part_out = static_cast<float*>(workspace);
    p.part_stat = reinterpret_cast<float2*>(p.part_out + batch->num_rows * q->num_heads * plan.parts * head_dim);
    p.part_chosen = reinterpret_cast<int32_t*>(p.part_stat + batch->num_rows * q->num_heads * plan.parts);
    return attend(p, &plan, e4m3, head_dim, dtype, batch, static_cast<cudaStream_t>(stream), what);
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
    p.parts = 1;
    p.few = p.tiles = SplitRule{1, 1, 1, 0};
    return attend(p, nullptr, false, head_dim, dtype, batch, static_cast<cudaStream_t>(stream), what);
}

}  // extern "C"
