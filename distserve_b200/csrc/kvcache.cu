// Writing new tokens' K and V rows into one layer of the paged pools and reading sequences back, in the pools' own
// 16-bit type or quantised to e4m3 with a power-of-two scale per row (layout and definition: include/kvmig.h).
//
// Both are copies: what bounds them is HBM for long calls and launch latency for a decoding step's.  A warp works on one
// token, so that sequence, position and block are found once per warp, and takes the token's rows in batches whose loads
// are all issued before the first is used; a token's batches are shared between as many warps as fill the device several
// times over.  Measured: 9.6k tokens of 40 heads quantised in 59.5 us (5.0 TB/s), 34k tokens of 4 heads read back in
// 25.3 us (4.2 TB/s).  Two accesses a batch and blocks of 128 threads were best (1: 61.6 / 25.4 us, 4: 62.6 / 31.2;
// blocks of 256: 59.7 / 26.6); warps that take 4 or 16 neighbouring tokens, so that a tile is read in longer runs, lose
// (71 / 29 us).
#include "kvcache_device.cuh"
#include "kvmig_common.h"

#include <algorithm>
#include <cmath>

namespace kvmig {

int check_rows(const kvmig_rows* r, int64_t head_dim, int64_t num_rows, const char* what) {
    if (!r) return fail(KVMIG_EINVAL, "%s: NULL argument", what);
    if (r->num_heads <= 0 || r->num_heads > (1 << 16)) return fail(KVMIG_EINVAL, "%s: %lld heads", what, (long long)r->num_heads);
    if (num_rows > 0 && !r->data) return fail(KVMIG_EINVAL, "%s: address is NULL", what);
    if ((uintptr_t)r->data % 16) return fail(KVMIG_EINVAL, "%s: address is not a multiple of 16 bytes", what);
    if (r->row_stride % 8 || r->head_stride % 8 || r->row_stride < 0 || r->head_stride < 0)
        return fail(KVMIG_EINVAL, "%s: strides (%lld, %lld) must be non-negative multiples of 8 elements", what,
                    (long long)r->row_stride, (long long)r->head_stride);
    if (r->num_heads > 1 && r->head_stride < head_dim)
        return fail(KVMIG_EINVAL, "%s: head stride %lld is less than head_dim %lld", what, (long long)r->head_stride, (long long)head_dim);
    return 0;
}

int check_batch(const kvmig_batch* b, bool tables, bool lens, const char* what) {
    if (!b) return fail(KVMIG_EINVAL, "%s: batch is NULL", what);
    if (b->num_seqs < 0 || b->num_rows < 0 || b->max_rows < 0) return fail(KVMIG_EINVAL, "%s: negative count in batch", what);
    if (b->num_seqs >= INT32_MAX || b->num_rows > INT32_MAX || b->max_rows > INT32_MAX)
        return fail(KVMIG_ELIMIT, "%s: more than 2^31-1 rows or sequences", what);
    if (b->num_seqs > 0 && (!b->starts || (lens && !b->seq_lens))) return fail(KVMIG_EINVAL, "%s: starts or seq_lens is NULL", what);
    if (tables) {
        if (b->max_blocks < 0 || b->table_stride < b->max_blocks) return fail(KVMIG_EINVAL, "%s: table_stride is less than max_blocks", what);
        if (b->max_blocks > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: more than 2^31-1 blocks in a table", what);
        if (b->num_seqs > 0 && b->max_blocks > 0 && !b->block_tables) return fail(KVMIG_EINVAL, "%s: block_tables is NULL", what);
    }
    return 0;
}

int check_pools(const void* k_cache, const void* v_cache, const kvmig_pool_shape* shape, int64_t layer, int dtype, const char* what) {
    int rc = check_shape(shape, what);
    if (rc) return rc;
    if (dtype != KVMIG_F16 && dtype != KVMIG_BF16) return fail(KVMIG_EINVAL, "%s: unknown dtype %d", what, dtype);
    if (!k_cache || !v_cache) return fail(KVMIG_EINVAL, "%s: a pool pointer is NULL", what);
    if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16) return fail(KVMIG_EINVAL, "%s: a pool's address is not a multiple of 16 bytes", what);
    if (layer < 0 || layer >= shape->num_layers)
        return fail(KVMIG_EINVAL, "%s: layer %lld is outside the pool (%lld layers)", what, (long long)layer, (long long)shape->num_layers);
    if (shape->elem_size != 1 && shape->elem_size != 2)
        return fail(KVMIG_EINVAL, "%s: pools hold 16-bit values or e4m3 codes, not elements of %lld bytes", what, (long long)shape->elem_size);
    const bool quantised = shape->elem_size == 1;
    const int64_t head_dim = shape->head_dim - (quantised ? KVMIG_SCALE_BYTES : 0);
    if (head_dim <= 0 || head_dim % 16 || head_dim > 256)
        return fail(KVMIG_EINVAL, "%s: head_dim %lld is not a multiple of 16 up to 256", what, (long long)head_dim);
    if (quantised && shape->block_size % 4)
        return fail(KVMIG_EINVAL, "%s: block_size %lld of a quantised pool is not a multiple of 4", what, (long long)shape->block_size);
    if (shape->num_heads > (1 << 16) || shape->block_size > (1 << 16))
        return fail(KVMIG_ELIMIT, "%s: more than 65536 heads or token slots in a block", what);
    return 0;
}

namespace {

constexpr int kThreads = 128;

struct RowsView {
    char* data;
    int64_t row_stride, head_stride;   // bytes
};

struct MoveParams {
    RowsView k, v;                     // the rows outside the cache
    CacheView cache;
    BatchView batch;
    int32_t heads, head_dim;
    int32_t parts, batches;            // warps per token, and the batches that they share
};

constexpr int64_t kFillWarps = 148 * 192;
constexpr int kUnroll = 2;             // accesses of a batch, per lane

struct Place {
    int64_t block;                     // byte offset of the block in the pool; -1: there is none, -2: nothing to do here
    int offset;                        // of the token in its block
};

template <bool WRITE>
__device__ __forceinline__ Place find_place(const MoveParams& p, int token) {
    Place at{-2, 0};
    const int i = find_sequence(p.batch.starts, p.batch.num_seqs, token);
    const Sequence s = sequence_at(p.batch, i);
    int64_t pos = (int64_t)token - s.first;
    if (!s.valid || pos < 0 || pos >= s.rows) return at;
    if (WRITE) pos += (int64_t)p.batch.seq_lens[i] - s.rows;
    if (pos < 0) return at;
    const int id = pos <= INT32_MAX ? block_of(p.batch, p.cache, i, (int)pos) : -1;
    if (id < 0) at.block = WRITE ? -2 : -1;
    else at.block = id * p.cache.block_stride;
    at.offset = (int)(pos % p.cache.block_size);
    return at;
}

// 16-bit pools.  A token's K and V are 2 * heads * head_dim / 8 pieces of 16 bytes; a batch is 32 * kUnroll pieces.
template <bool WRITE>
__global__ void __launch_bounds__(kThreads) kv_cache_move(const __grid_constant__ MoveParams p) {
    const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), token = warp / p.parts;
    if (token >= p.batch.num_rows) return;
    const Place at = find_place<WRITE>(p, (int)token);
    if (at.block == -2) return;
    const unsigned per_head = p.head_dim / 8, half = p.heads * per_head, all = 2 * half;
    for (int batch = (int)(warp % p.parts); batch < p.batches; batch += p.parts) {
        uint4 x[kUnroll];
        uint4* to[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            unsigned c = (batch * kUnroll + u) * 32 + (threadIdx.x & 31);
            to[u] = nullptr;
            if (c >= all) continue;
            const bool is_v = c >= half;
            c -= is_v ? half : 0;
            const unsigned head = c / per_head, piece = c % per_head;
            const RowsView& r = is_v ? p.v : p.k;
            char* row = r.data + token * r.row_stride + head * r.head_stride + piece * 16;
            char* cached = (is_v ? p.cache.v : p.cache.k) + at.block + (int64_t)head * p.cache.head_stride + (int64_t)at.offset * p.head_dim * 2 + piece * 16;
            to[u] = reinterpret_cast<uint4*>(WRITE ? cached : row);
            x[u] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);       // NaN in both types
            if (WRITE || at.block >= 0) x[u] = __ldcs(reinterpret_cast<const uint4*>(WRITE ? row : cached));
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (to[u]) *to[u] = x[u];
    }
}

// Quantised pools.  A lane has 16 values of a row in two pieces of 8, a row is a group of `width` lanes (head_dim / 16
// rounded up to a power of two), so that its largest magnitude needs no shared memory, and a batch is kUnroll rows for
// each group of lanes.
template <bool WRITE, bool BF16>
__global__ void __launch_bounds__(kThreads) kv_cache_move_e4m3(const __grid_constant__ MoveParams p, int width) {
    using H = Half<BF16>;
    const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), token = warp / p.parts;
    if (token >= p.batch.num_rows) return;
    const Place at = find_place<WRITE>(p, (int)token);
    if (at.block == -2) return;
    const int lane = threadIdx.x & 31, sub = lane & (width - 1), group = lane / width, groups = 32 / width;
    const bool active = sub * 16 < p.head_dim;
    const int second = p.head_dim / 2;                              // of the lane's pieces: where it begins, in values
    const int all = 2 * p.heads;
    const int64_t scales_at = (int64_t)p.cache.block_size * p.head_dim;
    for (int batch = (int)(warp % p.parts); batch < p.batches; batch += p.parts) {
        uint4 a[kUnroll], b[kUnroll];                               // write: the row's pieces; read: a.xy and b.xy, the codes
        float scale[kUnroll];
        char *row[kUnroll], *codes[kUnroll];                        // the lane's pieces outside the cache and in it
        float* scale_at[kUnroll];
        bool there[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            int r = (batch * kUnroll + u) * groups + group;
            there[u] = r < all && active;
            const bool is_v = r >= p.heads;
            r -= is_v ? p.heads : 0;
            const RowsView& rows = is_v ? p.v : p.k;
            row[u] = rows.data + token * rows.row_stride + r * rows.head_stride + sub * 16;
            char* tile = (is_v ? p.cache.v : p.cache.k) + at.block + (int64_t)r * p.cache.head_stride;
            codes[u] = tile + (int64_t)at.offset * p.head_dim + sub * 8;
            scale_at[u] = reinterpret_cast<float*>(tile + scales_at) + at.offset;
            a[u] = b[u] = make_uint4(0, 0, 0, 0);
            scale[u] = 0.f;
            if (WRITE && there[u]) {
                a[u] = __ldcs(reinterpret_cast<const uint4*>(row[u]));
                b[u] = __ldcs(reinterpret_cast<const uint4*>(row[u] + second * 2));
            } else if (there[u] && at.block >= 0) {
                const uint2 lo = __ldg(reinterpret_cast<const uint2*>(codes[u])), hi = __ldg(reinterpret_cast<const uint2*>(codes[u] + second));
                a[u].x = lo.x;
                a[u].y = lo.y;
                b[u].x = hi.x;
                b[u].y = hi.y;
                scale[u] = __ldg(scale_at[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (WRITE) {
                const uint32_t w[8] = {a[u].x, a[u].y, a[u].z, a[u].w, b[u].x, b[u].y, b[u].z, b[u].w};
                uint32_t top = 0;                                   // of magnitudes as bit patterns: a NaN is larger than everything
#pragma unroll
                for (int j = 0; j < 8; ++j) top = __vmaxu2(top, w[j] & 0x7fff7fffu);
                for (int d = width >> 1; d; d >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
                top = max(top & 0xffffu, top >> 16);
                float inverse;
                const float s = row_scale<BF16>(top, &inverse);
                uint32_t out[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 lo = H::to_float2(w[2 * j]), hi = H::to_float2(w[2 * j + 1]);
                    out[j] = encode4(lo.x * inverse, lo.y * inverse, hi.x * inverse, hi.y * inverse);
                }
                if (!there[u]) continue;
                *reinterpret_cast<uint2*>(codes[u]) = make_uint2(out[0], out[1]);
                *reinterpret_cast<uint2*>(codes[u] + second) = make_uint2(out[2], out[3]);
                if (sub == 0) *scale_at[u] = s;
            } else if (there[u]) {
                uint4 lo, hi;
                widen16<BF16>(make_uint4(a[u].x, a[u].y, b[u].x, b[u].y), scale[u], lo, hi);
                if (at.block < 0) lo = hi = make_uint4(H::kNan2, H::kNan2, H::kNan2, H::kNan2);
                *reinterpret_cast<uint4*>(row[u]) = lo;
                *reinterpret_cast<uint4*>(row[u] + second * 2) = hi;
            }
        }
    }
}

template <bool WRITE>
int move_rows(const kvmig_rows* k, const kvmig_rows* v, int dtype, void* k_cache, void* v_cache, const kvmig_pool_shape* shape,
              int64_t layer, const kvmig_batch* batch, cudaStream_t stream) {
    const char* what = WRITE ? "cache_write" : "cache_read";
    int rc = check_pools(k_cache, v_cache, shape, layer, dtype, what);
    if (!rc) rc = check_batch(batch, true, WRITE, what);
    if (rc) return rc;
    const bool quantised = shape->elem_size == 1;
    const int64_t head_dim = shape->head_dim - (quantised ? KVMIG_SCALE_BYTES : 0);
    if (!(rc = check_rows(k, head_dim, batch->num_rows, WRITE ? "cache_write: k" : "cache_read: k_out")))
        rc = check_rows(v, head_dim, batch->num_rows, WRITE ? "cache_write: v" : "cache_read: v_out");
    if (rc) return rc;
    if (k->num_heads != shape->num_heads || v->num_heads != shape->num_heads)
        return fail(KVMIG_EINVAL, "%s: the rows have %lld and %lld heads, the pools %lld", what, (long long)k->num_heads,
                    (long long)v->num_heads, (long long)shape->num_heads);
    int dev;
    CU_TRY(cudaGetDevice(&dev));
    if (batch->num_rows == 0 || batch->num_seqs == 0) return 0;
    MoveParams p;
    auto view = [](const kvmig_rows* r) { return RowsView{static_cast<char*>(r->data), r->row_stride * 2, r->head_stride * 2}; };
    p.k = view(k);
    p.v = view(v);
    const int64_t tile = shape->block_size * shape->head_dim * shape->elem_size;
    const int64_t at_layer = layer * shape->num_heads * tile;
    p.cache = CacheView{static_cast<char*>(k_cache) + at_layer, static_cast<char*>(v_cache) + at_layer,
                        shape->num_layers * shape->num_heads * tile, (int32_t)tile, (int32_t)shape->num_blocks,
                        (int32_t)shape->block_size};
    p.batch = BatchView{batch->starts, batch->seq_lens, batch->block_tables, batch->table_stride, (int32_t)batch->num_seqs,
                        (int32_t)batch->num_rows, (int32_t)batch->max_rows, (int32_t)batch->max_blocks};
    p.heads = (int32_t)shape->num_heads;
    p.head_dim = (int32_t)head_dim;
    int width = 1;
    while (width * 16 < head_dim) width *= 2;
    const int64_t pieces = quantised ? 2 * shape->num_heads : 2 * shape->num_heads * head_dim / 8;
    const int64_t per_batch = kUnroll * (quantised ? 32 / width : 32);
    p.batches = (int32_t)((pieces + per_batch - 1) / per_batch);
    p.parts = (int32_t)std::min<int64_t>(p.batches, std::max<int64_t>(kFillWarps / batch->num_rows, 1));
    const int64_t grid = (batch->num_rows * p.parts + kThreads / 32 - 1) / (kThreads / 32);
    if (grid > INT32_MAX) return fail(KVMIG_ELIMIT, "%s: too many rows for one call", what);
    if (!quantised) kv_cache_move<WRITE><<<(unsigned)grid, kThreads, 0, stream>>>(p);
    else if (dtype == KVMIG_BF16) kv_cache_move_e4m3<WRITE, true><<<(unsigned)grid, kThreads, 0, stream>>>(p, width);
    else kv_cache_move_e4m3<WRITE, false><<<(unsigned)grid, kThreads, 0, stream>>>(p, width);
    CU_TRY(cudaGetLastError());
    g_cache_launches++;
    return 0;
}

}  // namespace

}  // namespace kvmig

using namespace kvmig;

extern "C" {

int kvmig_cache_write(const kvmig_rows* k, const kvmig_rows* v, int dtype, void* k_cache, void* v_cache,
                      const kvmig_pool_shape* shape, int64_t layer, const kvmig_batch* batch, void* stream) {
    clear_error();
    return move_rows<true>(k, v, dtype, k_cache, v_cache, shape, layer, batch, static_cast<cudaStream_t>(stream));
}

int kvmig_cache_read(void* k_cache, void* v_cache, const kvmig_pool_shape* shape, int64_t layer, const kvmig_batch* batch,
                     const kvmig_rows* k_out, const kvmig_rows* v_out, int dtype, void* stream) {
    clear_error();
    return move_rows<false>(k_out, v_out, dtype, k_cache, v_cache, shape, layer, batch, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
