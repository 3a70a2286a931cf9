// The loading warps of the tensor-core attention kernels: they fill a ring of 128-key tiles, K and V in turn, in the layout
// that the products read (columns of 64 values, 128-byte rows, swizzled).
//
// Tiles go through the copy engine, a box for each block and 64 values, or, from quantised pools, as bulk copies of codes
// and scales into a second ring, whose tiles these warps then widen to 16 bits.  What lies behind the last key of a part
// comes along with its block, but may be anything: the softmax masks its scores, and its values V are overwritten with
// zeros here.  Block sizes that do not tile 128 keys are copied 16 bytes at a time, zeros where there is no key.
#pragma once

#include "kvattn_device.cuh"
#include "tcgen05.cuh"

namespace kvmig {

constexpr int kTileKeys = 128;

// Byte offset of 16-byte piece j of row r in a tile.
__device__ __forceinline__ uint32_t tile_offset(int r, int j) {
    return (uint32_t)((j >> 3) * (kTileKeys * 128) + r * 128 + (((j & 7) ^ (r & 7)) << 4));
}

// Codes are widened as kvmig_cache_read gives them, in the rows' type.
template <int HD, bool BF16, bool PAGED, bool E4M3, int WARPS, int SLOTS, int RAW_SLOTS>
struct TileLoader {
    static constexpr int kSlot = kTileKeys * HD * 2, kRawSlot = kTileKeys * (HD + 4);
    static constexpr int kPieces = HD / 8, kRowsAtOnce = 32 / kPieces;        // of a 16-bit row; rows that a warp copies at once
    static constexpr int kRowPieces = HD / 16, kRawRows = 32 / kRowPieces;    // the same for codes
    static constexpr int kPerBox = E4M3 ? 2 : HD / 64;
    static constexpr int kLag = 2;                                            // tiles copied piecewise that may be in flight

    const AttnParams& p;
    const AttnMaps& maps;
    const int w, lane, seq, kv_head, first_row, begin, end;
    unsigned char *const ring, *const raw;
    const uint32_t full, empty, raw_full, raw_empty, tail;
    volatile int* const flags;
    bool bad = false, ok = true;             // a block that is not there; no wait has run out
    int issued = 0;                          // tiles that the copy engine was given

    // The engine's copies of a paged tile are dealt over the loading warps, one to a lane: box `box_of` of the tile and its
    // left or right 64 values (codes or scales for quantised pools).  Block ids are read a step ahead.
    int box_of, part_of, id = -2, ahead = -2;    // -2: no copy, -1: no such block
    bool dealt;
    int64_t at_k[4], at_v[4];                // byte offsets of four keys of a tile, r = lane + 32 x; -1 if there is no such key

    __device__ __forceinline__ TileLoader(const AttnParams& p_, const AttnMaps& maps_, int w_, int seq_, int kv_head_, int first_row_, int begin_,
                                          int end_, unsigned char* ring_, unsigned char* raw_, uint32_t full_, uint32_t empty_, uint32_t raw_full_,
                                          uint32_t raw_empty_, uint32_t tail_, volatile int* flags_)
        : p(p_), maps(maps_), w(w_), lane(threadIdx.x & 31), seq(seq_), kv_head(kv_head_), first_row(first_row_), begin(begin_), end(end_),
          ring(ring_), raw(raw_), full(full_), empty(empty_), raw_full(raw_full_), raw_empty(raw_empty_), tail(tail_), flags(flags_) {
        const int deal = lane * WARPS + w;
        box_of = deal / kPerBox;
        part_of = deal % kPerBox;
        dealt = PAGED && p.box > 0 && box_of < kTileKeys / max(p.box, 1);
    }

    __device__ __forceinline__ bool by_engine() const { return p.box > 0; }
    __device__ __forceinline__ int keys_of(int c) const { return min(end - begin - c / 2 * kTileKeys, kTileKeys); }     // keys that tile c has

    __device__ __forceinline__ void look_ahead(int i) {
        const int key = begin + i * kTileKeys + box_of * p.box;
        ahead = -2;
        if (!dealt || key >= end) return;
        const int entry = key / p.cache.block_size;
        ahead = entry < p.batch.max_blocks ? p.batch.block_tables[seq * p.batch.table_stride + entry] : -1;
        if (ahead == -2) ahead = -1;
    }

    // This lane's copy of tile c has a source.
    __device__ __forceinline__ bool engine_block(int c) {
        if (c % 2 == 0) {
            id = ahead == -2 || (unsigned)ahead < (unsigned)p.cache.num_blocks ? ahead : -1;
            bad |= id == -1;
            look_ahead(c / 2 + 1);
        }
        return id >= 0;
    }

    __device__ __forceinline__ void look_up(int i) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int key = begin + i * kTileKeys + lane + 32 * x;
            at_k[x] = at_v[x] = -1;
            if (key >= end) continue;
            if (PAGED) {
                const int block = block_of(p.batch, p.cache, seq, key);
                const int64_t offset = key % p.cache.block_size;
                if (block < 0) bad = true;
                else at_k[x] = at_v[x] = block * p.cache.block_stride + (int64_t)kv_head * p.cache.head_stride + (E4M3 ? offset << 40 : offset * HD * 2);
            } else {
                at_k[x] = (int64_t)(first_row + key) * p.k.row_stride + kv_head * p.k.head_stride;
                at_v[x] = (int64_t)(first_row + key) * p.v.row_stride + kv_head * p.v.head_stride;
            }
        }
    }
    __device__ __forceinline__ int64_t of_row(int r, bool is_v) const {
        return r < 32 ? (is_v ? at_v[0] : at_k[0]) : r < 64 ? (is_v ? at_v[1] : at_k[1]) : r < 96 ? (is_v ? at_v[2] : at_k[2]) : (is_v ? at_v[3] : at_k[3]);
    }

    // Loads `count` tiles.  first_loaded() is called by every warp once its copies from before are done.
    template <typename F>
    __device__ __forceinline__ void run(int count, F first_loaded) {
        if (PAGED) look_ahead(0);
        if constexpr (E4M3) run_e4m3(count, first_loaded);
        else run_16(count, first_loaded);
        copy_wait<0>();
        if (!ok) drain();
    }

    // A wait has run out: the engine's copies still in flight get a bounded chance to land before their memory is given back.
    __device__ __forceinline__ void drain() {
        constexpr int kRing = E4M3 ? RAW_SLOTS : SLOTS;
        for (int c = max(issued - kRing, 0); c < issued; ++c) {
            int quiet = 0;
            const bool short_v = !E4M3 && c % 2 && keys_of(c) < kTileKeys;
            const uint32_t bar = short_v ? tail : (E4M3 ? raw_full : full) + c % kRing * 8;
            barrier_wait_warp(bar, short_v ? 0 : c / kRing & 1, &quiet);
        }
    }

    template <typename F>
    __device__ __forceinline__ void run_16(int count, F first_loaded) {
        const int kv_heads = p.heads / p.group;
        for (int c = 0; c < count + kLag; ++c) {
            if (c < count) {
                const int slot = c % SLOTS;
                const uint32_t to = shared_address(ring) + slot * kSlot;
                const int keys = keys_of(c);
                const bool short_v = c % 2 && keys < kTileKeys;
                const uint32_t bar = short_v && by_engine() ? tail : full + slot * 8;
                if (c >= SLOTS && !(ok = barrier_wait_warp(empty + slot * 8, (c / SLOTS - 1) & 1, flags))) break;
                if (by_engine()) {
                    issued = c + 1;
                    const void* map = c % 2 ? &maps.v : &maps.k;
                    const int key = begin + c / 2 * kTileKeys;
                    if (!PAGED) {
                        if (lane == 0) {
                            if (w > 0) {
                                barrier_arrive(bar);
                            } else {
                                barrier_expect(bar, kSlot);
                                for (int h = 0; h < HD / 64; ++h) box_copy(to + h * kTileKeys * 128, map, h * 64, kv_head, first_row + key, bar);
                            }
                        }
                    } else {
                        const bool there = engine_block(c);
                        const int copies = __popc(__ballot_sync(0xffffffffu, there));
                        if (lane == 0) barrier_expect(bar, copies * p.box * 128);
                        __syncwarp();
                        if (there)
                            box_copy(to + part_of * kTileKeys * 128 + box_of * p.box * 128, map, part_of * 64,
                                     ((id * p.layers + p.layer) * kv_heads + kv_head) * p.cache.block_size + (key + box_of * p.box) % p.cache.block_size, bar);
                    }
                    if (short_v) {                                            // the last tile: this barrier is used once
                        ok = barrier_wait_warp(tail, 0, flags);
                        for (int x = w * 32 + lane; x < (kTileKeys - keys) * kPieces; x += WARPS * 32)
                            *reinterpret_cast<uint4*>(ring + slot * kSlot + tile_offset(keys + x / kPieces, x % kPieces)) = make_uint4(0, 0, 0, 0);
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) barrier_arrive(full + slot * 8);
                    }
                } else {
                    look_up(c / 2);
                    const char* data = PAGED ? (c % 2 ? p.cache.v : p.cache.k) : (c % 2 ? p.v.data : p.k.data);
                    for (int g = w; g < kTileKeys / kRowsAtOnce; g += WARPS) {
                        const int r = g * kRowsAtOnce + lane / kPieces, j = lane % kPieces;
                        const int64_t at = __shfl_sync(0xffffffffu, of_row(g * kRowsAtOnce, c % 2), r & 31);
                        copy16(to + tile_offset(r, j), data + (at >= 0 ? at + j * 16 : 0), at >= 0);
                    }
                }
            }
            copy_commit();
            if (c >= kLag) {
                copy_wait<kLag>();
                fence_async_shared();
                __syncwarp();
                if (c == kLag) first_loaded();
                if (lane == 0 && !by_engine()) barrier_arrive(full + (c - kLag) % SLOTS * 8);
            }
        }
    }

    // Codes and scales of tile c into the ring of bytes.
    __device__ __forceinline__ void fetch(int c) {
        const int slot = c % RAW_SLOTS;
        const uint32_t to = shared_address(raw) + slot * kRawSlot, bar = raw_full + slot * 8;
        const char* data = c % 2 ? p.cache.v : p.cache.k;
        if (by_engine()) {
            if (c >= RAW_SLOTS && !(ok = barrier_wait_warp(raw_empty + slot * 8, (c / RAW_SLOTS - 1) & 1, flags))) return;
            issued = c + 1;
            const bool there = engine_block(c);
            const int offset = (begin + c / 2 * kTileKeys + box_of * p.box) % p.cache.block_size;
            const uint32_t bytes = part_of ? p.box * 4 : p.box * HD, sum = __reduce_add_sync(0xffffffffu, there ? bytes : 0);
            if (lane == 0) barrier_expect(bar, sum);
            __syncwarp();
            if (there) {
                const char* tile_at = data + id * p.cache.block_stride + (int64_t)kv_head * p.cache.head_stride;
                if (part_of) bulk_copy(to + kTileKeys * HD + box_of * p.box * 4, tile_at + (int64_t)p.cache.block_size * HD + offset * 4, bytes, bar);
                else bulk_copy(to + box_of * p.box * HD, tile_at + (int64_t)offset * HD, bytes, bar);
            }
            return;
        }
        look_up(c / 2);
        for (int g = w; g < kTileKeys / kRawRows; g += WARPS) {
            const int r = g * kRawRows + lane / kRowPieces, j = lane % kRowPieces;
            const int64_t packed = __shfl_sync(0xffffffffu, of_row(g * kRawRows, false), r & 31);
            const int64_t tile_at = packed & 0xffffffffffll;
            const int offset = (int)(packed >> 40);
            const bool there = packed >= 0;
            copy16(to + r * HD + j * 16, data + (there ? tile_at + offset * HD + j * 16 : 0), there);
            if (j == 0) copy4(to + kTileKeys * HD + r * 4, data + (there ? tile_at + (int64_t)p.cache.block_size * HD + offset * 4 : 0), there);
        }
    }

    template <typename F>
    __device__ __forceinline__ void run_e4m3(int count, F first_loaded) {
        constexpr int kAhead = RAW_SLOTS - 1;
        // a warp's share of a tile, read before any of it is written: the loads do not wait for the stores
        constexpr int kShare = (kTileKeys / kRawRows + WARPS - 1) / WARPS;
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
            if (c < count && ok) fetch(c);
            copy_commit();
        }
        for (int c = 0; c < count && ok; ++c) {
            if (c + kAhead < count) fetch(c + kAhead);
            copy_commit();
            copy_wait<kAhead>();
            __syncwarp();
            const int slot = c % SLOTS, raw_slot = c % RAW_SLOTS;
            if (!ok || (by_engine() && !(ok = barrier_wait_warp(raw_full + raw_slot * 8, c / RAW_SLOTS & 1, flags)))) break;
            const unsigned char* from = raw + raw_slot * kRawSlot;
            uint4 codes[kShare];
            float scale[kShare];
#pragma unroll
            for (int x = 0; x < kShare; ++x) {
                const int g = w + x * WARPS, r = min(g, kTileKeys / kRawRows - 1) * kRawRows + lane / kRowPieces, j = lane % kRowPieces;
                codes[x] = *reinterpret_cast<const uint4*>(from + r * HD + j * 16);
                scale[x] = *reinterpret_cast<const float*>(from + kTileKeys * HD + r * 4);
            }
            if (c >= SLOTS && !(ok = barrier_wait_warp(empty + slot * 8, (c / SLOTS - 1) & 1, flags))) break;
            unsigned char* to = ring + slot * kSlot;
            const int keys = keys_of(c);
#pragma unroll
            for (int x = 0; x < kShare; ++x) {
                const int g = w + x * WARPS, r = g * kRawRows + lane / kRowPieces, j = lane % kRowPieces;
                if (g >= kTileKeys / kRawRows) break;
                uint4 lo, hi;
                widen16<BF16>(codes[x], scale[x], lo, hi);
                if (c % 2 && r >= keys) lo = hi = make_uint4(0, 0, 0, 0);
                const bool second = j >= kRowPieces / 2;                  // half of the lanes store their second piece first: other banks
                *reinterpret_cast<uint4*>(to + tile_offset(r, 2 * j + second)) = second ? hi : lo;
                *reinterpret_cast<uint4*>(to + tile_offset(r, 2 * j + 1 - second)) = second ? lo : hi;
            }
            fence_async_shared();
            __syncwarp();
            if (c == 0) first_loaded();
            if (lane == 0) {
                barrier_arrive(raw_empty + raw_slot * 8);
                barrier_arrive(full + slot * 8);
            }
        }
    }
};

}  // namespace kvmig
