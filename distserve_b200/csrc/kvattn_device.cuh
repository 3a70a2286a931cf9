// What the attention kernels share: their parameters, and wrappers of the instructions they use.
#pragma once

#include <cuda.h>

#include "kvcache_device.cuh"

namespace kvmig {

struct AttnRows {
    char* data;
    int64_t row_stride, head_stride;   // bytes
};

// How the keys of a sequence are cut into parts, each a block's work: in units of kSplitKeys keys, no part shorter than
// `least` units nor than the whole call's work over `blocks`, and never more than `parts` of them.
constexpr int kSplitKeys = 128;
struct SplitRule {
    int32_t parts, least, blocks;
    int32_t cuts;      // > 0: a row tile's keys are cut into this many parts on average, whatever fits at once
};

struct AttnParams {
    AttnRows q, out, k, v;             // k, v: whole prompts only
    CacheView cache;
    BatchView batch;
    int32_t heads, group;              // query heads, query heads per KV head
    float scale_log2;                  // scale * log2(e): exponentials are taken to base 2
    // Sequences of up to few_rows rows per KV head belong to the kernel for few rows, the others to the tile kernel.
    int64_t few_rows;
    SplitRule few, tiles;              // how each cuts a sequence's keys into parts
    int32_t few_tile;                  // rows of a block of the former
    int32_t parts;                     // the parts' partial results, with room for this many:
    float* part_out;                   // [row][head][part][head_dim], sums before the division
    float2* part_stat;                 // [row][head][part]: running maximum (base 2) and sum
    int32_t* part_chosen;              // units of a part (part_units): few rows, tiles
    int32_t box;                       // keys that the copy engine moves at once; 0: it cannot follow this layout
    int32_t q_box;                     // the same for Q: 1 if a tile of 128 rows is one box of tokens x query heads
    int32_t layers, layer;
    bool few_followed, tiles_followed; // another grid of this call comes after
};

// Maps of K and V for the copy engine: rows of head_dim values, copied in boxes of 64 values by up to 128 rows.
struct AttnMaps {
    CUtensorMap k, v, q;
};

// What a sequence adds to the work of its kernel (TILES: the tile kernel, else the one for few rows).  One with too many rows has
// one tile and no keys, as in work_of: the host has sized the grid for no more.
struct Share {
    unsigned units, tiles;
};
template <bool TILES>
__device__ __forceinline__ Share share_of(const AttnParams& p, int tile, int seq) {
    const Sequence s = sequence_at(p.batch, seq);
    const int tokens = p.batch.seq_lens[seq];              // loaded beside its rows, not after a look at them (4 chunks: 0.5 us)
    const int64_t total = (int64_t)s.rows * p.group;
    const bool too_many = s.rows > p.batch.max_rows;
    Share w;
    w.units = (unsigned)(too_many ? 0 : min(max(tokens, 0), capacity(p.batch, p.cache)) + kSplitKeys - 1) / kSplitKeys;
    w.tiles = (unsigned)min(((too_many ? 1 : total) + tile - 1) / tile, (int64_t)1 << 20);
    return total == 0 || (total > p.few_rows) != TILES ? Share{0, 0} : w;
}

// Units of a part, before `parts` is looked at: from the whole batch's work, which every warp that asks adds up.  With t
// row tiles in all, cutting to work / (blocks - t) units leaves no more than `blocks` parts, whatever the lengths; cutting to
// work / (cuts t) units, no more than (cuts + 1) t.
template <bool TILES>
__device__ __forceinline__ int even_units(const AttnParams& p, SplitRule rule, int tile) {
    if (rule.parts == 1) return 0;
    const int lane = threadIdx.x & 31, kv_heads = p.heads / p.group;
    unsigned long long sum = 0;
    unsigned tiles = 0;
    for (int i = lane; i < p.batch.num_seqs; i += 32) {
        const Share w = share_of<TILES>(p, tile, i);
        sum += w.units * (unsigned long long)w.tiles;
        tiles += w.tiles;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
    }
    if (rule.cuts > 0) return (int)fminf(ceilf((float)sum / ((float)max(tiles, 1u) * rule.cuts)), 1e6f);
    const float blocks = fmaxf((float)rule.blocks - (float)tiles * kv_heads, 0.5f * rule.blocks);
    return (int)fminf((float)sum * kv_heads / blocks, 1e6f) + 1;
}

// Keys of a part, for a sequence of `keys` of them: as few parts as that allows, and those alike.
__device__ __forceinline__ int64_t part_keys(int keys, SplitRule rule, int units) {
    const int all = (keys + kSplitKeys - 1) / kSplitKeys, most = max(max((all + rule.parts - 1) / rule.parts, rule.least), units);
    if (all <= most) return (int64_t)most * kSplitKeys;
    const int parts = (all + most - 1) / most;
    return (int64_t)((all + parts - 1) / parts) * kSplitKeys;
}

constexpr int kUncut = 1 << 24;        // units of a part where no sequence is cut

// The same for the tile kernel, whose blocks have an SM each (rule.blocks is two for each): of up to 19 ways to cut, one to a
// lane, the one that should be over first.  Time is counted in units of kSplitKeys keys; a block's start is worth 3 of
// them, leaving a partial result and its joining 5 more, the join's launch 3.  Long pieces begin first, so what is expected is
// the largest of: all work spread evenly, the waves of the longest pieces, and as many waves as there are of the shortest.
// No more pieces than rule.blocks, or than there are tiles.
__device__ __forceinline__ int tile_units(const AttnParams& p, SplitRule rule, int tile) {
    if (rule.parts == 1) return 0;
    const int lane = threadIdx.x & 31, n = p.batch.num_seqs;
    if (n > 32) return even_units<true>(p, rule, tile);
    const Share mine = lane < n ? share_of<true>(p, tile, lane) : Share{0, 0};
    const unsigned units = mine.units;
    const float count = (float)mine.tiles * (p.heads / p.group);          // row tiles of all KV heads
    float work = units * count, tiles = count;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        work += __shfl_xor_sync(0xffffffffu, work, d);
        tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
    }
    const unsigned longest = __reduce_max_sync(0xffffffffu, units);
    if (longest <= 2 * rule.least) return kUncut;          // joining would cost more than it saves
    const unsigned shortest_part = max((units + rule.parts - 1) / rule.parts, (unsigned)rule.least);      // see part_keys
    // lanes 0..15: the longest sequence in lane + 1 pieces; 16..18: no more pieces than make one to three waves
    const float slots = rule.blocks / 2, room = slots * (lane - 15) - tiles;
    const unsigned unit = lane < 16 ? (longest + lane) / (lane + 1) : (unsigned)fminf(work / fmaxf(room, 1.f), 1e6f) + 1;
    float all = 0.f, pieces = 0.f, top = 0.f, tops = 0.f, low = 1e9f;
    bool cut = false;
    for (int i = 0; i < n; ++i) {
        const unsigned u = __shfl_sync(0xffffffffu, units, i), most = max(__shfl_sync(0xffffffffu, shortest_part, i), unit);
        const float c = __shfl_sync(0xffffffffu, count, i);
        if (c == 0.f) continue;
        const float parts = u <= most ? 1.f : floorf(__fdividef((float)(u + most) - 0.5f, (float)most)) + (u >> 20 ? 1.f : 0.f);     // exact to 2^20
        const float many = c * parts, piece = ceilf(__fdividef((float)u, parts)) + (parts > 1.f ? 8.f : 3.f);
        cut |= parts > 1.f;
        all += many * piece;
        pieces += many;
        if (piece >= top) tops = piece == top ? tops + many : many;
        top = fmaxf(top, piece);
        low = fminf(low, piece);
    }
    float time = fmaxf(all / slots, fmaxf(ceilf(tops / slots) * top, ceilf(pieces / slots) * low)) + (cut ? 3.f : 0.f);
    if (lane > 18 || (lane > 15 && room <= 0.f) || (lane > 0 && pieces > fmaxf(rule.blocks, tiles))) time = 3e38f;
    const unsigned best = __reduce_min_sync(0xffffffffu, (__float_as_uint(time) & ~31u) | lane);         // of equals the fewest pieces
    return __shfl_sync(0xffffffffu, cut, best & 31) ? (int)__shfl_sync(0xffffffffu, unit, best & 31) : kUncut;
}

// Asked by every block; the first leaves the answer for the join.
template <bool TILES>
__device__ __forceinline__ int part_units(const AttnParams& p, SplitRule rule, int tile) {
    const int units = TILES ? tile_units(p, rule, tile) : even_units<false>(p, rule, tile);
    if (p.parts > 1 && blockIdx.x == 0 && threadIdx.x == 0) p.part_chosen[TILES] = units;
    return units;
}

// Row tiles of a sequence (one for a sequence with too many rows, whose rows become NaN; none if it is not the
// kernel's that asks, see part_units), and the keys and the number of its parts.
struct TileWork {
    int tiles, parts;
    int64_t part;
    int keys;               // of its longest part
};
template <bool PAGED, bool TILES>
__device__ __forceinline__ TileWork work_of(const AttnParams& p, SplitRule rule, int tile, int seq, int units) {
    TileWork w = {0, 1, INT64_MAX, 0};
    const Sequence s = sequence_at(p.batch, seq);
    const int64_t total = (int64_t)s.rows * p.group;
    if (total == 0 || (total > p.few_rows) != TILES) return w;
    if (s.rows > p.batch.max_rows) {
        w.tiles = 1;
        return w;
    }
    w.tiles = (int)((total + tile - 1) / tile);
    if (PAGED) {
        const int len = min(max(p.batch.seq_lens[seq], 0), capacity(p.batch, p.cache));
        w.part = part_keys(len, rule, units);
        w.parts = max((int)((len + w.part - 1) / w.part), 1);
        w.keys = (int)min(w.part, (int64_t)len);
    }
    return w;
}

// The c-th piece of the call's work for a KV head: a row tile and a part of a sequence's keys.  Long pieces come first:
// over the cache, sequences with long parts before others; of whole prompts, the last tiles of all of them, which under
// the causal mask have the most keys, before the first.  (More than 32 sequences, a lane each, are taken in their order.)
// Nothing is launched for pieces that do not exist, because a block needs its shared memory, an SM to itself in the tile
// kernel, even to return.
template <bool PAGED, bool TILES>
__device__ __forceinline__ bool find_work(const AttnParams& p, SplitRule rule, int units, int rows, int c, int& seq, int& tile, int& split, int64_t& part) {
    const int lane = threadIdx.x & 31, n = p.batch.num_seqs;
    auto sum = [](int x) { return __reduce_add_sync(0xffffffffu, x); };
    for (int first = 0; first < n; first += 32) {
        const TileWork w = first + lane < n ? work_of<PAGED, TILES>(p, rule, rows, first + lane, units) : TileWork{0, 1, 0, 0};
        const int all = sum(w.tiles * w.parts);
        if (c >= all) {
            c -= all;
            continue;
        }
        int level = -1, before = 0, mine = w.tiles * w.parts;       // pieces of this lane, and of those that come before it
        if (PAGED && n <= 32) {
            const int keys = w.keys;
            for (int i = 0; i < n; ++i) {
                const int other = __shfl_sync(0xffffffffu, keys, i), pieces = __shfl_sync(0xffffffffu, mine, i);
                if (other > keys || (other == keys && i < lane)) before += pieces;
            }
        } else {
            if (n > 1 && n <= 32) {
                // the largest tile number such that more than c pieces have it or a larger one
                int high = __reduce_max_sync(0xffffffffu, w.tiles);
                level = 0;
                while (level < high) {
                    const int mid = (level + high + 1) / 2;
                    if (sum(max(w.tiles - mid, 0) * w.parts) > c) level = mid;
                    else high = mid - 1;
                }
                c -= sum(max(w.tiles - level - 1, 0) * w.parts);
                mine = w.tiles > level ? w.parts : 0;
            }
            before = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, before, d);
                if (lane >= d) before += x;
            }
            before -= mine;
        }
        const int owner = __ffs(__ballot_sync(0xffffffffu, c >= before && c < before + mine)) - 1;
        const int rest = c - __shfl_sync(0xffffffffu, before, owner), parts = __shfl_sync(0xffffffffu, w.parts, owner);
        seq = first + owner;
        part = __shfl_sync(0xffffffffu, w.part, owner);
        split = rest % parts;
        tile = __shfl_sync(0xffffffffu, w.tiles, owner) - 1 - rest / parts;
        if (level >= 0) tile = level;
        return true;
    }
    return false;
}

// Lets the next grid of the stream begin.  Only between the grids of one call, which are made for it: another kernel of
// this library that is allowed to begin early (a migration) must not pass one that reads or writes the pools.
__device__ __forceinline__ void let_next_begin(bool followed) {
    if (followed) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes (or 4) from global to shared memory without a register in between; zeros where `valid` is false, and then
// nothing is read.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
    return x;
}
// Four 8x8 matrices of 16-bit values, transposed on the way into registers.
__device__ __forceinline__ uint4 load_matrices_transposed(uint32_t row) {
    uint4 x;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(row) : "memory");
    return x;
}

// d += a b for a 16 x 16 tile a, a 16 x 8 tile b and 32-bit sums.
template <bool BF16>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The larger of three, NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float x;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(x) : "f"(a), "f"(b), "f"(c));
    return x;
}

__device__ __forceinline__ float not_a_number() { return __uint_as_float(0x7fffffffu); }

}  // namespace kvmig
