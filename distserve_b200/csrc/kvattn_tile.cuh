// Attention of many rows, over the paged cache or over packed prompts, on the 5th-generation tensor cores.
//
// A block takes 256 rows (token x query head of a group) of one sequence and KV head as two tiles of 128, and walks over
// the keys 128 at a time:
//   S = Q K^T   128 x 128 x head_dim, both operands in shared memory, sums in tensor memory;
//   P = 2^(scale S - m), rounded to 16 bits, written back over S's columns;
//   O += P V    128 x head_dim x 128, P from tensor memory, sums in tensor memory.
// Each tile has a warpgroup with a thread per row for the softmax, so no value crosses threads.  While one tile's
// softmax runs the tensor core works on the other's products.  One warp issues all of them, which keeps the tiles in
// opposite phases (a warp for each tile lets them fall into step: 150 us instead of 130 for 4096 tokens, 32/4 heads of
// 128).  The remaining warps fill a ring of K and V tiles in shared memory (kvattn_load.cuh).
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time; until then P may be as large
// as 256, which costs no precision.  Tensor memory: S0 S1 O0 O1, 128 columns each.
//
// Measured: one prompt of 4096 tokens, 32/4 heads of 128: 137 us in bf16, 1.0 PFLOP/s, 0.6 of the library's best rate; 155 us in
// fp16, 0.89 PFLOP/s.
// A step of 256 rows by 128 keys takes 3100 cycles where its products need 2048: each tile waits for its own chain of
// scores (512 cycles and a wake-up), softmax (2000, of which the special function unit needs 1024) and products.  Tried
// and slower: a quarter or half of the exponentials as polynomials (2%, 8%), two softmax threads per row (50%), a warp for
// each tile's products (15%).
#pragma once

#include "kvattn_load.cuh"

namespace kvmig {

constexpr int kTileRows = 128, kBlockRows = 2 * kTileRows;
constexpr int kSoftmaxThreads = 256;
constexpr float kLazy = 8.f;                 // the maximum may lag behind by this many powers of two

template <int HD, bool E4M3> struct TileShape {
    static constexpr int kSlot = kTileKeys * HD * 2;                        // a 16-bit tile of K, V or Q
    static constexpr int kSlots = E4M3 ? 3 : 5;
    static constexpr int kLoadWarps = E4M3 ? 7 : 3, kThreads = kSoftmaxThreads + kLoadWarps * 32 + 32;
    // Registers of a softmax thread and of the others: together what the block is launched with (168 or 128 a thread).
    // Over quantised pools 196 bytes a thread are spilled and 216 reloaded (76 and 88 at a head_dim of 64).
    static constexpr int kSoftmaxRegisters = E4M3 ? 200 : 208, kOtherRegisters = E4M3 ? 56 : 88;
    static constexpr int kRawSlot = E4M3 ? kTileKeys * (HD + 4) : 0;        // codes, then scales
    static constexpr int kRawSlots = E4M3 ? 3 : 0;
    static constexpr int kBarriers = 2 * kSlots + 1 + 8 + 2 + 2 * kRawSlots;
    static constexpr int kRing = 2 * kSlot, kRaw = kRing + kSlots * kSlot, kBars = kRaw + kRawSlots * kRawSlot;
    static constexpr int kShared = kBars + kBarriers * 8 + 64 + 1024;       // and room to align the start to 1024
};

__device__ unsigned int g_attention_timeouts;      // blocks that gave up waiting

// The grid may start while the grid before it, which it does not depend on, still runs, but must not end before it:
// what follows in the stream waits for this one only.
__device__ __forceinline__ void finish_after_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int HD, bool BF16, bool PAGED, bool E4M3>
__global__ void __launch_bounds__((TileShape<HD, E4M3>::kThreads), 1) attend_tiles(const __grid_constant__ AttnParams p, const __grid_constant__ AttnMaps maps) {
    using T = TileShape<HD, E4M3>;
    using H = Half<BF16>;
    constexpr int kPieces = HD / 8;                    // 16-byte pieces of a 16-bit row
    constexpr int kLoadWarps = T::kLoadWarps, kTileThreads = T::kThreads;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + (1024 - (shared_address(smem_raw) & 1023)) % 1024;
    const uint32_t base = shared_address(smem);
    const uint32_t bars = base + T::kBars;
    auto full = [&](int s) { return bars + s * 8; };
    auto empty = [&](int s) { return bars + (T::kSlots + s) * 8; };
    const uint32_t q_full = bars + 2 * T::kSlots * 8, s_full = q_full + 8, p_half = s_full + 16, p_full = p_half + 16, pv_done = p_full + 16,
                   drained = pv_done + 16, tail = drained + 8, raw_full = tail + 8, raw_empty = raw_full + T::kRawSlots * 8;
    volatile int* flags = reinterpret_cast<volatile int*>(smem + T::kBars + T::kBarriers * 8);    // failed, bad, tensor memory

    let_next_begin(p.tiles_followed);                  // the join waits for the end of this grid
    // Which rows and keys: one warp finds out while others set up.
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_heads = p.heads / p.group, kv_head = blockIdx.x % kv_heads;
    volatile int* const work = flags + 3;              // sequence (-1: nothing to do), first row in it, keys [begin, end) and whether they are all
    if (warp == 0) {
        int seq = -1, tile = 0, split = 0;
        int64_t part = 1;
        const bool any = find_work<PAGED, true>(p, p.tiles, PAGED ? part_units<true>(p, p.tiles, kBlockRows) : 0, kBlockRows, blockIdx.x / kv_heads, seq, tile, split, part);
        if (lane == 0) {
            const Sequence s = sequence_at(p.batch, any ? seq : 0);
            const int tokens = PAGED ? max(p.batch.seq_lens[any ? seq : 0], 0) : s.rows, len = PAGED ? min(tokens, capacity(p.batch, p.cache)) : tokens;
            work[0] = any ? seq : -1;
            work[1] = tile;
            work[2] = (int)(part * split);
            work[3] = (int)min(part * (split + 1), (int64_t)len);
            work[4] = part >= len;
            work[5] = split;
            work[6] = s.first;
            work[7] = s.rows;
            work[8] = tokens;
            flags[0] = 0;
            flags[1] = tokens > len;                   // the table is too short for the sequence
        }
    } else if (threadIdx.x == 32) {
        for (int i = 0; i < T::kSlots; ++i) {
            barrier_init(full(i), kLoadWarps);
            barrier_init(empty(i), 1);
        }
        barrier_init(q_full, kLoadWarps);
        barrier_init(drained, 1);
        barrier_init(tail, kLoadWarps);
        for (int i = 0; i < T::kRawSlots; ++i) {
            barrier_init(raw_full + i * 8, kLoadWarps);
            barrier_init(raw_empty + i * 8, kLoadWarps);
        }
        for (int t = 0; t < 2; ++t) {
            barrier_init(s_full + t * 8, 1);
            barrier_init(p_half + t * 8, 4);
            barrier_init(p_full + t * 8, 4);
            barrier_init(pv_done + t * 8, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_shared();
    }
    if (warp == kTileThreads / 32 - 1) tmem_alloc(shared_address(const_cast<int*>(flags + 2)), 512);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    struct { int begin, end; } range = {work[2], work[3]};
    struct { int first, rows; } s = {work[6], work[7]};
    const int seq = work[0], split = work[5], first_pos = work[8] - s.rows;
    const bool whole = work[4];
    const int64_t total = (int64_t)s.rows * p.group, row0 = (int64_t)work[1] * kBlockRows;
    if (seq < 0 || s.rows > p.batch.max_rows) {
        if (seq >= 0)
            for (int64_t x = threadIdx.x; x < total * (HD / 8); x += kTileThreads) {
                const int64_t r = x / (HD / 8);
                *reinterpret_cast<uint4*>(p.out.data + (s.first + r / p.group) * p.out.row_stride +
                                          (kv_head * p.group + r % p.group) * p.out.head_stride + x % (HD / 8) * 16) =
                    make_uint4(H::kNan2, H::kNan2, H::kNan2, H::kNan2);
            }
        if (warp == kTileThreads / 32 - 1) tmem_free(__shfl_sync(0xffffffffu, flags[2], 0), 512);
        finish_after_predecessor();
        return;
    }
    // Row r of the block is token token0 + (skip + r) / group, query head (skip + r) % group of the group.
    const int token0 = (int)(row0 / p.group), here = (int)min((int64_t)kBlockRows, total - row0);
    const unsigned group = p.group, skip = (unsigned)(row0 - (int64_t)token0 * group);
    int n[2];                                          // key tiles of each row tile
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int end = min((t + 1) * kTileRows, here);
        const int keys = end <= t * kTileRows ? 0 : (int)min((int64_t)range.end, (int64_t)first_pos + token0 + (skip + end - 1) / group + 1) - range.begin;
        n[t] = keys > 0 ? (keys + kTileKeys - 1) / kTileKeys : 0;
    }
    const int steps = max(n[0], n[1]);
    const uint32_t tmem = __shfl_sync(0xffffffffu, flags[2], 0);
    // A whole warp waits, and goes on or gives up together.
    auto warp_wait = [&](uint32_t bar, uint32_t parity) { return barrier_wait_warp(bar, parity, flags); };
    // The sign of the scale is taken by the products and a scale of zero by Q, so that the maximum of the scores is theirs too.
    const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);

    if (warp < kSoftmaxThreads / 32) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kSoftmaxRegisters));
        // ---- softmax: a thread per row -------------------------------------------------------------------
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;             // this warp's 32 rows of tensor memory
        const uint32_t s_at = tmem + t * kTileKeys + lanes, o_at = tmem + 2 * kTileKeys + t * 128 + lanes;
        const bool there = (int)threadIdx.x < here;
        const int token = token0 + (skip + threadIdx.x) / group;
        const int last = there ? (int)min((int64_t)first_pos + token, (int64_t)range.end - 1) : -1;      // last key that the row sees
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = 0; i < n[t]; ++i) {
            if (!(ok = warp_wait(s_full + t * 8, i & 1))) break;
            tmem_fence_after();
            const int seen = last - (range.begin + i * kTileKeys);      // columns up to this one count
            const bool masked = __any_sync(0xffffffffu, seen < kTileKeys - 1);
            uint32_t a[64], b[64];
            tmem_load_async(a, s_at);
            tmem_load_async(b, s_at + 64);
            tmem_wait(a);
            tmem_wait(b);
            if (masked) {
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    a[j] = j <= seen ? a[j] : 0xff800000u;
                    b[j] = j + 64 <= seen ? b[j] : 0xff800000u;
                }
            }
            const uint64_t scale2 = pair(scale, scale);
            uint64_t sum[2] = {0, 0};
            // Probabilities of 64 keys into 32 registers, two to a register.
            // The maximum; NaN if a score is, and then everything of this row becomes NaN.
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            auto probabilities = [&](const uint32_t (&x)[64], uint32_t (&w)[32], uint64_t shift2, bool find_top) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (find_top) {
                        tops[j % 2] = max_nan(tops[j % 2], __uint_as_float(a[2 * j]), __uint_as_float(a[2 * j + 1]));
                        tops[j % 2 + 2] = max_nan(tops[j % 2 + 2], __uint_as_float(b[2 * j]), __uint_as_float(b[2 * j + 1]));
                    }
                    const uint64_t e = fma_pair(pair(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), scale2, shift2);
                    float2 y = unpair(e);
                    y.x = exp2_fast(y.x);
                    y.y = exp2_fast(y.y);
                    sum[j % 2] = add_pair(sum[j % 2], pair(y.x, y.y));
                    w[j] = H::from_float2(y.x, y.y);
                }
            };
            auto hand_over = [&](uint32_t at, const uint32_t (&w)[32], uint32_t bar) {
                tmem_store(at, w);
                tmem_wait_store();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(bar);
            };
            uint32_t w[32];
            // Every step but the first begins with the maximum so far, as if this tile did not raise it beyond the allowance.
            uint64_t shift2 = pair(m == -INFINITY ? 0.f : -m, m == -INFINITY ? 0.f : -m);
            if (i > 0) {
                probabilities(a, w, shift2, true);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    tops[j % 2] = max_nan(tops[j % 2], __uint_as_float(a[2 * j]), __uint_as_float(a[2 * j + 1]));
                    tops[j % 2 + 2] = max_nan(tops[j % 2 + 2], __uint_as_float(b[2 * j]), __uint_as_float(b[2 * j + 1]));
                }
            }
            const float top = max_nan(max_nan(tops[0], tops[1], tops[2]), tops[3], -INFINITY) * scale;
            const bool grown = i == 0 || !(top <= m + kLazy);
            if (__any_sync(0xffffffffu, grown)) {
                if (i > 0) {
                    if (!(ok = warp_wait(pv_done + t * 8, (i - 1) & 1))) break;
                    tmem_fence_after();
                    const float keep = grown ? exp2_fast(m - top) : 1.f;
                    l *= keep;
#pragma unroll
                    for (int j = 0; j < HD; j += 32) {
                        uint32_t o[32];
                        tmem_load(o, o_at + j);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                        tmem_store(o_at + j, o);
                    }
                }
                if (grown) m = top;
                shift2 = pair(m == -INFINITY ? 0.f : -m, m == -INFINITY ? 0.f : -m);
                sum[0] = sum[1] = 0;
                probabilities(a, w, shift2, false);
            }
            hand_over(s_at + 64, w, p_half + t * 8);
            probabilities(b, w, shift2, false);
            hand_over(s_at + 96, w, p_full + t * 8);
            const float2 parts = unpair(add_pair(sum[0], sum[1]));
            l += parts.x + parts.y;
        }
        __syncwarp();
        asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads + kLoadWarps * 32) : "memory");                  // the loading warps have said what they found
        if (ok && n[t] > 0) ok = warp_wait(pv_done + t * 8, (n[t] - 1) & 1);
        tmem_fence_after();
        if (m == -INFINITY) l = 0.f;                                     // no key: zeros
        if (!ok || flags[0] || flags[1]) l = not_a_number();
        const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
        const int64_t out_row = s.first + token, head = kv_head * group + (skip + threadIdx.x) % group;
        const int64_t place = (out_row * p.heads + head) * p.parts + split;
        char* to = p.out.data + out_row * p.out.row_stride + head * p.out.head_stride;
        if (there && !whole) p.part_stat[place] = make_float2(m, l);
#pragma unroll
        for (int j = 0; j < HD; j += 32) {
            uint32_t o[32];
            __syncwarp();
            if (n[t] > 0) {
                tmem_load(o, o_at + j);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            if (!there) continue;
            if (whole) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t h[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) h[x] = H::from_float2(__uint_as_float(o[e + 2 * x]) * inv, __uint_as_float(o[e + 2 * x + 1]) * inv);
                    *reinterpret_cast<uint4*>(to + (j + e) * 2) = make_uint4(h[0], h[1], h[2], h[3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<uint4*>(p.part_out + place * HD + j + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
        }
        tmem_fence_before();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegisters));
      if (warp < kSoftmaxThreads / 32 + kLoadWarps) {
        // ---- loading -------------------------------------------------------------------------------------
        if (!E4M3 && p.box > 0 && lane == 0) {
            prefetch_map(&maps.k);
            prefetch_map(&maps.v);
        }
        const int w = warp - kSoftmaxThreads / 32;
        constexpr int kRowsAtOnce = 32 / kPieces;                       // rows that a warp copies with one instruction
        const bool q_by_engine = p.q_box > 0 && p.scale_log2 != 0.f;
        if (q_by_engine) {
            // 128 rows are 128 / group tokens of all the group's heads, and row0 is the first head of one.
            if (w == 0 && lane == 0 && steps > 0) {
                barrier_expect(q_full, 2 * T::kSlot);
                for (int t = 0; t < 2; ++t)
                    for (int h = 0; h < HD / 64; ++h)
                        box_copy(base + t * T::kSlot + h * kTileRows * 128, &maps.q, h * 64, kv_head * (int)group, s.first + token0 + t * (kTileRows / (int)group), q_full);
            }
        } else {
            for (int x = 0; x < kBlockRows; x += 32) {                  // each lane finds the place of one row of 32
                const int mine = x + lane;
                const bool there = mine < here && p.scale_log2 != 0.f;
                const unsigned token = (skip + mine) / group, head = (skip + mine) % group;
                const int64_t at = there ? (int64_t)(s.first + token0 + token) * p.q.row_stride + (int64_t)(kv_head * group + head) * p.q.head_stride : -1;
                for (int g = w; g < 32 / kRowsAtOnce; g += kLoadWarps) {
                    const int r = g * kRowsAtOnce + lane / kPieces, j = lane % kPieces;
                    const int64_t from = __shfl_sync(0xffffffffu, at, r);
                    copy16(base + (x / kTileRows) * T::kSlot + tile_offset(x % kTileRows + r, j), p.q.data + (from >= 0 ? from + j * 16 : 0), from >= 0);
                }
            }
        }
        copy_commit();
        TileLoader<HD, BF16, PAGED, E4M3, kLoadWarps, T::kSlots, T::kRawSlots> loader(p, maps, w, seq, kv_head, s.first, range.begin, range.end,
                                                                                   smem + T::kRing, smem + T::kRaw, full(0), empty(0), raw_full,
                                                                                   raw_empty, tail, flags);
        loader.run(2 * steps, [&] {
            if (lane == 0 && !(q_by_engine && w == 0)) barrier_arrive(q_full);
        });
        if (!loader.ok && q_by_engine && w == 0) {                      // Q's copies too
            int quiet = 0;
            barrier_wait_warp(q_full, 0, &quiet);
        }
        if (loader.bad) flags[1] = 1;
        __threadfence_block();
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"n"(kSoftmaxThreads + kLoadWarps * 32) : "memory");
    } else {
        // ---- products: one lane issues them all -----------------------------------------------------------
        if (steps > 0) {
            const uint32_t s_kind = product_kind(BF16, kTileRows, kTileKeys, false, p.scale_log2 < 0.f);
            constexpr uint32_t o_kind = product_kind(BF16, kTileRows, HD, true, false);
            const bool leader = elect_one();
            const uint64_t q_desc = operand(base, 16, 1024), k_desc = operand(base + T::kRing, 16, 1024),
                           v_desc = operand(base + T::kRing, kTileKeys * 128, 1024);
            bool ok = warp_wait(q_full, 0);
            auto scores = [&](int t, int slot) {
                const uint64_t a = q_desc + t * (T::kSlot >> 4), b = k_desc + slot * (T::kSlot >> 4);
                if (leader) {
#pragma unroll
                    for (int x = 0; x < HD / 16; ++x) {
                        const uint32_t step = ((x / 4) * (kTileKeys * 128) + (x % 4) * 32) >> 4;
                        mma_shared(tmem + t * kTileKeys, a + step, b + step, s_kind, x > 0);
                    }
                    mma_commit(s_full + t * 8);
                }
                __syncwarp();
            };
            auto outputs = [&](int t, int slot, int half, bool add) {   // 64 keys
                const uint64_t b = v_desc + slot * (T::kSlot >> 4);
                if (leader) {
#pragma unroll
                    for (int y = 0; y < kTileKeys / 32; ++y) {
                        const int x = half * (kTileKeys / 32) + y;
                        mma_tmem(tmem + 2 * kTileKeys + t * 128, tmem + t * kTileKeys + 64 + x * 8, b + x * (2048 >> 4), o_kind, add || y > 0);
                    }
                    if (half) mma_commit(pv_done + t * 8);
                }
                __syncwarp();
            };
            auto release = [&](int slot) {
                if (leader) mma_commit(empty(slot));
                __syncwarp();
            };
            if (ok) ok = warp_wait(full(0), 0);
            if (ok) {
                tmem_fence_after();
                if (n[0] > 0) scores(0, 0);
                if (n[1] > 0) scores(1, 0);
                release(0);
            }
            int slot = 0, phase = 0;                                    // of the tile that was last waited for
            for (int i = 0; i < steps && ok; ++i) {
                auto next = [&](int& at, int& ph) { if (++at == T::kSlots) { at = 0; ph ^= 1; } };
                next(slot, phase);
                const int v_slot = slot;
                if (!(ok = warp_wait(full(v_slot), phase))) break;
                const bool more = i + 1 < steps;
                if (more) next(slot, phase);
                bool k_ready = false;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (i >= n[t] || !ok) continue;
                    if (!(ok = warp_wait(p_half + t * 8, i & 1))) continue;
                    tmem_fence_after();
                    outputs(t, v_slot, 0, i > 0);
                    if (i + 1 < n[t] && !k_ready) {
                        if (!(ok = warp_wait(full(slot), phase))) continue;
                        k_ready = true;
                    }
                    if (!(ok = warp_wait(p_full + t * 8, i & 1))) continue;
                    tmem_fence_after();
                    outputs(t, v_slot, 1, true);
                    if (i + 1 < n[t]) scores(t, slot);
                }
                if (!ok) break;
                release(v_slot);
                if (more) release(slot);
            }
            if (!ok) {
                // products still in flight read shared memory and write tensor memory: give them their chance to end
                if (leader) {
                    atomicAdd(&g_attention_timeouts, 1u);
                    mma_commit(drained);
                }
                int quiet = 0;
                barrier_wait(drained, 0, &quiet);
            }
        }
        __syncwarp();
      }
    }
    __syncthreads();
    if (warp == kTileThreads / 32 - 1) {
        tmem_fence_after();
        tmem_free(tmem, 512);
    }
    finish_after_predecessor();
}

}  // namespace kvmig
