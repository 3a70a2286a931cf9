// Attention of few rows over the paged cache: a decoding step's single tokens and short drafts.
//
// A block takes rows of one sequence that share a KV head, up to 16 or 32 of them (tokens x query heads of the group), and
// one part of that sequence's keys.  Every K and V value is used for a few rows only, so the kernel is bound by reading
// the cache; all else is arranged around keeping reads in flight:
//   * blocks have 4 warps, two blocks to an SM, so that one's start hides behind the other's stream; 8 where whole
//     sequences leave SMs without a block;
//   * each warp has its own ring of stages of 16 keys in shared memory, filled by cp.async and drained by that warp
//     alone: no barrier of the block until the end, and about 96 KiB in flight per SM (two blocks);
//   * warps take the groups of 16 keys in turn and keep their own running maximum, sum and output, joined at the end;
//   * products run on m16n8k16 matrix instructions with the rows padded to 16 or 32.  Contraction order is free, so K
//     fragments are read as 16 consecutive bytes per lane and Q's values are permuted to match, once;
//   * e4m3 codes widen to 16 bits in registers; K's scales multiply the scores.  V's scale s_j goes into the exponent,
//     P_j = 2^(score_j + log2 s_j - m + 15), so that no P_j leaves fp16 at the upper end, and the sum counts P_j / s_j.  At the
//     lower end fp16 holds P_j to eleven bits down to 2^-29 of its largest value and to 2^-40 of it below.  A row's scale is the
//     size of its values, so that is what a value weighs in the output, but for a row of zeros, whose scale is 1 whatever
//     its neighbours' are: one that would raise m counts with kZeroRowScale instead, or it would push the others out of the range.
// Measured: 64 requests with 40 heads of 128, 41k cached tokens, 838 MB: 137 us (6.1 TB/s, 95% of a copy); 32 requests of
// 2000 tokens, 16 heads: 85 us from 16 bits (6.1 TB/s), 76 us from e4m3 (3.6 TB/s).  From e4m3 it is latency that bounds it: DRAM
// is 43% busy and 0.43 of the issue slots are used, by two warps to a scheduler that each go through a chain of copies, widening,
// products, maximum, exponentials and products for 16 keys (4.1 cycles from one instruction of a warp to its next, 1.3 of them
// for the result of the one before, 0.8 for copies).  A third block per SM with a smaller ring gained nothing.
// Rows of zeros cost short sequences something, since their maxima still grow: 16 requests of 300 tokens, 12 heads of 64, 9.4 us
// without the look for them and the shift by 2^15, 10.2 with; 64 of 640, 40 heads, 127 and 129; 32 of 2000 as before.  A vote per
// group of 16 keys ahead of the scores took 2-4% of all of them, the same code as a function or a second turn 2-5% of 32 rows.
#pragma once

#include "kvattn_device.cuh"

namespace kvmig {

constexpr int kFewKeys = 16;
// Rows of a sequence and KV head up to which this kernel is used.  Beyond 32 it reads the cache twice, which the tile kernel
// beats on 16-bit pools (8 sequences of 4000 tokens, 16 KV heads: 32 rows 73 us here and 76 there, 48 rows 109 and 77) but not
// where it has to widen codes for tiles of 256 rows (64 rows 116 and 147, 96 rows 204 and 146).
constexpr int few_most(bool e4m3) { return e4m3 ? 64 : 32; }

// Quantised pools: P_j's largest value is 2^15 (kTopLog2).  The sum counts P_j 2^-6 / s_j (kSumUnit), since 1 / s_j alone reaches
// 2^100 and 2^-120: neither that nor the sum of 2^18 keys leaves the range of 32 bits.
constexpr float kTopLog2 = 15.f, kTop = 0x1p15f, kSumUnit = 0x1p-6f;
// The scale that a V row of zeros counts with where it would raise the maximum: 2^-64.  Below those of the other rows it leaves
// P_j its range; and weights down to 2^-24 are in the sum while scales differ by less than 2^117.  So zeros go with any V of
// fp16 rows (scales 2^-32 .. 2^8), and with bf16 rows of 2^-70 .. 2^60.
constexpr float kZeroRowLog2 = -64.f, kZeroRowScale = 0x1p-64f;

template <int HD, bool E4M3, int MT, int WARPS> struct FewShape {
    static constexpr int kRows = 16 * MT;
    static constexpr int kRowBytes = HD * (E4M3 ? 1 : 2);
    static constexpr int kTile = kFewKeys * kRowBytes;                          // K or V of one stage
    static constexpr int kStage = 2 * kTile + (E4M3 ? 2 * kFewKeys * 4 : 0);    // and the scales behind them
    static constexpr int kStages = 24576 / kStage < 8 ? 24576 / kStage : 8;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kJoin = kRows * (HD + 2) * 4;                       // a warp's result, in its own ring
    static constexpr int kShared = WARPS * (kRing > kJoin ? kRing : kJoin);
};

template <int HD, bool BF16, bool E4M3, int MT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 8 / WARPS) attend_few(const __grid_constant__ AttnParams p) {
    using S = FewShape<HD, E4M3, MT, WARPS>;
    using H = Half<BF16>;
    constexpr int kSteps = HD / 16;                       // contraction steps of q . k
    constexpr int kChunks = S::kRowBytes / 16;            // 16-byte pieces of a cached row
    constexpr int kFlip = kChunks >= 8 ? 4 : 0;           // odd keys swap their 64-byte halves: no bank conflicts
    auto turn = [](int r) { return kChunks >= 8 ? r & 7 : (r >> 1) & 3; };   // V's pieces are turned by the key for ldmatrix
    constexpr bool kBf16 = BF16 && !E4M3;                 // e4m3 codes widen to fp16 with one instruction, whatever Q's type
    using In = Half<kBf16>;
    extern __shared__ __align__(128) unsigned char smem[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, c = lane & 3;
    let_next_begin(p.few_followed);                        // the tile kernel's rows are others, the join waits
    const int kv_heads = p.heads / p.group, kv_head = blockIdx.x % kv_heads;
    int seq, tile, split = 0;
    int64_t part = INT64_MAX;                              // keys of a part
    if (p.few.parts > 1) {
        if (!find_work<true, false>(p, p.few, part_units<false>(p, p.few, S::kRows), S::kRows, blockIdx.x / kv_heads, seq, tile, split, part)) return;
    } else {                                               // whole sequences: nothing to look for
        const int tiles = gridDim.x / (kv_heads * p.batch.num_seqs);
        seq = blockIdx.x / kv_heads % p.batch.num_seqs;
        tile = tiles - 1 - blockIdx.x / kv_heads / p.batch.num_seqs;
    }
    const Sequence s = sequence_at(p.batch, seq);
    const int tokens = max(p.batch.seq_lens[seq], 0);
    const int64_t total = (int64_t)s.rows * p.group;
    const bool too_many = s.rows > p.batch.max_rows;
    if (total <= (int64_t)tile * S::kRows || total > p.few_rows || (too_many && tile > 0)) return;
    const int row0 = tile * S::kRows;                      // row r of the block: token (row0 + r) / group, query head % group
    const int rows = too_many ? 0 : (int)min(total - row0, (int64_t)S::kRows);
    const int first_pos = tokens - s.rows;                 // position of the first token; may be negative
    const int len = min(tokens, capacity(p.batch, p.cache));
    const bool whole = part >= len;                                            // one part has everything
    struct { int begin, end; } range = {(int)(part * split), 0};
    if (!too_many) range.end = whole ? len : (int)min(part * (split + 1), (int64_t)len);

    // Q: lane (quad, c) has rows quad and quad + 8 of each 16.  16-bit pools: step t, values 32 (t/2) + 8 c + 4 (t%2) + 0..3;
    // quantised pools: 64 (t/4) + 16 c + 4 (t%4) + 0..3.
    uint32_t q[MT][kSteps][4];
    int last[MT][2];                                       // the last key that each of the lane's rows sees
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = x * 16 + quad + half * 8;
            const bool there = r < rows;
            const unsigned token = there ? (unsigned)(row0 + r) / (unsigned)p.group : 0, head = there ? (unsigned)(row0 + r) % (unsigned)p.group : 0;
            last[x][half] = first_pos + (int)token;
            const char* at = p.q.data + (int64_t)(s.first + (int)token) * p.q.row_stride + (int64_t)(kv_head * p.group + (int)head) * p.q.head_stride;
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
                const int d = E4M3 ? 64 * (t / 4) + 16 * c + 4 * (t % 4) : 32 * (t / 2) + 8 * c + 4 * (t % 2);
                uint2 w = make_uint2(0, 0);
                if (there) w = __ldg(reinterpret_cast<const uint2*>(at + d * 2));
                q[x][t][half] = w.x;
                q[x][t][half + 2] = w.y;
            }
        }
    // bf16 rows over a quantised pool go through fp16 times a power of two that brings the row's largest value to
    // 2^14 .. 2^15: eight bits of fraction fit, and what is lost below 2^-24 is 2^-40 of that value.
    float row_factor[MT][2];
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            row_factor[x][half] = p.scale_log2;
            if (BF16 && E4M3) {
                uint32_t top = 0;
#pragma unroll
                for (int t = 0; t < kSteps; ++t) top = __vmaxu2(top, __vmaxu2(q[x][t][half] & 0x7fff7fffu, q[x][t][half + 2] & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = min(max((int)(top >> 7) - 127 - 14, -100), 112);     // of the largest value, minus 14
                const float up = __uint_as_float((uint32_t)(127 - e) << 23);
                row_factor[x][half] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int t = 0; t < kSteps; ++t)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float2 f = Half<true>::to_float2(q[x][t][half + 2 * w]);
                        q[x][t][half + 2 * w] = Half<false>::from_float2(f.x * up, f.y * up);
                    }
            }
        }

    unsigned char* ring = smem + warp * (S::kShared / WARPS);
    const uint32_t ring_at = shared_address(ring);
    bool bad = too_many || tokens > len;                  // the table is too short for the sequence

    // Loading.  Where blocks hold whole groups of 16 keys, the usual case, a group is one run of bytes.  Otherwise lanes
    // 0..15 each look up one key.  Either is done for the next stage while this one is copied.
    const bool grouped = p.cache.block_size % kFewKeys == 0;
    const int shift = (p.cache.block_size & (p.cache.block_size - 1)) == 0 ? 31 - __clz(p.cache.block_size) : -1;
    const int32_t* const table = p.batch.block_tables + seq * p.batch.table_stride;
    const int64_t head_offset = (int64_t)kv_head * p.cache.head_stride;
    const int groups = (range.end - range.begin + kFewKeys - 1) / kFewKeys;
    const int mine = groups > warp ? (groups - warp + WARPS - 1) / WARPS : 0;
    auto first_key = [&](int i) { return range.begin + (warp + i * WARPS) * kFewKeys; };
    auto look_up = [&](int i, int64_t& tile, int& offset) {   // byte offset of the key's tile, -1: nothing to load
        tile = -1;
        offset = 0;
        const int key = first_key(i) + (grouped ? 0 : lane & 15);
        if (i < mine && key < range.end) {
            const int entry = shift >= 0 ? key >> shift : key / p.cache.block_size;
            const int id = entry < p.batch.max_blocks ? table[entry] : -1;
            if ((unsigned)id >= (unsigned)p.cache.num_blocks) bad = true;
            else tile = id * p.cache.block_stride + head_offset;
            offset = key - entry * p.cache.block_size;
        }
    };
    int64_t next_tile;
    int next_offset;
    look_up(0, next_tile, next_offset);
    auto issue = [&](int i) {
        if (i < mine) {
            const uint32_t at = ring_at + (i % S::kStages) * S::kStage;
            if (grouped) {
                const int64_t rows_at = next_tile < 0 ? 0 : next_tile + (int64_t)next_offset * S::kRowBytes;
                const int count = next_tile < 0 ? 0 : range.end - first_key(i);       // keys that are there, if fewer than 16
                const char *k_from = p.cache.k + rows_at + lane * 16, *v_from = p.cache.v + rows_at + lane * 16;
#pragma unroll
                for (int u = 0; u < kChunks / 2; ++u) {
                    const int piece = u * 32 + lane, r = piece / kChunks, j = piece % kChunks;
                    const bool valid = r < count;
                    copy16(at + r * S::kRowBytes + ((j ^ ((r & 1) * kFlip)) * 16), valid ? k_from + u * 512 : p.cache.k, valid);
                    copy16(at + S::kTile + r * S::kRowBytes + ((j ^ turn(r)) * 16), valid ? v_from + u * 512 : p.cache.v, valid);
                }
                if (E4M3) {
                    const bool valid = (lane & 15) < count;
                    const int64_t from = next_tile + (int64_t)p.cache.block_size * HD + (next_offset + (lane & 15)) * 4;
                    copy4(at + 2 * S::kTile + lane * 4, (lane < 16 ? p.cache.k : p.cache.v) + (valid ? from : 0), valid);
                }
            } else {
#pragma unroll
                for (int u = 0; u < kChunks / 2; ++u) {
                    const int piece = u * 32 + lane, r = piece / kChunks, j = piece % kChunks;
                    const int64_t tile = __shfl_sync(0xffffffffu, next_tile, r);
                    const int64_t from = tile + (int64_t)__shfl_sync(0xffffffffu, next_offset, r) * S::kRowBytes + j * 16;
                    const bool valid = tile >= 0;
                    copy16(at + r * S::kRowBytes + ((j ^ ((r & 1) * kFlip)) * 16), p.cache.k + (valid ? from : 0), valid);
                    copy16(at + S::kTile + r * S::kRowBytes + ((j ^ turn(r)) * 16), p.cache.v + (valid ? from : 0), valid);
                }
                if (E4M3) {
                    const int64_t tile = __shfl_sync(0xffffffffu, next_tile, lane & 15);
                    const int64_t from = tile + (int64_t)p.cache.block_size * HD + __shfl_sync(0xffffffffu, next_offset, lane & 15) * 4;
                    copy4(at + 2 * S::kTile + lane * 4, (lane < 16 ? p.cache.k : p.cache.v) + (tile >= 0 ? from : 0), tile >= 0);
                }
            }
            look_up(i + 1, next_tile, next_offset);
        }
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);

    const int seen_by_all = min(first_pos + row0 / p.group + 1, range.end);    // keys before this one are seen by every row
    float m[MT][2], l[MT][2], o[MT][HD / 8][4];             // of rows quad and quad + 8 of each 16
#pragma unroll
    for (int x = 0; x < MT; ++x) {
        m[x][0] = m[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.f;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x][n][e] = 0.f;
    }
    for (int i = 0; i < mine; ++i) {
        issue(i + S::kStages - 1);
        copy_wait<S::kStages - 1>();
        __syncwarp();
        const uint32_t k_at = ring_at + (i % S::kStages) * S::kStage, v_at = k_at + S::kTile;
        // scores of 16 keys: tile n has keys 8 n + 2 c + {0, 1} of the lane's rows
        float sc[MT][2][4] = {};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int r = n * 8 + quad;
#pragma unroll
            for (int j = 0; j < kChunks / 4; ++j) {
                const uint4 w = load_shared16(k_at + r * S::kRowBytes + (((j * 4 + c) ^ ((r & 1) * kFlip)) * 16));
                const uint32_t in[4] = {w.x, w.y, w.z, w.w};
                if (E4M3) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t b0 = widen2(in[t]), b1 = widen2(in[t] >> 16);
#pragma unroll
                        for (int x = 0; x < MT; ++x) mma_16x8x16<kBf16>(sc[x][n], q[x][j * 4 + t], b0, b1);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        mma_16x8x16<kBf16>(sc[x][n], q[x][j * 2], in[0], in[1]);
                        mma_16x8x16<kBf16>(sc[x][n], q[x][j * 2 + 1], in[2], in[3]);
                    }
                }
            }
        }
        const int key = first_key(i) + 2 * c;
        float* const scales = reinterpret_cast<float*>(ring + (i % S::kStages) * S::kStage + 2 * S::kTile);     // K's, then V's
        float k_scale[2][2], lift[2][2];                       // K's scale, log2 of V's
        if (E4M3) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    k_scale[n][e] = scales[n * 8 + 2 * c + e];
                    lift[n][e] = __log2f(scales[kFewKeys + n * 8 + 2 * c + e]);
                }
        }
        float inverse[2][2];                                   // of V's scale
        auto find_inverse = [&] {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float scale = scales[kFewKeys + n * 8 + 2 * c + e];
                    inverse[n][e] = scale == 0.f ? 0.f : __fdividef(kSumUnit, scale);              // 0: a key that is not there
                }
        };
        if (E4M3) find_inverse();
        const bool all = first_key(i) + kFewKeys <= seen_by_all;               // every row sees all of these keys
        float top[MT][2];
        auto find_top = [&] {
#pragma unroll
            for (int x = 0; x < MT; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[x][h] = fmaxf(fmaxf(m[x][h], fmaxf(sc[x][0][2 * h], sc[x][0][2 * h + 1])), fmaxf(sc[x][1][2 * h], sc[x][1][2 * h + 1]));
#pragma unroll
                    for (int d = 1; d < 4; d <<= 1) top[x][h] = fmaxf(top[x][h], __shfl_xor_sync(0xffffffffu, top[x][h], d));
                }
        };
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y = sc[x][n][e] * (E4M3 ? row_factor[x][e / 2] * k_scale[n][e & 1] : row_factor[x][e / 2]);
                    if (E4M3) y += lift[n][e & 1];
                    const int at = key + n * 8 + (e & 1);
                    if (!all) y = at <= last[x][e / 2] && at < range.end ? y : -INFINITY;
                    sc[x][n][e] = y;
                }
        find_top();
        bool grown = false;
#pragma unroll
        for (int x = 0; x < MT; ++x) grown |= top[x][0] > m[x][0] || top[x][1] > m[x][1];
        auto is_one = [](float log2_scale) { return fabsf(log2_scale) < 0.5f; };        // log2 is approximate, scales are powers of two
        if (__any_sync(0xffffffffu, grown)) {
            if (E4M3 && __any_sync(0xffffffffu, is_one(lift[0][0]) || is_one(lift[0][1]) || is_one(lift[1][0]) || is_one(lift[1][1]))) {
                // Whose rows of V are zeros?  A lane looks at half of key (lane & 15)'s.
                uint32_t codes = 0;
#pragma unroll 1
                for (int u = 0; u < kChunks / 2; ++u) {
                    const uint4 w = load_shared16(v_at + (lane & 15) * S::kRowBytes + (lane >> 4) * (S::kRowBytes / 2) + u * 16);
                    codes |= w.x | w.y | w.z | w.w;
                }
                uint32_t zeros = __ballot_sync(0xffffffffu, scales[kFewKeys + (lane & 15)] == 1.f && (codes & 0x7f7f7f7fu) == 0);
                zeros &= zeros >> 16;
                if (zeros >> lane & 1) scales[kFewKeys + lane] = kZeroRowScale;
                __syncwarp();
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (zeros >> (n * 8 + 2 * c + e) & 1) {
#pragma unroll
                            for (int x = 0; x < MT; ++x) {
                                sc[x][n][e] += kZeroRowLog2;
                                sc[x][n][e + 2] += kZeroRowLog2;
                            }
                        }
                find_top();
                find_inverse();
            }
#pragma unroll
            for (int x = 0; x < MT; ++x) {
                float keep[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    keep[h] = m[x][h] == top[x][h] ? 1.f : exp2_fast(m[x][h] - top[x][h]);
                    m[x][h] = top[x][h];
                    l[x][h] *= keep[h];
                }
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][n][e] *= keep[e / 2];
            }
        }
        uint32_t a[MT][4];
#pragma unroll
        for (int x = 0; x < MT; ++x) {
            constexpr float top_log2 = E4M3 ? kTopLog2 : 0.f;
            const float base[2] = {m[x][0] == -INFINITY ? 0.f : m[x][0] - top_log2, m[x][1] == -INFINITY ? 0.f : m[x][1] - top_log2};   // a row without a key yet
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = exp2_fast(sc[x][n][e] - base[e / 2]);
                    sc[x][n][e] = y;
                    l[x][e / 2] += E4M3 ? y * inverse[n][e & 1] : y;
                }
            a[x][0] = In::from_float2(sc[x][0][0], sc[x][0][1]);
            a[x][1] = In::from_float2(sc[x][0][2], sc[x][0][3]);
            a[x][2] = In::from_float2(sc[x][1][0], sc[x][1][1]);
            a[x][3] = In::from_float2(sc[x][1][2], sc[x][1][3]);
        }
        // o += P V: a lane gives ldmatrix the row of key (lane & 15), and the left or right of two neighbouring pieces
#pragma unroll
        for (int j = 0; j < kChunks; j += 2) {
            const int r = lane & 15, piece = j + (lane >> 4);
            const uint4 w = load_matrices_transposed(v_at + r * S::kRowBytes + ((piece ^ turn(r)) * 16));
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            if (E4M3) {
                // a register has, for two keys, two neighbouring values each: even ones and odd ones make two tiles
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const uint32_t pick = y & 1 ? 0x4431 : 0x4420;
                    const uint32_t b0 = widen2(__byte_perm(in[y & 2], 0, pick)), b1 = widen2(__byte_perm(in[(y & 2) + 1], 0, pick));
#pragma unroll
                    for (int x = 0; x < MT; ++x) mma_16x8x16<kBf16>(o[x][j * 2 + y], a[x], b0, b1);
                }
            } else {
#pragma unroll
                for (int x = 0; x < MT; ++x) {
                    mma_16x8x16<kBf16>(o[x][j], a[x], in[0], in[1]);
                    mma_16x8x16<kBf16>(o[x][j + 1], a[x], in[2], in[3]);
                }
            }
        }
        __syncwarp();                                          // the stage may be filled again
    }
    copy_wait<0>();
    bad = __any_sync(0xffffffffu, bad);
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int d = 1; d < 4; d <<= 1) l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], d);
            if (E4M3) l[x][h] *= 1.f / (kTop * kSumUnit);
            if (bad) l[x][h] = not_a_number();
        }

    // Join the warps: each leaves its maximum, sum and output in what was its ring.
    __syncwarp();
    float* join = reinterpret_cast<float*>(ring);
    float* out = join + S::kRows * 2;
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = x * 16 + quad + h * 8;
            if (c == 0) {
                join[r * 2] = m[x][h];
                join[r * 2 + 1] = l[x][h];
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                // columns of the lane's values: 8 n + 2 c + {0, 1}, or of the even/odd tiles 16 (n/2) + 4 c + n%2 + {0, 2}
                const int d = E4M3 ? 16 * (n / 2) + 4 * c + n % 2 : 8 * n + 2 * c, step = E4M3 ? 2 : 1;
                constexpr float down = E4M3 ? 1.f / kTop : 1.f;
                out[r * HD + d] = o[x][n][2 * h] * down;
                out[r * HD + d + step] = o[x][n][2 * h + 1] * down;
            }
        }
    __syncthreads();
    const int64_t written = too_many ? total : rows;          // all of a sequence's rows become NaN if there are too many
    constexpr int kPairs = HD / 2;
    for (int64_t x = threadIdx.x; x < written * kPairs; x += WARPS * 32) {
        const int64_t r = x / kPairs;
        const int d = (int)(x % kPairs) * 2, in = too_many ? 0 : (int)r;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, reinterpret_cast<const float*>(smem + w * (S::kShared / WARPS))[in * 2]);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* from = reinterpret_cast<const float*>(smem + w * (S::kShared / WARPS));
            const float f = exp2_fast(from[in * 2] - base);
            const float2 v = *reinterpret_cast<const float2*>(from + S::kRows * 2 + in * HD + d);
            l += f * from[in * 2 + 1];
            a += f * v.x;
            b += f * v.y;
        }
        const int64_t row = s.first + (row0 + r) / p.group, head = kv_head * p.group + (row0 + r) % p.group;
        if (too_many || whole) {
            const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);           // no key: zeros; NaN stays
            if (split == 0)
                *reinterpret_cast<uint32_t*>(p.out.data + row * p.out.row_stride + head * p.out.head_stride + d * 2) = H::from_float2(a * inv, b * inv);
        } else {
            const int64_t place = (row * p.heads + head) * p.parts + split;
            *reinterpret_cast<float2*>(p.part_out + place * HD + d) = make_float2(a, b);
            if (d == 0) p.part_stat[place] = make_float2(m, l);
        }
    }
}

// Joins the parts' partial results, in their order.  (64 results of 37 parts each: 7 us with a block for each, 19 us with a
// warp for each.)  WIDE: a block per row and query head, whose warps share the parts;
// else a warp for each.  No more blocks than the device holds at once, so that most warps find the batch in the
// first-level cache.  The grid begins while its predecessor still runs and waits for it before it reads results.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
template <int HD, bool BF16, bool WIDE>
__global__ void __launch_bounds__(kJoinThreads) attend_join(const __grid_constant__ AttnParams p) {
    constexpr int N = HD / 32;                                // values of a lane
    __shared__ float shared[WIDE ? kJoinWarps * (HD + 2) : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = WIDE ? warp : 0, step = WIDE ? kJoinWarps : 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int few_units = p.few.parts > 1 ? p.part_chosen[0] : kUncut, tile_units = p.tiles.parts > 1 ? p.part_chosen[1] : kUncut;
    if (few_units == kUncut && tile_units == kUncut) return;
    const int64_t items = (int64_t)p.batch.num_rows * p.heads, stride = (int64_t)gridDim.x * (WIDE ? 1 : kJoinWarps);
    for (int64_t item = (int64_t)blockIdx.x * (WIDE ? 1 : kJoinWarps) + (WIDE ? 0 : warp); item < items; item += stride) {
        const int row = (int)(item / p.heads), head = (int)(item % p.heads);
        const int seq = find_sequence(p.batch.starts, p.batch.num_seqs, row);
        const Sequence s = sequence_at(p.batch, seq);
        if (row < s.first || row - s.first >= s.rows || s.rows > p.batch.max_rows) continue;
        const int len = min(max(p.batch.seq_lens[seq], 0), capacity(p.batch, p.cache));
        const bool few = (int64_t)s.rows * p.group <= p.few_rows;
        const int64_t per = part_keys(len, few ? p.few : p.tiles, few ? few_units : tile_units);
        if (per >= len) continue;                             // written by its only part
        const int parts = (int)((len + per - 1) / per);
        const int64_t place = item * p.parts;
        float m = -INFINITY, l = 0.f, o[N] = {};
        for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_stat[place + i].x);
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 4
        for (int i = first; i < parts; i += step) {
            const float2 stat = p.part_stat[place + i];
            const float f = exp2_fast(stat.x - base);
            l += f * stat.y;
            const float* from = p.part_out + (place + i) * HD + lane * N;
#pragma unroll
            for (int n = 0; n < N; n += 2) {
                const float2 v = *reinterpret_cast<const float2*>(from + n);
                o[n] += f * v.x;
                o[n + 1] += f * v.y;
            }
        }
        if (WIDE) {
            __syncthreads();                                  // the previous item has been read
            float* mine = shared + warp * (HD + 2);
            if (lane == 0) mine[HD] = l;
#pragma unroll
            for (int n = 0; n < N; ++n) mine[lane * N + n] = o[n];
            __syncthreads();
            if (warp > 0) continue;
#pragma unroll
            for (int w = 1; w < kJoinWarps; ++w) {
                l += shared[w * (HD + 2) + HD];
#pragma unroll
                for (int n = 0; n < N; ++n) o[n] += shared[w * (HD + 2) + lane * N + n];
            }
        }
        const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
        uint32_t* to = reinterpret_cast<uint32_t*>(p.out.data + (int64_t)row * p.out.row_stride + (int64_t)head * p.out.head_stride) + lane * (N / 2);
#pragma unroll
        for (int n = 0; n < N; n += 2) to[n / 2] = Half<BF16>::from_float2(o[n] * inv, o[n + 1] * inv);
    }
}

}  // namespace kvmig
