// Attention of few rows over the paged cache: a decoding step's single tokens and short drafts.
//
// A block takes the rows of one sequence that share a KV head, up to 16 of them (tokens x query heads of the group), and
// one split of that sequence's keys.  Every K and V value is used for 16 rows at most, so the kernel is bound by reading
// the cache; all else is arranged around keeping reads in flight:
//   * each warp has its own ring of stages of 16 keys in shared memory, filled by cp.async and drained by that warp
//     alone: no barrier of the block until the end, and about 96 KiB in flight per SM (two blocks);
//   * warps take the groups of 16 keys in turn and keep their own running maximum, sum and output, joined at the end;
//   * products run on m16n8k16 matrix instructions with the rows padded to 16.  Contraction order is free, so K
//     fragments are read as 16 consecutive bytes per lane and Q's values are permuted to match, once;
//   * e4m3 codes widen to 16 bits in registers; K's scales multiply the scores.  V's scale s_j goes into the exponent,
//     P_j = 2^(score_j + log2 s_j - m), and the sum counts P_j / s_j: nothing can leave the 16-bit range that way.
#pragma once

#include "kvattn_device.cuh"

namespace kvmig {

constexpr int kFewWarps = 4, kFewRows = 16, kFewKeys = 16;

template <int HD, bool E4M3> struct FewShape {
    static constexpr int kRowBytes = HD * (E4M3 ? 1 : 2);
    static constexpr int kTile = kFewKeys * kRowBytes;                          // K or V of one stage
    static constexpr int kStage = 2 * kTile + (E4M3 ? 2 * kFewKeys * 4 : 0);    // and the scales behind them
    static constexpr int kStages = 24576 / kStage < 8 ? 24576 / kStage : 8;
    static constexpr int kRing = kStages * kStage;
    static constexpr int kJoin = kFewRows * (HD + 2) * 4;                       // a warp's result, in its own ring
    static constexpr int kShared = kFewWarps * (kRing > kJoin ? kRing : kJoin);
};

template <int HD, bool BF16, bool E4M3>
__global__ void __launch_bounds__(kFewWarps * 32) attend_few(const __grid_constant__ AttnParams p) {
    using S = FewShape<HD, E4M3>;
    using H = Half<BF16>;
    constexpr int kSteps = HD / 16;                       // contraction steps of q . k
    constexpr int kChunks = S::kRowBytes / 16;            // 16-byte pieces of a cached row
    constexpr int kFlip = kChunks >= 8 ? 4 : 0;           // odd keys swap their 64-byte halves: no bank conflicts
    auto turn = [](int r) { return kChunks >= 8 ? r & 7 : (r >> 1) & 3; };   // V's pieces are turned by the key for ldmatrix
    extern __shared__ __align__(128) unsigned char smem[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, c = lane & 3;
    const int kv_heads = p.heads / p.group;
    const int kv_head = blockIdx.x % kv_heads, seq = blockIdx.x / kv_heads, split = blockIdx.y;
    const Sequence s = sequence_at(p.batch, seq);
    if (s.rows == 0) return;
    const bool too_many = s.rows > p.batch.max_rows;
    const int rows = too_many ? 0 : s.rows * p.group;     // rows of the tile: token * group + query head of the group
    const int tokens = max(p.batch.seq_lens[seq], 0), first_pos = tokens - s.rows;   // position of the first row; may be negative
    const int len = min(tokens, capacity(p.batch, p.cache));
    KeyRange range = split_range(len, p.splits, split);
    const bool whole = split_range(len, p.splits, 0).end == len;               // one split has everything
    if (split > 0 && (whole || range.begin >= len)) return;
    if (too_many) range.end = range.begin;

    // Q: lane (quad, c) has rows quad and quad + 8.  16-bit pools: step t, values 32 (t/2) + 8 c + 4 (t%2) + 0..3;
    // quantised pools: 64 (t/4) + 16 c + 4 (t%4) + 0..3.
    uint32_t q[kSteps][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int r = quad + half * 8;
        const bool there = r < rows;
        const char* at = p.q.data + (int64_t)(s.first + (there ? r / p.group : 0)) * p.q.row_stride +
                         (int64_t)(kv_head * p.group + (there ? r % p.group : 0)) * p.q.head_stride;
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            const int d = E4M3 ? 64 * (t / 4) + 16 * c + 4 * (t % 4) : 32 * (t / 2) + 8 * c + 4 * (t % 2);
            uint2 w = make_uint2(0, 0);
            if (there) w = __ldg(reinterpret_cast<const uint2*>(at + d * 2));
            q[t][half] = w.x;
            q[t][half + 2] = w.y;
        }
    }
    // The last key that each of the lane's two rows sees.
    const int last0 = first_pos + quad / p.group, last1 = first_pos + (quad + 8) / p.group;

    unsigned char* ring = smem + warp * (S::kShared / kFewWarps);
    const uint32_t ring_at = shared_address(ring);
    bool bad = too_many || tokens > len;                  // the table is too short for the sequence

    // Loading.  Lanes 0..15 each look up one key of the stage to be loaded, one stage ahead of its copies.
    const int64_t head_offset = (int64_t)kv_head * p.cache.head_stride;
    const int groups = (range.end - range.begin + kFewKeys - 1) / kFewKeys;
    const int mine = groups > warp ? (groups - warp + kFewWarps - 1) / kFewWarps : 0;
    auto first_key = [&](int i) { return range.begin + (warp + i * kFewWarps) * kFewKeys; };
    auto look_up = [&](int i, int64_t& tile, int& offset) {   // byte offset of the key's tile, -1: nothing to load
        tile = -1;
        offset = 0;
        const int key = first_key(i) + (lane & 15);
        if (i < mine && key < range.end) {
            const int id = block_of(p.batch, p.cache, seq, key);
            if (id < 0) bad = true;
            else tile = id * p.cache.block_stride + head_offset;
            offset = key % p.cache.block_size;
        }
    };
    int64_t next_tile;
    int next_offset;
    look_up(0, next_tile, next_offset);
    auto issue = [&](int i) {
        if (i < mine) {
            const uint32_t at = ring_at + (i % S::kStages) * S::kStage;
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
            look_up(i + 1, next_tile, next_offset);
        }
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue(i);

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // of rows quad and quad + 8
    float o[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (int i = 0; i < mine; ++i) {
        issue(i + S::kStages - 1);
        copy_wait<S::kStages - 1>();
        __syncwarp();
        const uint32_t k_at = ring_at + (i % S::kStages) * S::kStage, v_at = k_at + S::kTile;
        // scores of 16 keys: tile n has keys 8 n + 2 c + {0, 1} of the lane's two rows
        float sc[2][4] = {};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int r = n * 8 + quad;
#pragma unroll
            for (int j = 0; j < kChunks / 4; ++j) {
                const uint4 w = load_shared16(k_at + r * S::kRowBytes + (((j * 4 + c) ^ ((r & 1) * kFlip)) * 16));
                if (E4M3) {
                    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int t = 0; t < 4; ++t) mma_16x8x16<BF16>(sc[n], q[j * 4 + t], widen2<BF16>(in[t]), widen2<BF16>(in[t] >> 16));
                } else {
                    mma_16x8x16<BF16>(sc[n], q[j * 2], w.x, w.y);
                    mma_16x8x16<BF16>(sc[n], q[j * 2 + 1], w.z, w.w);
                }
            }
        }
        const int key = first_key(i) + 2 * c;
        float inverse[2][2];                                  // 1 / V's scale
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float ks[2] = {p.scale_log2, p.scale_log2}, lift[2] = {0.f, 0.f};
            if (E4M3) {
                const float* scales = reinterpret_cast<const float*>(ring + (i % S::kStages) * S::kStage + 2 * S::kTile) + n * 8 + 2 * c;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    ks[e] *= scales[e];
                    lift[e] = __log2f(scales[16 + e]);
                    inverse[n][e] = __fdividef(1.f, scales[16 + e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = key + n * 8 + (e & 1), last = e < 2 ? last0 : last1;
                const float x = sc[n][e] * ks[e & 1] + lift[e & 1];
                sc[n][e] = at <= last && at < range.end ? x : -INFINITY;
            }
        }
        float top0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
        float top1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, d));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, d));
        }
        top0 = fmaxf(m0, top0);
        top1 = fmaxf(m1, top1);
        if (__any_sync(0xffffffffu, top0 > m0 || top1 > m1)) {
            const float keep0 = m0 == top0 ? 1.f : exp2_fast(m0 - top0), keep1 = m1 == top1 ? 1.f : exp2_fast(m1 - top1);
            m0 = top0;
            m1 = top1;
            l0 *= keep0;
            l1 *= keep1;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
                o[n][0] *= keep0;
                o[n][1] *= keep0;
                o[n][2] *= keep1;
                o[n][3] *= keep1;
            }
        }
        const float base0 = m0 == -INFINITY ? 0.f : m0, base1 = m1 == -INFINITY ? 0.f : m1;   // a row that has seen no key yet
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[n][e] = exp2_fast(sc[n][e] - (e < 2 ? base0 : base1));
                // a key that is not there may have any scale: it adds nothing
                const float add = E4M3 ? (sc[n][e] == 0.f ? 0.f : sc[n][e] * inverse[n][e & 1]) : sc[n][e];
                if (e < 2) l0 += add;
                else l1 += add;
            }
        const uint32_t a[4] = {H::from_float2(sc[0][0], sc[0][1]), H::from_float2(sc[0][2], sc[0][3]),
                               H::from_float2(sc[1][0], sc[1][1]), H::from_float2(sc[1][2], sc[1][3])};
        // o += P V: a lane gives ldmatrix the row of key (lane & 15), and the left or right of two neighbouring pieces
#pragma unroll
        for (int j = 0; j < kChunks; j += 2) {
            const int r = lane & 15, piece = j + (lane >> 4);
            const uint4 w = load_matrices_transposed(v_at + r * S::kRowBytes + ((piece ^ turn(r)) * 16));
            if (E4M3) {
                // a register has, for two keys, two neighbouring values each: even ones and odd ones make two tiles
                const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mma_16x8x16<BF16>(o[(j + x) * 2], a, widen2<BF16>(__byte_perm(in[2 * x], 0, 0x4420)), widen2<BF16>(__byte_perm(in[2 * x + 1], 0, 0x4420)));
                    mma_16x8x16<BF16>(o[(j + x) * 2 + 1], a, widen2<BF16>(__byte_perm(in[2 * x], 0, 0x4431)), widen2<BF16>(__byte_perm(in[2 * x + 1], 0, 0x4431)));
                }
            } else {
                mma_16x8x16<BF16>(o[j], a, w.x, w.y);
                mma_16x8x16<BF16>(o[j + 1], a, w.z, w.w);
            }
        }
        __syncwarp();                                          // the stage may be filled again
    }
    copy_wait<0>();
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (__any_sync(0xffffffffu, bad)) l0 = l1 = not_a_number();

    // Join the warps: each leaves its maximum, sum and output in what was its ring.
    __syncwarp();
    float* join = reinterpret_cast<float*>(ring);
    if (c == 0) {
        join[quad * 2] = m0;
        join[quad * 2 + 1] = l0;
        join[(quad + 8) * 2] = m1;
        join[(quad + 8) * 2 + 1] = l1;
    }
    float* out = join + kFewRows * 2;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
        // columns of the lane's values: 8 n + 2 c + {0, 1}, or of the even/odd tiles 16 (n/2) + 4 c + n%2 + {0, 2}
        const int d = E4M3 ? 16 * (n / 2) + 4 * c + n % 2 : 8 * n + 2 * c, step = E4M3 ? 2 : 1;
        out[quad * HD + d] = o[n][0];
        out[quad * HD + d + step] = o[n][1];
        out[(quad + 8) * HD + d] = o[n][2];
        out[(quad + 8) * HD + d + step] = o[n][3];
    }
    __syncthreads();
    const int64_t total = (int64_t)s.rows * p.group;          // all of a sequence's rows become NaN if there are too many
    constexpr int kPairs = HD / 2;
    for (int64_t x = threadIdx.x; x < total * kPairs; x += kFewWarps * 32) {
        const int64_t r = x / kPairs;
        const int d = (int)(x % kPairs) * 2, in = too_many ? 0 : (int)r;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) m = fmaxf(m, reinterpret_cast<const float*>(smem + w * (S::kShared / kFewWarps))[in * 2]);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, a = 0.f, b = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float* from = reinterpret_cast<const float*>(smem + w * (S::kShared / kFewWarps));
            const float f = exp2_fast(from[in * 2] - base);
            const float2 v = *reinterpret_cast<const float2*>(from + kFewRows * 2 + in * HD + d);
            l += f * from[in * 2 + 1];
            a += f * v.x;
            b += f * v.y;
        }
        const int64_t row = s.first + r / p.group, head = kv_head * p.group + r % p.group;
        if (too_many || whole) {
            const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);           // no key: zeros; NaN stays
            if (split == 0)
                *reinterpret_cast<uint32_t*>(p.out.data + row * p.out.row_stride + head * p.out.head_stride + d * 2) = H::from_float2(a * inv, b * inv);
        } else {
            const int64_t part = (row * p.heads + head) * p.splits + split;
            *reinterpret_cast<float2*>(p.part_out + part * HD + d) = make_float2(a, b);
            if (d == 0) p.part_stat[part] = make_float2(m, l);
        }
    }
}

// Joins the splits' partial results, in their order: a warp per row and query head.
template <int HD, bool BF16>
__global__ void __launch_bounds__(128) attend_join(const __grid_constant__ AttnParams p) {
    constexpr int N = HD / 32;                                // values of a lane
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), row64 = warp / p.heads;
    if (row64 >= p.batch.num_rows) return;
    const int row = (int)row64, head = (int)(warp % p.heads);
    const int seq = find_sequence(p.batch.starts, p.batch.num_seqs, row);
    const Sequence s = sequence_at(p.batch, seq);
    if (row < s.first || row - s.first >= s.rows || s.rows > p.batch.max_rows) return;
    const int len = min(max(p.batch.seq_lens[seq], 0), capacity(p.batch, p.cache));
    if (split_range(len, p.splits, 0).end == len) return;     // written by its only split
    const int64_t part = warp * p.splits;
    float m = -INFINITY, l = 0.f, o[N] = {};
    for (int i = 0; i < p.splits && split_range(len, p.splits, i).begin < len; ++i) m = fmaxf(m, p.part_stat[part + i].x);
    const float base = m == -INFINITY ? 0.f : m;
    for (int i = 0; i < p.splits && split_range(len, p.splits, i).begin < len; ++i) {
        const float2 stat = p.part_stat[part + i];
        const float f = exp2_fast(stat.x - base);
        l += f * stat.y;
        const float* from = p.part_out + (part + i) * HD + lane * N;
#pragma unroll
        for (int n = 0; n < N; n += 2) {
            const float2 v = *reinterpret_cast<const float2*>(from + n);
            o[n] += f * v.x;
            o[n + 1] += f * v.y;
        }
    }
    const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
    uint32_t* to = reinterpret_cast<uint32_t*>(p.out.data + (int64_t)row * p.out.row_stride + (int64_t)head * p.out.head_stride) + lane * (N / 2);
#pragma unroll
    for (int n = 0; n < N; n += 2) to[n / 2] = Half<BF16>::from_float2(o[n] * inv, o[n + 1] * inv);
}

}  // namespace kvmig
