// Device code shared by the cache kernels (kvcache.cu) and the attention kernels (kvattn.cu): where a token lies in
// a paged pool, and the conversions between 16-bit rows and e4m3 codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace kvmig {

// One layer of a pool pair, and the block tables that lead into it.  Byte addresses: a pool of more than 2^31
// elements is ordinary, so every product with a block number is 64-bit.
struct CacheView {
    char* k;                       // address of (block 0, this layer, head 0)
    char* v;
    int64_t block_stride;          // bytes from one block to the next
    int32_t head_stride;           // bytes from one head's tile to the next
    int32_t num_blocks, block_size;
};

struct BatchView {
    const int32_t* starts;
    const int32_t* seq_lens;
    const int32_t* block_tables;
    int64_t table_stride;
    int32_t num_seqs, num_rows, max_rows, max_blocks;
};

// The last sequence that starts at or before row t, found by all lanes of a warp together: each step probes 32
// places at once, so a batch of up to 32 sequences takes one load and one of up to 1024 two.
__device__ __forceinline__ int find_sequence(const int32_t* starts, int n, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, count = n;                       // the answer is in [lo, lo + count)
    while (count > 1) {
        const int step = (count + 31) / 32;
        const int at = lo + lane * step;
        const bool before = at < lo + count && starts[at] <= t;
        const int hits = __popc(__ballot_sync(0xffffffffu, before));
        if (hits == 0) return lo;
        const int next = lo + (hits - 1) * step;
        count = min(step, lo + count - next);
        lo = next;
    }
    return lo;
}

struct Sequence {
    int first, rows;    // its rows
    bool valid;
};

__host__ __device__ __forceinline__ Sequence sequence_at(const BatchView& b, int i) {
    Sequence s;
    s.first = b.starts[i];
    const int end = b.starts[i + 1];
    s.valid = s.first >= 0 && end >= s.first && end <= b.num_rows;
    s.rows = s.valid ? end - s.first : 0;
    return s;
}

// Block that holds position `pos` (>= 0) of a sequence, or -1 if the table or the pool has no such block.
__host__ __device__ __forceinline__ int block_of(const BatchView& b, const CacheView& c, int seq, int pos) {
    const int entry = pos / c.block_size;
    if (entry >= b.max_blocks) return -1;
    const int id = b.block_tables[seq * b.table_stride + entry];
    return (unsigned)id < (unsigned)c.num_blocks ? id : -1;
}

// Tokens that a table has room for (kept below 2^31 so that positions rounded up to a tile still fit 32 bits).
__host__ __device__ __forceinline__ int capacity(const BatchView& b, const CacheView& c) {
    const int64_t n = (int64_t)b.max_blocks * c.block_size;
    return n < 0x7fff0000 ? (int)n : 0x7fff0000;
}

// ---- 16-bit types ----------------------------------------------------------------------------------------

template <bool BF16> struct Half;
template <> struct Half<false> {
    static constexpr uint32_t kInf = 0x7c00, kNan2 = 0x7fff7fff;
    static __device__ __forceinline__ float2 to_float2(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
    static __device__ __forceinline__ uint32_t from_float2(float a, float b) {
        __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float largest() { return 65504.f; }
};
template <> struct Half<true> {
    static constexpr uint32_t kInf = 0x7f80, kNan2 = 0x7fff7fff;
    static __device__ __forceinline__ float2 to_float2(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t from_float2(float a, float b) {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float largest() { return __uint_as_float(0x7f7f0000u); }
};

// ---- e4m3 codes ------------------------------------------------------------------------------------------

constexpr int kMinScaleExponent = -100;

// Scale of a row whose largest magnitude has the 16-bit pattern `top`: 2^e for the smallest e >= -100 with
// value <= 448 * 2^e (448 = 1.75 * 2^8), 1 for zero, NaN for an infinity or a NaN.  *inverse is 1 / scale, exact.
template <bool BF16>
__device__ __forceinline__ float row_scale(uint32_t top, float* inverse) {
    if (top >= Half<BF16>::kInf) {
        *inverse = __uint_as_float(0x7fffffffu);
        return *inverse;
    }
    if (top == 0) {
        *inverse = 1.f;
        return 1.f;
    }
    const uint32_t bits = __float_as_uint(Half<BF16>::to_float2(top).x);
    int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kMinScaleExponent);
    *inverse = __uint_as_float(uint32_t(127 - e) << 23);
    return __uint_as_float(uint32_t(127 + e) << 23);
}

__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

__device__ __forceinline__ float2 decode2(uint32_t codes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes & 0xffffu), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Pairs of 32-bit floats: one instruction for both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ float2 unpair(uint64_t x) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(x));
    return f;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t x;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(a), "l"(b), "l"(c));
    return x;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t x;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
    return x;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t x;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
    return x;
}

// Two e4m3 codes (the low 16 bits) as two 16-bit floats; exact.
__device__ __forceinline__ uint32_t widen2(uint32_t codes) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes & 0xffffu), __NV_E4M3);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 e4m3 codes times their row's scale as 16-bit values: values beyond the type's largest become that.
template <bool BF16>
__device__ __forceinline__ void widen16(const uint4& codes, float scale, uint4& lo, uint4& hi) {
    const uint32_t in[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t out[8];
    if (!BF16 && scale >= 0x1p-24f && scale <= 128.f) {
        // the scale is a 16-bit value itself and no product leaves the range
        const __half2 s = __float2half2_rn(scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t w = widen2(in[j / 2] >> (j % 2 * 16));
            const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&w), s);
            out[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
    } else if (BF16 && scale <= 0x1p100f) {
        const uint64_t s = pair(scale, scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 f = decode2(in[j / 2] >> (j % 2 * 16)), y = unpair(mul_pair(pair(f.x, f.y), s));
            out[j] = Half<true>::from_float2(y.x, y.y);
        }
    } else {
        using H = Half<BF16>;
        const float top = H::largest();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float2 f = decode2(in[j / 2] >> (j % 2 * 16));
            f.x *= scale;
            f.y *= scale;
            f.x = f.x > top ? top : f.x < -top ? -top : f.x;
            f.y = f.y > top ? top : f.y < -top ? -top : f.y;
            out[j] = H::from_float2(f.x, f.y);
        }
    }
    lo = make_uint4(out[0], out[1], out[2], out[3]);
    hi = make_uint4(out[4], out[5], out[6], out[7]);
}

}  // namespace kvmig
