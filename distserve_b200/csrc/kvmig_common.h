// What the library's translation units share on the host side: the error convention and the counters
// (defined in kvmig.cu), and the checks of the cache and attention entry points (kvcache.cu).
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/kvmig.h"

namespace kvmig {

// Records the text of a failure for kvmig_last_error() and returns `code`.
int fail(int code, const char* fmt, ...);
void clear_error();
int check_shape(const kvmig_pool_shape* s, const char* what);

// Blocks of the attention kernels on the current device that gave up waiting (their rows are NaN); waits for the device.
int64_t attention_timeouts();

extern std::atomic<int64_t> g_cache_launches, g_attention_launches;

#define CU_TRY(expr)                                                                       \
    do {                                                                                   \
        cudaError_t e_ = (expr);                                                           \
        if (e_ != cudaSuccess)                                                             \
            return fail(KVMIG_ECUDA, "%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e_), \
                        __FILE__, __LINE__);                                               \
    } while (0)

int check_rows(const kvmig_rows* r, int64_t head_dim, int64_t num_rows, const char* what);
int check_batch(const kvmig_batch* b, bool tables, bool lens, const char* what);
int check_pools(const void* k_cache, const void* v_cache, const kvmig_pool_shape* shape, int64_t layer, int dtype, const char* what);

}  // namespace kvmig
