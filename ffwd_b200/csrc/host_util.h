// Host helpers shared by the translation units that implement C entry points
// (defined in engine.cu).
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace fb {

// Records the calling thread's error message and prints it to stderr.
void fail(const char *fmt, ...);
// Clears the calling thread's error message.
void clear_error();

// Kernel launches issued by this process.
extern std::atomic<long long> g_launches;

#define CK(expr)                                                                              \
    do {                                                                                      \
        cudaError_t _e = (cudaError_t)(expr);                                                 \
        if (_e != cudaSuccess) {                                                              \
            ::fb::fail("%s failed: %s (%s:%d)", #expr, cudaGetErrorString(_e), __FILE__,      \
                       __LINE__);                                                             \
            return -1;                                                                        \
        }                                                                                     \
    } while (0)

// Kernel launch wrappers return a cudaError_t value; count every launch.
#define LAUNCH(expr)                   \
    do {                               \
        ::fb::g_launches.fetch_add(1); \
        CK(expr);                      \
    } while (0)

// 2-D row-major tensor map of [rows, cols] elements of `esz` bytes with a row
// stride of ld elements; box = box_rows x box_cols.  -1 (with a message) on failure.
int make_map_ld(CUtensorMap *m, const void *ptr, uint64_t rows, uint64_t cols, uint64_t ld,
                uint32_t box_rows, uint32_t box_cols, CUtensorMapSwizzle sw,
                CUtensorMapDataType dt, int esz);

}  // namespace fb
