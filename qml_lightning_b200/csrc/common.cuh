// Shared helpers for the qmlb200 kernels (error reporting, launch checks, small device utilities).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "qmlb200.h"

namespace qmlb {

// Stores a printf-style message in a thread-local buffer returned by qmlb_last_error().
void set_error(const char *fmt, ...);

// Returns QMLB_OK or records the pending CUDA launch error under `what`.
int check_launch(const char *what);

inline cudaStream_t as_stream(qmlb_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

// Opt a kernel into as much dynamic shared memory as it may have.  Always the same size, whatever this call wants: a smaller one
// could come between the setting and the launch of another host thread.
int opt_in_smem(const void *kernel, size_t bytes, const char *what);

// The same when more than 48 KB of dynamic shared memory are wanted.
template <typename K>
inline int ensure_smem(K kernel, size_t bytes, const char *what) {
    return bytes > 48 * 1024 ? opt_in_smem(reinterpret_cast<const void *>(kernel), bytes, what) : QMLB_OK;
}

}  // namespace qmlb

#define QMLB_REQUIRE(cond, ...)              \
    do {                                     \
        if (!(cond)) {                       \
            qmlb::set_error(__VA_ARGS__);    \
            return QMLB_ERR_INVALID;         \
        }                                    \
    } while (0)

#define QMLB_FULL_MASK 0xffffffffu

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(QMLB_FULL_MASK, v, o);
    return v;
}
