// Error reporting and library identification for the qmlb200 C ABI.
#include <stdarg.h>
#include <stdio.h>

#include <atomic>

#include "common.cuh"

namespace qmlb {

static thread_local char g_error[512] = "";

void set_error(const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

int check_launch(const char *what) {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return QMLB_OK;
    set_error("%s: %s", what, cudaGetErrorString(e));
    return QMLB_ERR_CUDA;
}

// Shared memory that a kernel's own variables take, asked once per kernel; < 0: error.  The table is filled without a lock: a thread
// that finds no entry yet asks by itself.
static int own_smem(const void *kernel) {
    constexpr int SIZE = 1024;
    struct Entry {
        std::atomic<const void *> kernel{nullptr};
        std::atomic<int> bytes_plus_one{0};
    };
    static Entry table[SIZE];
    Entry *free_entry = nullptr;
    const size_t first = (reinterpret_cast<uintptr_t>(kernel) >> 4) % SIZE;
    for (int i = 0; i < SIZE && free_entry == nullptr; ++i) {
        Entry &e = table[(first + i) % SIZE];
        const void *k = e.kernel.load(std::memory_order_acquire);
        if (k == nullptr && e.kernel.compare_exchange_strong(k, kernel)) k = kernel;
        if (k != kernel) continue;
        if (const int v = e.bytes_plus_one.load(std::memory_order_acquire)) return v - 1;
        free_entry = &e;
    }
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess) return -1;
    if (free_entry) free_entry->bytes_plus_one.store((int)a.sharedSizeBytes + 1, std::memory_order_release);
    return (int)a.sharedSizeBytes;
}

int opt_in_smem(const void *kernel, size_t bytes, const char *what) {
    const int own = own_smem(kernel);
    if (own < 0) return check_launch(what);
    const size_t limit = 227 * 1024 - (size_t)own;
    if (bytes > limit) {
        set_error("%s: needs %zu bytes of shared memory per block, above the limit of %zu", what, bytes, limit);
        return QMLB_ERR_UNSUPPORTED;
    }
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)limit);
    if (e != cudaSuccess) {
        set_error("%s: cudaFuncSetAttribute(%zu): %s", what, limit, cudaGetErrorString(e));
        return QMLB_ERR_CUDA;
    }
    return QMLB_OK;
}

}  // namespace qmlb

extern "C" const char *qmlb_last_error(void) { return qmlb::g_error; }

extern "C" int qmlb_version(void) { return 100; }
