// Host side of the TMA tiles of the grouped products: the driver's encoder, looked up once through the runtime.
#include "tcgen.cuh"

#include <atomic>

namespace qmlb {

namespace {
using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                            const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::atomic<Encode> g_encode{nullptr};

Encode encoder() {
    Encode f = g_encode.load(std::memory_order_acquire);
    if (f == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return nullptr;
        f = reinterpret_cast<Encode>(p);
        g_encode.store(f, std::memory_order_release);      // every thread would store the same address
    }
    return f;
}
}  // namespace

int encode_tiles(CUtensorMap *map, const void *base, bool bf16, uint64_t cols, uint64_t rows, uint64_t planes, uint64_t row_bytes,
                 uint32_t box_rows, const char *what) {
    Encode f = encoder();
    if (f == nullptr) {
        set_error("%s: the driver offers no tensor-map encoder", what);
        return QMLB_ERR_CUDA;
    }
    const cuuint64_t dims[3] = {cols, rows, planes}, strides[2] = {row_bytes, row_bytes * rows};
    const cuuint32_t box[3] = {64, box_rows, 1}, step[3] = {1, 1, 1};
    auto encode = [&]() {
        return f(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, planes > 0 ? 3 : 2, const_cast<void *>(base),
                 dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
        // A thread whose first CUDA call this is (a backward pass runs in one): the encoder belongs to the driver, which does not bind
        // the device's context by itself as the runtime's calls do.
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
    }
    if (r != CUDA_SUCCESS) {
        set_error("%s: tensor map refused (code %d, %llu x %llu x %llu)", what, (int)r, (unsigned long long)cols, (unsigned long long)rows,
                  (unsigned long long)planes);
        return QMLB_ERR_CUDA;
    }
    return QMLB_OK;
}

}  // namespace qmlb
