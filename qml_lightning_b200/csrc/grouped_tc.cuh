// Tensor-core parts of the grouped products, called by the entry points in grouped_matmul.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace qmlb {

size_t grouped_tc_workspace(size_t n, int G, int K, int N, int transpose);
int grouped_tc(const void *x, const void *W, const int *start, int dtype, size_t n, int G, int K, int N, int transpose, void *out,
               void *workspace, cudaStream_t st);
int grouped_tc_timeouts();

size_t grouped_wgrad_tc_workspace(size_t n, int G, int K, int N);
int grouped_wgrad_tc(const void *x, const void *dy, const int *start, int dtype, size_t n, int G, int K, int N, void *dW, void *workspace,
                     cudaStream_t st);
int grouped_wgrad_tc_timeouts();

// float32
size_t grouped_pair_workspace(size_t n, int G, int K, int N, int transpose);
int grouped_pair(const float *x, const float *W, const int *start, size_t n, int G, int K, int N, int transpose, float *out, void *workspace,
                 cudaStream_t st);
size_t grouped_wgrad_pair_workspace(size_t n, int G, int K, int N);
int grouped_wgrad_pair(const float *x, const float *dy, const int *start, size_t n, int G, int K, int N, float *dW, void *workspace, cudaStream_t st);
int grouped_pair_timeouts();

// sums over rows in parts: rows per part, parts that go to scratch, and their sum
int wgrad_split(size_t n, int G, int ktiles, int ntiles, int part_cost);
size_t wgrad_slots(size_t n, int G, int split);
int wgrad_join(void *dW, int dtype, const int *start, size_t n, int G, int K, int N, int split, int row, const float *partial, cudaStream_t st);

}  // namespace qmlb
