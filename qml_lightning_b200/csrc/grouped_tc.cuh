// Tensor-core parts of the grouped products, called by the entry points in grouped_matmul.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace qmlb {

size_t grouped_tc_workspace(int G, int K, int N);
int grouped_tc(const void *x, const void *W, const int *start, int dtype, size_t n, int G, int K, int N, int transpose, void *out,
               void *workspace, cudaStream_t st);
int grouped_tc_timeouts();

size_t grouped_wgrad_tc_workspace(size_t n, int G, int K, int N);
int grouped_wgrad_tc(const void *x, const void *dy, const int *start, int dtype, size_t n, int G, int K, int N, void *dW, void *workspace,
                     cudaStream_t st);
int grouped_wgrad_tc_timeouts();

}  // namespace qmlb
