// Matrix products over ragged groups of rows, one matrix per group:
//
//   forward          y[r, :]  = x[r, :] W[g]         rows r of group g: group_start[g] <= r < group_start[g + 1]
//   transposed       dx[r, :] = dy[r, :] W[g]^T      (gradient of the rows)
//   weight gradient  dW[g]    = x_g^T dy_g           (sum over the rows of the group; zero for an empty group)
//
// Rows in front of the first and behind the last group give zero rows.  The group bounds live on the device and are
// clamped to [0, n], so the host never waits for them and no value of theirs leads outside the tensors.
// This file: the entry points, and FFMA kernels for few rows (any size, alignment and element type), where a product is bound by
// reading the matrices and by latency; everything else goes to the tensor cores (grouped_tc.cu, grouped_wgrad_tc.cu for 16-bit
// rows, grouped_pair_tc.cu for float32).
#include "grouped_tc.cuh"
#include "typed.cuh"

namespace {

constexpr int BM = 64, BN = 64, BK = 16, PAD = 4;      // tile of the gradient kernel
constexpr int MAX_GROUPS = 1024;

__device__ __forceinline__ int clamped(const int *start, int g, int n) { return min(max(start[g], 0), n); }

// Few rows: a block takes 32 columns of one group's result.  Lanes are columns, the warps split the depth, and every thread
// keeps ROWS sums, so a matrix is read once per ROWS rows, in whole lines; the warps' sums meet in shared memory.  A transposed
// matrix passes through a padded tile per warp.  What counts is latency: all loads of a stretch of the depth, rows and matrix,
// are in flight before the first is used (addresses are clamped instead of tested).
constexpr int ROWS = 8;
template <typename T, bool TRANS>
__global__ void __launch_bounds__(TRANS ? 256 : 512, TRANS ? 4 : 2)
few_rows_kernel(const T *__restrict__ x, const T *__restrict__ W, const int *__restrict__ start, int G, int n, int K, int N, int w_cols,
                T *__restrict__ y) {
    constexpr int WARPS = TRANS ? 8 : 16, THREADS = WARPS * 32, DEPTH = WARPS * 32, PER = 32;      // each warp: 32 of the depth
    __shared__ __align__(16) float xs[DEPTH][ROWS];
    __shared__ float turn[TRANS ? WARPS : 1][32][TRANS ? 33 : 1];
    float(*sums)[ROWS][32] = reinterpret_cast<float(*)[ROWS][32]>(&xs[0][0]);      // [WARPS][ROWS][32], once the depth is through
    static_assert(WARPS * 32 <= DEPTH, "the sums fit over the rows");
    const int g = blockIdx.y, col0 = blockIdx.x * 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = col0 + lane;
    const int s = clamped(start, g, n), e = clamped(start, g + 1, n);
    if (g == 0 && blockIdx.z == 0) {                       // zero rows outside the groups
        const int first = clamped(start, 0, n), last = max(clamped(start, G, n), first);
        for (int r = warp; r < n; r += WARPS)
            if ((r < first || r >= last) && c < N) y[(size_t)r * N + c] = qmlb::from_f32<T>(0.f);
    }
    const T *Wg = W + (size_t)g * K * N;
    for (int r0 = s + blockIdx.z * ROWS; r0 < e; r0 += gridDim.z * ROWS) {
        float acc[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) acc[i] = 0.f;
        for (int k0 = 0; k0 < K; k0 += DEPTH) {
            const int ka = k0 + warp * PER, m = min(PER, K - ka);              // this warp's part of the depth (m may be negative)
            T w[PER];
            if (!TRANS) {
#pragma unroll
                for (int i = 0; i < PER; ++i) w[i] = Wg[(size_t)min(ka + i, K - 1) * w_cols + min(c, N - 1)];
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) w[i] = Wg[(size_t)min(col0 + i, N - 1) * w_cols + min(ka + lane, K - 1)];
            }
            T v[ROWS * DEPTH / THREADS];                                       // one k per thread, ROWS rows
#pragma unroll
            for (int i = 0; i < ROWS; ++i) v[i] = x[(size_t)min(r0 + i, e - 1) * K + min(k0 + (int)threadIdx.x, K - 1)];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ROWS; ++i) xs[threadIdx.x][i] = k0 + (int)threadIdx.x < K ? qmlb::to_f32(v[i]) : 0.f;
            if (TRANS) {
#pragma unroll
                for (int i = 0; i < PER; ++i) turn[warp][i][lane] = qmlb::to_f32(w[i]);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float u = i < m ? (TRANS ? turn[warp][lane][i] : qmlb::to_f32(w[i])) : 0.f;      // behind the depth both are zero
                const float4 a = *reinterpret_cast<const float4 *>(&xs[warp * PER + i][0]), b = *reinterpret_cast<const float4 *>(&xs[warp * PER + i][4]);
                acc[0] = fmaf(a.x, u, acc[0]); acc[1] = fmaf(a.y, u, acc[1]); acc[2] = fmaf(a.z, u, acc[2]); acc[3] = fmaf(a.w, u, acc[3]);
                acc[4] = fmaf(b.x, u, acc[4]); acc[5] = fmaf(b.y, u, acc[5]); acc[6] = fmaf(b.z, u, acc[6]); acc[7] = fmaf(b.w, u, acc[7]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ROWS; ++i) sums[warp][i][lane] = acc[i];
        __syncthreads();
        if (warp < ROWS) {                                   // one row per warp
            float t = 0.f;
#pragma unroll
            for (int q = 0; q < WARPS; ++q) t += sums[q][warp][lane];
            if (r0 + warp < e && c < N) y[(size_t)(r0 + warp) * N + c] = qmlb::from_f32<T>(t);
        }
        __syncthreads();
    }
}

// block = (64 x 64 tile of dW[g], g); sums over the rows of the group
template <typename T>
__global__ void __launch_bounds__(256)
wgrad_kernel(const T *__restrict__ x, const T *__restrict__ dy, const int *__restrict__ start, int n, int K, int N, T *__restrict__ dW) {
    __shared__ __align__(16) float As[BK][BM + PAD];
    __shared__ __align__(16) float Bs[BK][BN + PAD];
    const int g = blockIdx.z, k0 = blockIdx.x * BM, c0 = blockIdx.y * BN;
    const int s = clamped(start, g, n), e = max(clamped(start, g + 1, n), s);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int lr = tid >> 4, lc = (tid & 15) * 4;
    float acc[4][4] = {};
    for (int r0 = s; r0 < e; r0 += BK) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool in = r0 + lr < e;
            As[lr][lc + q] = (in && k0 + lc + q < K) ? qmlb::to_f32(x[(size_t)(r0 + lr) * K + k0 + lc + q]) : 0.f;
            Bs[lr][lc + q] = (in && c0 + lc + q < N) ? qmlb::to_f32(dy[(size_t)(r0 + lr) * N + c0 + lc + q]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < BK; ++kk) {
            const float4 a = *reinterpret_cast<const float4 *>(&As[kk][ty * 4]);
            const float4 b = *reinterpret_cast<const float4 *>(&Bs[kk][tx * 4]);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = k0 + ty * 4 + i, c = c0 + tx * 4 + j;
            if (k < K && c < N) dW[((size_t)g * K + k) * N + c] = qmlb::from_f32<T>(acc[i][j]);
        }
}

template <typename T>
int run_few_rows(const void *x, const void *W, const int *start, int G, int n, int K, int N, int transpose, void *y, cudaStream_t st) {
    const int in = transpose ? N : K, out = transpose ? K : N;
    // blocks that share a group's rows: for twice the average group; the rest of a larger group takes turns
    const int turns = (2 * n / G + ROWS - 1) / ROWS, z = turns < 1 ? 1 : turns > 16 ? 16 : turns;
    const dim3 grid((unsigned)((out + 31) / 32), (unsigned)G, (unsigned)z);
    if (transpose)
        few_rows_kernel<T, true><<<grid, 256, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(W), start, G, n, in, out, N, static_cast<T *>(y));
    else
        few_rows_kernel<T, false><<<grid, 512, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(W), start, G, n, in, out, N, static_cast<T *>(y));
    return qmlb::check_launch("qmlb_grouped_matmul");
}

template <typename T>
int run_wgrad(const void *x, const void *dy, const int *start, int G, int n, int K, int N, void *dW, cudaStream_t st) {
    dim3 grid((unsigned)((K + BM - 1) / BM), (unsigned)((N + BN - 1) / BN), (unsigned)G);
    wgrad_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(dy), start, n, K, N, static_cast<T *>(dW));
    return qmlb::check_launch("qmlb_grouped_matmul_wgrad");
}

// Few rows or many.  The FFMA kernel takes a few us and 2 n K N operations at 10 TFLOP/s, the tensor-core path 24 us and 16 bytes per
// matrix element for the images; about equal at n = 9 G + 8e7 / (K N).  (Whole calls, of which the host takes 18 us.  3 groups, 336 x
// 256: 23 against 30 us at n = 512, 28 against 30 at 1,024, 50 against 31 at 2,000, transposed 23 against 23 to 30, 36 against 24 to 30,
// 63 against 24; 32 groups, 1,024 x 1,024: 63 against 114 us at n = 256, 89 against 115 at 512, 154 against 117 at 1,024, transposed 81
// against 111, 114 against 112, 198 against 112; 64 groups, 256 x 512: 32 against 37 at 512, 45 against 38 at 1,024, transposed 30
// against 46, 35 against 46.)  Beyond 2,048 rows a block would walk too many of them.
bool few_rows(size_t n, int G, int K, int N) { return n <= 2048 && (double)n <= 9.0 * G + 8e7 / ((double)K * N); }
// Gradient of the matrices.  float32: 19 against 19 to 24 us at n = 256, 44 against 24 to 30 us at n = 1,024 (3 groups, 336 x 256).  16-bit: 6 to
// 10 against 16 us (which are mostly launches) while the result is small; 57 against 34 us for 32 groups, 1,024 x 1,024.
bool few_rows_grad(size_t n, int G, int K, int N, int dtype) {
    return dtype == QMLB_F32 ? n < 256 : n <= 128 && (double)G * K * N <= 4e6;
}

}  // namespace

extern "C" size_t qmlb_grouped_matmul_workspace_bytes(size_t n, int ngroups, int K, int N, int dtype, int transpose) {
    if (n == 0 || ngroups <= 0 || K <= 0 || N <= 0) return 0;
    if (dtype == QMLB_F32) return few_rows(n, ngroups, K, N) ? 0 : qmlb::grouped_pair_workspace(n, ngroups, K, N, transpose);
    return qmlb::grouped_tc_workspace(n, ngroups, K, N, transpose);
}

extern "C" int qmlb_grouped_matmul(const void *x, const void *W, const int *group_start, int dtype, size_t n, int ngroups, int K, int N,
                                   int transpose, void *out, void *workspace, size_t workspace_bytes, qmlb_stream_t stream) {
    QMLB_REQUIRE(W && group_start && ((x && out) || n == 0), "qmlb_grouped_matmul: null tensor");
    QMLB_REQUIRE(qmlb::dtype_size(dtype) != 0, "qmlb_grouped_matmul: unknown element type %d", dtype);
    QMLB_REQUIRE(ngroups > 0 && ngroups <= MAX_GROUPS, "qmlb_grouped_matmul: 1..%d groups supported", MAX_GROUPS);
    QMLB_REQUIRE(K > 0 && N > 0 && K <= 1 << 20 && N <= 1 << 20, "qmlb_grouped_matmul: bad sizes");
    QMLB_REQUIRE(n < ((size_t)1 << 31) - (1 << 20), "qmlb_grouped_matmul: too many rows");
    if (n == 0) return QMLB_OK;
    cudaStream_t st = qmlb::as_stream(stream);
    if (dtype == QMLB_F32 && few_rows(n, ngroups, K, N)) return run_few_rows<float>(x, W, group_start, ngroups, (int)n, K, N, transpose, out, st);
    QMLB_REQUIRE(workspace && workspace_bytes >= qmlb_grouped_matmul_workspace_bytes(n, ngroups, K, N, dtype, transpose),
                 "qmlb_grouped_matmul: workspace too small");
    QMLB_REQUIRE(((uintptr_t)workspace & 255) == 0, "qmlb_grouped_matmul: workspace must be 256-byte aligned");
    if (dtype == QMLB_F32)
        return qmlb::grouped_pair(static_cast<const float *>(x), static_cast<const float *>(W), group_start, n, ngroups, K, N, transpose,
                                  static_cast<float *>(out), workspace, st);
    return qmlb::grouped_tc(x, W, group_start, dtype, n, ngroups, K, N, transpose, out, workspace, st);
}

extern "C" size_t qmlb_grouped_matmul_wgrad_workspace_bytes(size_t n, int ngroups, int K, int N, int dtype) {
    if (n == 0 || ngroups <= 0 || K <= 0 || N <= 0) return 0;
    if (few_rows_grad(n, ngroups, K, N, dtype)) return 0;
    if (dtype == QMLB_F32) return qmlb::grouped_wgrad_pair_workspace(n, ngroups, K, N);
    return qmlb::grouped_wgrad_tc_workspace(n, ngroups, K, N);
}

extern "C" int qmlb_grouped_matmul_wgrad(const void *x, const void *dy, const int *group_start, int dtype, size_t n, int ngroups, int K, int N,
                                         void *dW, void *workspace, size_t workspace_bytes, qmlb_stream_t stream) {
    QMLB_REQUIRE(dW && group_start && ((x && dy) || n == 0), "qmlb_grouped_matmul_wgrad: null tensor");
    const int es = qmlb::dtype_size(dtype);
    QMLB_REQUIRE(es != 0, "qmlb_grouped_matmul_wgrad: unknown element type %d", dtype);
    QMLB_REQUIRE(ngroups > 0 && ngroups <= MAX_GROUPS, "qmlb_grouped_matmul_wgrad: 1..%d groups supported", MAX_GROUPS);
    QMLB_REQUIRE(K > 0 && N > 0 && K <= 1 << 20 && N <= 1 << 20, "qmlb_grouped_matmul_wgrad: bad sizes");
    QMLB_REQUIRE(n < ((size_t)1 << 31) - (1 << 20), "qmlb_grouped_matmul_wgrad: too many rows");
    cudaStream_t st = qmlb::as_stream(stream);
    if (n == 0) {
        if (cudaMemsetAsync(dW, 0, (size_t)ngroups * K * N * es, st) != cudaSuccess) return qmlb::check_launch("qmlb_grouped_matmul_wgrad(memset)");
        return QMLB_OK;
    }
    if (few_rows_grad(n, ngroups, K, N, dtype)) {
        if (dtype == QMLB_F32) return run_wgrad<float>(x, dy, group_start, ngroups, (int)n, K, N, dW, st);
        if (dtype == QMLB_F16) return run_wgrad<__half>(x, dy, group_start, ngroups, (int)n, K, N, dW, st);
        return run_wgrad<__nv_bfloat16>(x, dy, group_start, ngroups, (int)n, K, N, dW, st);
    }
    QMLB_REQUIRE(workspace && workspace_bytes >= qmlb_grouped_matmul_wgrad_workspace_bytes(n, ngroups, K, N, dtype),
                 "qmlb_grouped_matmul_wgrad: workspace too small");
    QMLB_REQUIRE(((uintptr_t)workspace & 255) == 0, "qmlb_grouped_matmul_wgrad: workspace must be 256-byte aligned");
    if (dtype == QMLB_F32)
        return qmlb::grouped_wgrad_pair(static_cast<const float *>(x), static_cast<const float *>(dy), group_start, n, ngroups, K, N,
                                        static_cast<float *>(dW), workspace, st);
    return qmlb::grouped_wgrad_tc(x, dy, group_start, dtype, n, ngroups, K, N, dW, workspace, st);
}
