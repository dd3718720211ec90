// Matrix products over ragged groups of rows, one matrix per group:
//
//   forward          y[r, :]  = x[r, :] W[g]         rows r of group g: group_start[g] <= r < group_start[g + 1]
//   transposed       dx[r, :] = dy[r, :] W[g]^T      (gradient of the rows)
//   weight gradient  dW[g]    = x_g^T dy_g           (sum over the rows of the group; zero for an empty group)
//
// Rows in front of the first and behind the last group give zero rows.  The group bounds live on the device and are
// clamped to [0, n], so the host never waits for them and no value of theirs leads outside the tensors.
// 64 x 64 tiles of FFMA products with 32-bit sums; any size, alignment and element type.
#include "grouped_tc.cuh"
#include "typed.cuh"

namespace {

constexpr int BM = 64, BN = 64, BK = 16, PAD = 4;
constexpr int MAX_GROUPS = 1024;

__device__ __forceinline__ int clamped(const int *start, int g, int n) { return min(max(start[g], 0), n); }

// tile number -> group and rows; false behind the last tile.  All threads of the block take part.
__device__ bool find_tile(const int *__restrict__ start, int G, int n, int tile, int *sh, int &g, int &row0, int &row1) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int before = 0, found = 0;
        for (int g0 = 0; g0 < G && !found; g0 += 32) {
            int s = 0, e = 0;
            if (g0 + lane < G) {
                s = clamped(start, g0 + lane, n);
                e = max(clamped(start, g0 + lane + 1, n), s);
            }
            const int t = (e - s + BM - 1) / BM;
            int inc = t;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(QMLB_FULL_MASK, inc, o);
                if (lane >= o) inc += v;
            }
            const bool here = tile >= before + inc - t && tile < before + inc;
            const unsigned m = __ballot_sync(QMLB_FULL_MASK, here);
            if (here) {
                sh[1] = g0 + lane;
                sh[2] = s + (tile - (before + inc - t)) * BM;
                sh[3] = e;
            }
            found = m != 0;
            before += __shfl_sync(QMLB_FULL_MASK, inc, 31);
        }
        if (lane == 0) sh[0] = found;
    }
    __syncthreads();
    g = sh[1];
    row0 = sh[2];
    row1 = sh[3];
    return sh[0] != 0;
}

template <typename T, bool TRANS>
__global__ void __launch_bounds__(256)
product_kernel(const T *__restrict__ x, const T *__restrict__ W, const int *__restrict__ start, int G, int n, int K, int N, int w_cols,
               T *__restrict__ y) {
    __shared__ __align__(16) float As[BK][BM + PAD];
    __shared__ __align__(16) float Bs[BK][BN + PAD];
    __shared__ int sh[4];
    int g, row0, row1;
    const int col0 = blockIdx.y * BN, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    // zero rows outside the groups: every block takes its share
    {
        const int first = clamped(start, 0, n), last = max(clamped(start, G, n), first);
        for (int r = blockIdx.x * 4 + (tid >> 6); r < n; r += gridDim.x * 4) {
            if (r >= first && r < last) continue;
            const int c = col0 + (tid & 63);
            if (c < N) y[(size_t)r * N + c] = qmlb::from_f32<T>(0.f);
        }
    }
    if (!find_tile(start, G, n, blockIdx.x, sh, g, row0, row1)) return;
    const T *Wg = W + (size_t)g * K * N;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += BK) {
        {
            const int r = tid >> 2, kk = (tid & 3) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                As[kk + q][r] = (row0 + r < row1 && k0 + kk + q < K) ? qmlb::to_f32(x[(size_t)(row0 + r) * K + k0 + kk + q]) : 0.f;
        }
        if (!TRANS) {
            const int k = tid >> 4, c = (tid & 15) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                Bs[k][c + q] = (k0 + k < K && col0 + c + q < N) ? qmlb::to_f32(Wg[(size_t)(k0 + k) * w_cols + col0 + c + q]) : 0.f;
        } else {
            const int c = tid >> 2, kk = (tid & 3) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                Bs[kk + q][c] = (k0 + kk + q < K && col0 + c < N) ? qmlb::to_f32(Wg[(size_t)(col0 + c) * w_cols + k0 + kk + q]) : 0.f;
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
    for (int i = 0; i < 4; ++i) {
        const int r = row0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = col0 + tx * 4 + j;
            if (r < row1 && c < N) y[(size_t)r * N + c] = qmlb::from_f32<T>(acc[i][j]);
        }
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
int run_product(const void *x, const void *W, const int *start, int G, int n, int K, int N, int transpose, void *y, cudaStream_t st) {
    const int in = transpose ? N : K, out = transpose ? K : N;
    // every group adds at most one partly filled tile
    dim3 grid((unsigned)((n + BM - 1) / BM + G), (unsigned)((out + BN - 1) / BN));
    if (transpose)
        product_kernel<T, true><<<grid, 256, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(W), start, G, n, in, out, N, static_cast<T *>(y));
    else
        product_kernel<T, false><<<grid, 256, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(W), start, G, n, in, out, N, static_cast<T *>(y));
    return qmlb::check_launch("qmlb_grouped_matmul");
}

template <typename T>
int run_wgrad(const void *x, const void *dy, const int *start, int G, int n, int K, int N, void *dW, cudaStream_t st) {
    dim3 grid((unsigned)((K + BM - 1) / BM), (unsigned)((N + BN - 1) / BN), (unsigned)G);
    wgrad_kernel<T><<<grid, 256, 0, st>>>(static_cast<const T *>(x), static_cast<const T *>(dy), start, n, K, N, static_cast<T *>(dW));
    return qmlb::check_launch("qmlb_grouped_matmul_wgrad");
}

bool few_rows(size_t n) { return n < 256; }

}  // namespace

extern "C" size_t qmlb_grouped_matmul_workspace_bytes(size_t n, int ngroups, int K, int N, int dtype, int transpose) {
    if (n == 0 || ngroups <= 0 || K <= 0 || N <= 0) return 256;
    if (dtype == QMLB_F32) return few_rows(n) ? 256 : qmlb::grouped_pair_workspace(n, ngroups, K, N, transpose);
    return qmlb::grouped_tc_workspace(ngroups, K, N);
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
    if (dtype == QMLB_F32 && few_rows(n)) return run_product<float>(x, W, group_start, ngroups, (int)n, K, N, transpose, out, st);
    QMLB_REQUIRE(workspace && workspace_bytes >= qmlb_grouped_matmul_workspace_bytes(n, ngroups, K, N, dtype, transpose),
                 "qmlb_grouped_matmul: workspace too small");
    QMLB_REQUIRE(((uintptr_t)workspace & 255) == 0, "qmlb_grouped_matmul: workspace must be 256-byte aligned");
    if (dtype == QMLB_F32)
        return qmlb::grouped_pair(static_cast<const float *>(x), static_cast<const float *>(W), group_start, n, ngroups, K, N, transpose,
                                  static_cast<float *>(out), workspace, st);
    return qmlb::grouped_tc(x, W, group_start, dtype, n, ngroups, K, N, transpose, out, workspace, st);
}

extern "C" size_t qmlb_grouped_matmul_wgrad_workspace_bytes(size_t n, int ngroups, int K, int N, int dtype) {
    if (n == 0 || ngroups <= 0 || K <= 0 || N <= 0) return 256;
    if (dtype == QMLB_F32) return few_rows(n) ? 256 : qmlb::grouped_wgrad_pair_workspace(n, ngroups, K, N);
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
    if (dtype == QMLB_F32 && few_rows(n)) return run_wgrad<float>(x, dy, group_start, ngroups, (int)n, K, N, dW, st);
    QMLB_REQUIRE(workspace && workspace_bytes >= qmlb_grouped_matmul_wgrad_workspace_bytes(n, ngroups, K, N, dtype),
                 "qmlb_grouped_matmul_wgrad: workspace too small");
    QMLB_REQUIRE(((uintptr_t)workspace & 255) == 0, "qmlb_grouped_matmul_wgrad: workspace must be 256-byte aligned");
    if (dtype == QMLB_F32)
        return qmlb::grouped_wgrad_pair(static_cast<const float *>(x), static_cast<const float *>(dy), group_start, n, ngroups, K, N,
                                        static_cast<float *>(dW), workspace, st);
    return qmlb::grouped_wgrad_tc(x, dy, group_start, dtype, n, ngroups, K, N, dW, workspace, st);
}
