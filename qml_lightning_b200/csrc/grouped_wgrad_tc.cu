// Gradient of the matrices of a grouped product on the tensor cores (fp16 or bf16 rows, 32-bit sums):
//
//   dW[g] = sum over the rows r of group g of x[r]^T dy[r]
//
// The rows are the depth of the product, so both operands lie in memory with their lines (64 columns of one row) across
// the depth; tcgen05.mma takes them that way and nothing is transposed.  A unit of work is one tile of 128 columns of x by
// NT columns of dy over at most `split` rows of one group.  Groups of one part are finished by their unit; the parts of the
// others go to scratch in 32 bits and a second kernel adds them in order, so the result never depends on scheduling.  Groups
// without rows are filled with zeros by warps 2-3.
// The split is chosen on the host from sizes alone (wgrad_split).  It is at most 16,384 rows, because the tensor core truncates
// when it adds: 1,024 additions are off by 3e-5 on average, far below the half step of the result.
// Roles as in the forward product.  The last slice of a part may hold rows of the next group: the issuing warp overwrites
// the lines up to the next multiple of 16 rows with zeros and leaves the other multiples out.
#include "grouped_rows.cuh"
#include "grouped_tc.cuh"

#include <string.h>

#include <type_traits>

namespace {

using namespace qmlb::tc;

constexpr int BM = 128;
constexpr uint32_t BOX = 8192;                   // 64 rows x 64 columns
constexpr int TMA_WARP = 0, MMA_WARP = 1, EPI_WARP = 4, LOAD_WARP = EPI_WARP + EPI_WARPS, LOAD_WARPS = 8;
constexpr int NTHREADS = LOAD_WARP * 32, NTHREADS_LOADED = NTHREADS + LOAD_WARPS * 32;

__device__ int g_timeouts = 0;

struct Shape {
    int n, G, K, N;
    int split;               // rows per part
    int ktiles, ntiles, NT;
    int stages;
    uint32_t b_boxes;        // boxes per stage of dy
    int x_access, dy_access, out_access;
};

template <typename T, bool LOADED>
__global__ void __launch_bounds__(LOADED ? NTHREADS_LOADED : NTHREADS, 1)
wgrad_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_dy, const T *__restrict__ x,
             const T *__restrict__ dy, const int *__restrict__ start, Shape p, T *__restrict__ dW, float *__restrict__ partial) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_free[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *sp = smem_raw + (sbase - smem_u32(smem_raw));
    const uint32_t stage_bytes = (2 + p.b_boxes) * BOX;
    unsigned char *epi = sp + (size_t)p.stages * stage_bytes;
    Groups gr;
    gr.start = reinterpret_cast<int *>(epi + EPI_BYTES);
    gr.parts = gr.start + p.G + 1;
    gr.split = gr.parts + p.G + 1;
    auto bar = [](const uint64_t &b) { return smem_u32(&b); };
    const bool tma_x = !LOADED || p.x_access == 16, tma_dy = !LOADED || p.dy_access == 16;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar(full[s]), LOADED ? 1 + LOAD_WARPS * 32 : 1);
            mbar_init(bar(empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(acc_full[i]), 1); mbar_init(bar(acc_free[i]), EPI_WARPS); }
        mbar_init(bar(done), 1);
        failed = 0;
        mbar_init_fence();
        if (tma_x) prefetch_map(&map_x);
        if (tma_dy) prefetch_map(&map_dy);
    }
    if (warp == MMA_WARP) tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    fence_before();
    read_groups(gr, start, p.G, p.n, p.split);
    fence_after();
    const uint32_t tmem = tmem_slot;
    const int tiles = p.ktiles * p.ntiles, total = gr.parts[p.G] * tiles;
    const volatile int *gave_up = &failed;
    // unit -> group, rows [r0, r1), first columns of x and dy
    auto locate = [&](int unit, int &g, int &r0, int &r1, int &k0, int &n0) {
        const int part = unit / tiles, tile = unit - part * tiles;
        g = gr.find(p.G, part);
        r0 = gr.start[g] + (part - gr.parts[g]) * p.split;
        r1 = min(r0 + p.split, gr.start[g + 1]);
        k0 = (tile / p.ntiles) * BM;
        n0 = (tile % p.ntiles) * p.NT;
    };

    if (warp == TMA_WARP) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                int g, r0, r1, k0, n0;
                locate(unit, g, r0, r1, k0, n0);
                const int xb = min(2, (p.K - k0 + 63) / 64), db = min((p.NT + 63) / 64, (p.N - n0 + 63) / 64);
                const uint32_t bytes = (uint32_t)((tma_x ? xb : 0) + (tma_dy ? db : 0)) * BOX;
                for (int r = r0; r < r1; r += BK, ++it) {
                    const int s = it % p.stages;
                    if (!mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up)) { ok = false; break; }
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes, b = a + 2 * BOX;
                    if (bytes) mbar_expect_tx(bar(full[s]), bytes);
                    else mbar_arrive(bar(full[s]));
                    if (tma_x)
                        for (int j = 0; j < xb; ++j) tma_2d(a + (uint32_t)j * BOX, &map_x, k0 + j * 64, r, bar(full[s]));
                    if (tma_dy)
                        for (int j = 0; j < db; ++j) tma_2d(b + (uint32_t)j * BOX, &map_dy, n0 + j * 64, r, bar(full[s]));
                }
            }
            if (!ok) failed = 1;
            for (int i = max(0, it - p.stages); i < it; ++i)          // no copy may be in flight when the block leaves
                for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(full[i % p.stages]), (uint32_t)(i / p.stages) & 1u); ++tries) {}
        }
    } else if (warp == MMA_WARP) {
        const uint32_t idesc = instr_desc(std::is_same<T, __nv_bfloat16>::value, true, true, BM, p.NT);
        int it = 0, j = 0;
        bool ok = true;
        for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x, ++j) {
            int g, r0, r1, k0, n0;
            locate(unit, g, r0, r1, k0, n0);
            const int buf = j & 1;
            bool w = mbar_wait(bar(acc_free[buf]), ((uint32_t)(j >> 1) & 1u) ^ 1u, gave_up);
            for (int r = r0; r < r1; r += BK, ++it) {
                const int s = it % p.stages;
                w = w && mbar_wait(bar(full[s]), (uint32_t)(it / p.stages) & 1u, gave_up, it ? WAIT_LIMIT : QMLB_TEST_FIRST_WAIT_POLLS);
                if (!__all_sync(QMLB_FULL_MASK, w)) { ok = false; break; }
                const uint32_t a = sbase + (uint32_t)s * stage_bytes;
                const int valid = min(BK, r1 - r), steps = (valid + 15) >> 4;
                if (valid & 15) {                                     // lines that belong to no row of this part
                    unsigned char *st = sp + (size_t)s * stage_bytes;
                    const int per_box = (steps * 16 - valid) * 8;
                    for (int i = lane; i < per_box * (int)(2 + p.b_boxes); i += 32)
                        *reinterpret_cast<uint4 *>(st + (size_t)(i / per_box) * BOX + (size_t)valid * 128 + (i % per_box) * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_smem();
                    __syncwarp();
                }
                if (LOADED) fence_async_smem();                       // copies and stores of the loading threads, as seen through the barrier
                fence_after();
                const uint32_t al = desc_lo(a, BOX), bl = desc_lo(a + 2 * BOX, BOX), d = tmem + (uint32_t)buf * BUF_COLS;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        if (k >= steps) break;
                        mma_f16(d, al + k * 128u, DESC_HI_SW128, bl + k * 128u, DESC_HI_SW128, idesc, (r > r0 || k) ? 1u : 0u);
                    }
                    mma_commit(bar(empty[s]));
                    if (r + BK >= r1) mma_commit(bar(acc_full[buf]));
                }
                __syncwarp();
            }
        }
        if (!ok) failed = 1;
        if (lane == 0) mma_commit(bar(done));
        __syncwarp();
        for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(done), 0u); ++tries) {}
    } else if (warp < EPI_WARP) {
        zero_empty_groups(gr, p.G, reinterpret_cast<unsigned char *>(dW), (size_t)p.K * p.N * 2, p.out_access, blockIdx.x * 2 + warp - 2, gridDim.x * 2, lane);
    } else if (warp < LOAD_WARP) {
        // warps w and w + 4 share a quarter of the rows and take every other 32 columns
        const int quarter = warp & 3, c_first = ((warp - EPI_WARP) >> 2) * 32;
        unsigned char *mine = epi + (warp - EPI_WARP) * EPI_TILE;
        int j = 0;
        bool ok = true;
        for (int unit = blockIdx.x; unit < total; unit += gridDim.x, ++j) {
            int g, r0, r1, k0, n0;
            locate(unit, g, r0, r1, k0, n0);
            const int buf = j & 1;
            const size_t slot = (size_t)(gr.split[g] + unit / tiles - gr.parts[g]);      // of a part of a sum
            const bool whole = gr.parts[g + 1] - gr.parts[g] == 1;
            const int row = k0 + quarter * 32, rows = min(32, p.K - row);
            ok = ok && mbar_wait(bar(acc_full[buf]), (uint32_t)(j >> 1) & 1u, gave_up);
            ok = __all_sync(QMLB_FULL_MASK, ok);
            if (!ok) failed = 1;
            fence_after();
            const uint32_t from = tmem + (uint32_t)buf * BUF_COLS + ((uint32_t)(quarter * 32) << 16);
            if (ok && c_first >= p.NT) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(acc_free[buf]));
            }
            for (int c = c_first; c < p.NT; c += 64) {
                uint32_t v[32];
                const int left = min(p.NT - c, p.N - n0 - c);
                if (ok) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (u * 16 < left) tmem_ld16(from + (uint32_t)(c + u * 16), v + u * 16);
                    tmem_ld_wait();
                    if (c + 64 >= p.NT) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(acc_free[buf]));
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < 32; ++u) v[u] = 0x7fc00000u;
                }
                if (left <= 0) continue;
                if (whole) {
                    stage_row<T>(mine, lane, v);
                    __syncwarp();
                    const size_t row_bytes = (size_t)p.N * 2;
                    unsigned char *to = reinterpret_cast<unsigned char *>(dW) + ((size_t)g * p.K + row) * row_bytes + (size_t)(n0 + c) * 2;
                    store_tile(mine, to, row_bytes, rows, min(32, left) * 2, lane, p.out_access);
                    __syncwarp();
                } else {
                    // part of a sum: 32 bits, [slot][K][ntiles * NT]
                    const size_t row_bytes = (size_t)p.ntiles * p.NT * 4;
                    unsigned char *to = reinterpret_cast<unsigned char *>(partial) + (slot * p.K + row) * row_bytes + (size_t)(n0 + c) * 4;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        stage_row_f32(mine, lane, v + h * 16);
                        __syncwarp();
                        // columns up to the tile's padding are written: the tile has room for them
                        const int cols = min(16, p.NT - c - h * 16);
                        if (cols > 0) store_rows<16>(mine, to + h * 64, row_bytes, rows, cols * 4, lane);
                        __syncwarp();
                    }
                }
            }
        }
    } else if (LOADED) {
        const int t = tid - LOAD_WARP * 32;
        const unsigned char *xs = reinterpret_cast<const unsigned char *>(x), *ds = reinterpret_cast<const unsigned char *>(dy);
        int it = 0;
        bool ok = true;
        for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
            int g, r0, r1, k0, n0;
            locate(unit, g, r0, r1, k0, n0);
            const int xb = min(2, (p.K - k0 + 63) / 64), db = min((p.NT + 63) / 64, (p.N - n0 + 63) / 64);
            for (int r = r0; r < r1; r += BK, ++it) {
                const int s = it % p.stages;
                ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up));
                if (!ok) break;
                const uint32_t a = sbase + (uint32_t)s * stage_bytes, b = a + 2 * BOX;
                if (!tma_x)
                    for (int q = 0; q < xb; ++q)
                        load_box<BK, LOAD_WARPS * 32>(xs, (size_t)p.K * 2, r, r1, (size_t)(k0 + q * 64) * 2, a + (uint32_t)q * BOX, t, p.x_access);
                if (!tma_dy)
                    for (int q = 0; q < db; ++q)
                        load_box<BK, LOAD_WARPS * 32>(ds, (size_t)p.N * 2, r, r1, (size_t)(n0 + q * 64) * 2, b + (uint32_t)q * BOX, t, p.dy_access);
                if (min(p.x_access, p.dy_access) >= 4) {
                    cp_async_arrive(bar(full[s]));              // when this thread's copies have landed
                } else {                                        // plain stores among them
                    cp_async_wait_all();
                    mbar_arrive(bar(full[s]));
                }
            }
        }
        cp_async_wait_all();                                     // no copy may be in flight when the block leaves
        if (!ok) failed = 1;
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (tid == 0 && failed) atomicAdd(&g_timeouts, 1);
    if (warp == MMA_WARP) tmem_free(tmem, TMEM_COLS);
}

// Groups of several parts: their sum, in order.  blockIdx.y takes the y-th of them (there are at most n / split); `row` is the
// row length of the parts.  VEC columns per thread: four, or one where that leaves too few threads to hide the latency.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
join_kernel(const int *__restrict__ start, const float *__restrict__ partial, int n, int G, int K, int N, int split, size_t row, T *__restrict__ dW) {
    extern __shared__ int sm[];
    __shared__ int which;
    Groups gr;
    gr.start = sm;
    gr.parts = sm + G + 1;
    gr.split = gr.parts + G + 1;
    read_groups(gr, start, G, n, split);
    if (threadIdx.x < 32) {
        int left = (int)blockIdx.y, found = -1;
        for (int g0 = 0; g0 < G && found < 0; g0 += 32) {
            const int g = g0 + (int)threadIdx.x;
            const unsigned m = __ballot_sync(QMLB_FULL_MASK, g < G && gr.parts[g + 1] - gr.parts[g] > 1);
            if (left < __popc(m)) found = g0 + (int)__fns(m, 0, left + 1);
            left -= __popc(m);
        }
        if (threadIdx.x == 0) which = found;
    }
    __syncthreads();
    const int g = which;
    if (g < 0) return;
    const int parts = gr.parts[g + 1] - gr.parts[g];
    const unsigned per_row = ((unsigned)N + VEC - 1u) / VEC;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)K * per_row; i += (size_t)gridDim.x * 256) {
        const unsigned k = (unsigned)(i / per_row), c = (unsigned)(i - (size_t)k * per_row) * VEC;
        const float *src = partial + ((size_t)gr.split[g] * K + k) * row + c;
        float s[VEC], v[8][VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = 0.f;
        for (int q = 0; q < parts; q += 8) {                     // addresses are clamped instead of tested: eight loads in flight
#pragma unroll
            for (int u = 0; u < 8; ++u) qmlb::load_f32<float, VEC>(src + (size_t)min(q + u, parts - 1) * K * row, v[u]);
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] += q + u < parts ? v[u][e] : 0.f;
        }
        T *to = dW + ((size_t)g * K + k) * N + c;
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c + e < (unsigned)N) to[e] = qmlb::from_f32<T>(s[e]);
    }
}

template <typename T>
int join(T *dW, const int *start, size_t n, int G, int K, int N, int split, size_t row, const float *partial, cudaStream_t st) {
    const size_t several = n / split < (size_t)G ? n / split : (size_t)G;       // groups of several parts, at most
    if (several == 0 || n == (size_t)split) return qmlb::check_launch("qmlb_grouped_matmul_wgrad");
    // Four values a thread once they fill the SMs (784 x 256, 5 groups of 330,000 rows: 203 us against 209 us for the whole call;
    // 18 groups of 240 x 1080: 174 against 201; 240 x 228: 26 against 24).  16 blocks an SM over the groups (8 groups of 2,048 x 2,048:
    // 620 us, with 8 blocks 636 us).
    const bool small = (size_t)K * N < (size_t)148 * 512;
    const size_t per = ((size_t)K * (small ? N : (N + 3) / 4) + 255) / 256, most = (148 * 16 + several - 1) / several;
    const dim3 grid((unsigned)(per < most ? per : most), (unsigned)several);
    const size_t smem = (size_t)3 * (G + 1) * 4;
    if (small) join_kernel<T, 1><<<grid, 256, smem, st>>>(start, partial, (int)n, G, K, N, split, row, dW);
    else join_kernel<T, 4><<<grid, 256, smem, st>>>(start, partial, (int)n, G, K, N, split, row, dW);
    return qmlb::check_launch("qmlb_grouped_matmul_wgrad");
}

Shape make_shape(size_t n, int G, int K, int N) {
    Shape p;
    p.n = (int)n;
    p.G = G;
    p.K = K;
    p.N = N;
    const int nt = (N + 255) / 256;
    p.NT = ((N + nt - 1) / nt + 15) / 16 * 16;
    p.ntiles = (N + p.NT - 1) / p.NT;
    p.ktiles = (K + BM - 1) / BM;
    p.b_boxes = (uint32_t)((p.NT + 63) / 64);
    p.split = qmlb::wgrad_split(n, G, p.ktiles, p.ntiles, 1536);
    return p;
}

template <typename T>
int run(const void *x, const void *dy, const int *start, size_t n, int G, int K, int N, void *dW, void *workspace, cudaStream_t st) {
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    Shape p = make_shape(n, G, K, N);
    p.x_access = qmlb::access_bytes((size_t)K * 2, 2, x);
    p.dy_access = qmlb::access_bytes((size_t)N * 2, 2, dy);
    p.out_access = qmlb::access_bytes((size_t)N * 2, 2, dW);
    const uint32_t stage = (2 + p.b_boxes) * BOX;
    const size_t fixed = EPI_BYTES + (size_t)3 * (G + 1) * 4 + 1024;
    p.stages = (int)((SMEM_LIMIT - fixed - 512) / stage);
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    const bool loaded = p.x_access < 16 || p.dy_access < 16;
    CUtensorMap mx, md;
    memset(&mx, 0, sizeof(mx));
    memset(&md, 0, sizeof(md));
    if (p.x_access == 16)
        if (int rc = qmlb::encode_tiles(&mx, x, bf16, (uint64_t)K, (uint64_t)n, 0, (uint64_t)K * 2, BK, "qmlb_grouped_matmul_wgrad")) return rc;
    if (p.dy_access == 16)
        if (int rc = qmlb::encode_tiles(&md, dy, bf16, (uint64_t)N, (uint64_t)n, 0, (uint64_t)N * 2, BK, "qmlb_grouped_matmul_wgrad")) return rc;
    const long units = ((long)(n / p.split) + G) * p.ktiles * p.ntiles;
    const int blocks = (int)(units < 148 ? units : 148);
    const size_t smem = fixed + (size_t)p.stages * stage;
    float *partial = static_cast<float *>(workspace);
    T *out = static_cast<T *>(dW);
    if (loaded) {
        if (int rc = qmlb::ensure_smem(wgrad_kernel<T, true>, smem, "qmlb_grouped_matmul_wgrad")) return rc;
        wgrad_kernel<T, true><<<blocks, NTHREADS_LOADED, smem, st>>>(mx, md, static_cast<const T *>(x), static_cast<const T *>(dy), start, p, out, partial);
    } else {
        if (int rc = qmlb::ensure_smem(wgrad_kernel<T, false>, smem, "qmlb_grouped_matmul_wgrad")) return rc;
        wgrad_kernel<T, false><<<blocks, NTHREADS, smem, st>>>(mx, md, static_cast<const T *>(x), static_cast<const T *>(dy), start, p, out, partial);
    }
    return join<T>(out, start, n, G, K, N, p.split, (size_t)p.ntiles * p.NT, partial, st);
}

}  // namespace

namespace qmlb {

// Rows per part, for the shortest time of 148 SMs that take (n / split + G) * tiles units in turn.  Two bounds of that time, in
// rows: whole rounds of units, and the even share plus one unit.  A unit costs its rows, 256 more for its first loads and its
// store, and `part_cost` more when it is a part of a group and goes through scratch in 32 bits (groups have n / G rows on
// average).  Between 256 and 16,384 rows.
int wgrad_split(size_t n, int G, int ktiles, int ntiles, int part_cost) {
    const double tiles = (double)ktiles * ntiles, sms = 148.0;
    double best = 0.0, least = -1.0;
    for (double s = 256.0; s <= 16384.0; s *= 1.1892071) {          // four steps per doubling
        const double units = ((double)n / s + G) * tiles, rounds = (double)(long)((units + sms - 1) / sms), parts = (double)n / (G * s);
        const double cost = 256.0 + part_cost * (parts < 1.0 ? parts : 1.0);
        const double whole = rounds * (s + cost), share = (n * tiles + units * cost) / sms + s, t = whole < share ? whole : share;
        if (least < 0.0 || t < least) { least = t; best = s; }
    }
    return ((int)best + BK - 1) / BK * BK;
}

// parts of groups of several parts: a group of r > split rows has at most 2 r / split
size_t wgrad_slots(size_t n, int G, int split) {
    const size_t parts = n / split;
    return parts < (size_t)G ? 2 * parts : parts + G;
}

int wgrad_join(void *dW, int dtype, const int *start, size_t n, int G, int K, int N, int split, int row, const float *partial, cudaStream_t st) {
    if (dtype == QMLB_F32) return join<float>(static_cast<float *>(dW), start, n, G, K, N, split, (size_t)row, partial, st);
    if (dtype == QMLB_F16) return join<__half>(static_cast<__half *>(dW), start, n, G, K, N, split, (size_t)row, partial, st);
    return join<__nv_bfloat16>(static_cast<__nv_bfloat16 *>(dW), start, n, G, K, N, split, (size_t)row, partial, st);
}

size_t grouped_wgrad_tc_workspace(size_t n, int G, int K, int N) {
    const Shape p = make_shape(n, G, K, N);
    return wgrad_slots(n, G, p.split) * K * p.ntiles * p.NT * 4 + 256;
}

int grouped_wgrad_tc(const void *x, const void *dy, const int *start, int dtype, size_t n, int G, int K, int N, void *dW, void *workspace,
                     cudaStream_t st) {
    return dtype == QMLB_F16 ? run<__half>(x, dy, start, n, G, K, N, dW, workspace, st) : run<__nv_bfloat16>(x, dy, start, n, G, K, N, dW, workspace, st);
}

int grouped_wgrad_tc_timeouts() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace qmlb
