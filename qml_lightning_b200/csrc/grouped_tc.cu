// Products of ragged groups of rows with one 16-bit matrix each on the tensor cores (fp16 or bf16 operands, 32-bit sums):
//
//   out[r, :] = in[r, :] B_g,   B_g = W[g] (forward) or W[g]^T (gradient of the rows),   rows r of group g
//
// One persistent block per SM walks tiles of 128 rows of one group by NT columns, column tiles fastest so that the row
// tile that neighbours share stays in L2.  Roles: warp 0 fetches 64-deep slices of both operands by TMA into a ring of
// stages, warp 1 issues tcgen05.mma (M = 128, N = NT, K = 16) into one of two tensor-memory accumulators, warps 4-11 drain
// the other one: 32 bits to the result type, through a padded shared-memory tile, out in pieces of 64 bytes.  Warps 2-3
// write the zero rows outside the groups.
// The matrices are read where they are: their rows run along N, which makes them an operand whose lines run along N in the
// forward product and along K in the transposed one; the instruction takes both.  A row tile may reach over the end of its
// group: those rows are read and multiplied (rows do not mix) and not stored.
// Rows whose address is no multiple of 16 bytes (odd widths, offset views) cannot be fetched by TMA one after the other.  Forward:
// every PERIOD-th row (2, 4 or 8) has the same offset from a 16-byte boundary, so a tile takes 128 rows of one offset, by a tensor
// map that starts at the boundary; its sums begin `shift` elements early, against zero rows of the matrix (coordinates in front of
// its first row), and the issuing warp overwrites what the rows bring there; small groups are copied instead.  (780 deep, 330,001 rows: 231 us with cp.async of
// 8 bytes, 177 us so; 781 deep: 664 us with 2-byte loads, 181 us so.)  Transposed, the matrix's lines would have to move along, so
// warps 12-19 bring the rows with cp.async of 8 or 4 bytes, or 2-byte loads, into the same swizzled stages.
// Sums longer than 16,384 values are cut, because the tensor core truncates when it adds (1,024 additions of one sign are off by up to
// 1e-4 of their sum): every piece fills an accumulator of its own, and the draining warps add them in 32 bits in a place of the
// workspace that only they use.
// Every wait is bounded; a block that gives up fills its remaining tiles with NaN and counts the event (qmlb_tc_timeouts).
#include "grouped_tc.cuh"
#include "grouped_rows.cuh"

#include <string.h>

#include <type_traits>

namespace {

using namespace qmlb::tc;

constexpr int BM = 128;                          // rows per tile
constexpr uint32_t A_BYTES = BM * BK * 2;
// Pairs of blocks fetch half of the matrix each, which pays when the sums are deep and the groups fill tiles of 256 rows.  Measured
// (bf16): 65,536 rows of 8 groups, 2,048 x 2,048: 508 -> 474 us, transposed 443 -> 395; 210,000 rows, 1,024 deep, 256 columns: 126 ->
// 116; but 256 deep, 784 columns (330,000 rows): 193 -> 238, and 336 deep, 256 columns (210,000 rows): 62 -> 70.
constexpr int PAIR_DEPTH = 768;
constexpr size_t PAIR_ROWS = 512;                // rows per group, on average
constexpr int PIECE = 256;                       // chunks of 64 values that one accumulator sums up
constexpr int SUMS = BM * 256;                   // 32-bit sums of one block
constexpr int MAX_BLOCKS = 148;
constexpr int TMA_WARP = 0, MMA_WARP = 1, EPI_WARP = 4, LOAD_WARP = EPI_WARP + EPI_WARPS, LOAD_WARPS = 8;
constexpr int NTHREADS = LOAD_WARP * 32, NTHREADS_LOADED = NTHREADS + LOAD_WARPS * 32;

__device__ int g_timeouts = 0;

struct Shape {
    int n, G, K, out;        // rows, groups, depth of the sums, columns of the result
    int NT, ntiles;          // columns per tile, column tiles
    int nchunks, stages;
    uint32_t b_bytes;        // one stage of the matrix operand
    int in_access;           // widest access that can follow the rows of `in` (16: TMA), in bytes
    int out_access;
    int period;              // rows that lie at the same offset from a 16-byte boundary: every period-th
    int shift[8];            // that offset, in elements
    float *sums;             // [blocks][SUMS], where a sum has several pieces
};

struct RowMaps { CUtensorMap map[8]; };          // one per offset

// DEEP: sums of several pieces, a variant of its own (210,000 rows of 256, transposed to 336 bf16: 67 us, by this variant 72 us)
template <typename T, bool TRANS, bool LOADED, bool PAIR, bool SHIFTED, bool DEEP>
__global__ void __launch_bounds__(LOADED ? NTHREADS_LOADED : NTHREADS, 1)
grouped_kernel(const __grid_constant__ RowMaps maps, const __grid_constant__ CUtensorMap map_w, const T *__restrict__ in,
               const int *__restrict__ start, Shape p, T *__restrict__ out) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_free[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *sp = smem_raw + (sbase - smem_u32(smem_raw));
    const uint32_t stage_bytes = A_BYTES + p.b_bytes;
    unsigned char *epi = sp + (size_t)p.stages * stage_bytes;
    Groups gr;
    gr.start = reinterpret_cast<int *>(epi + EPI_BYTES);
    gr.parts = gr.start + p.G + 1;
    gr.split = nullptr;
    auto bar = [](const uint64_t &b) { return smem_u32(&b); };
    static_assert(LOADED + PAIR + SHIFTED <= 1 && !(SHIFTED && TRANS) && !(LOADED && !TRANS), "one way to fetch rows");
    const int period = SHIFTED ? p.period : 1;
    constexpr int BLOCKS = PAIR ? 2 : 1, TILE_ROWS = BM * BLOCKS;
    const uint32_t rank = PAIR ? cluster_rank() : 0;            // the even block of a pair issues
    const int unit0 = blockIdx.x / BLOCKS, units = gridDim.x / BLOCKS;

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar(full[s]), LOADED ? 1 + LOAD_WARPS * 32 : 1);        // the TMA issuer, and the loading threads
            mbar_init(bar(empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(acc_full[i]), 1); mbar_init(bar(acc_free[i]), EPI_WARPS * BLOCKS); }
        mbar_init(bar(done), 1);
        failed = 0;
        mbar_init_fence();
        if (!LOADED) prefetch_map(&maps.map[0]);
        prefetch_map(&map_w);
    }
    if (warp == MMA_WARP) {
        if (PAIR) tmem_alloc_pair(smem_u32(&tmem_slot), TMEM_COLS);
        else tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    }
    fence_before();
    read_groups(gr, start, p.G, p.n, TILE_ROWS * period);
    if (PAIR) cluster_sync();                                   // both blocks' barriers are ready
    fence_after();
    const uint32_t tmem = tmem_slot;
    const int total = gr.parts[p.G] * p.ntiles * period;
    // tile -> group, first row of this block (the others follow in steps of `period`), end of the group, column tile
    auto locate = [&](int tile, int &g, int &row0, int &row1, int &col0) {
        const int mt = tile / p.ntiles, part = mt / period;
        col0 = (tile - mt * p.ntiles) * p.NT;
        g = gr.find(p.G, part);
        row0 = gr.start[g] + ((part - gr.parts[g]) * TILE_ROWS + (int)rank * BM) * period + (mt - part * period);
        row1 = gr.start[g + 1];
    };
    auto shift_of = [&](int row) { return SHIFTED ? p.shift[row % period] : 0; };
    auto chunks_of = [&](int row) { return SHIFTED ? (p.K + shift_of(row) + BK - 1) / BK : p.nchunks; };
    const volatile int *gave_up = &failed;

    if (warp == TMA_WARP) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int tile = unit0; tile < total && ok; tile += units) {
                int g, row0, row1, col0;
                locate(tile, g, row0, row1, col0);
                // Forward: boxes of 64 columns by 64 deep, as many as reach into the matrix; transposed: one box of the block's rows.
                // The even block of a pair expects what both fetch.
                const int own = p.NT / BLOCKS, bcol = col0 + (int)rank * own;
                auto boxes_at = [&](int col) { return TRANS ? 1 : max(0, min((own + 63) / 64, (p.out - col + 63) / 64)); };
                auto bytes_at = [&](int col) { return (LOADED ? 0u : A_BYTES) + (TRANS ? p.b_bytes : (uint32_t)boxes_at(col) * 8192u); };
                const int boxes = boxes_at(bcol);
                const uint32_t bytes = bytes_at(col0) + (PAIR ? bytes_at(col0 + own) : 0u);
                const int chunks = chunks_of(row0), shift = shift_of(row0);
                const CUtensorMap *rows_map = &maps.map[SHIFTED ? row0 % period : 0];
                for (int c = 0; c < chunks; ++c, ++it) {
                    const int s = it % p.stages;
                    if (!mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up)) { ok = false; break; }
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes, b = a + A_BYTES;
                    if (rank == 0) mbar_expect_tx(bar(full[s]), bytes);
                    if (PAIR) {
                        const uint32_t to = map_rank(bar(full[s]), 0);
                        tma_2d_pair(a, rows_map, c * BK, row0, to);
                        if (TRANS) tma_3d_pair(b, &map_w, c * BK, bcol, g, to);
                        else
                            for (int j = 0; j < boxes; ++j) tma_3d_pair(b + (uint32_t)j * 8192u, &map_w, bcol + j * 64, c * BK, g, to);
                    } else {
                        if (!LOADED) tma_2d(a, rows_map, c * BK, row0 / period, bar(full[s]));
                        if (TRANS) tma_3d(b, &map_w, c * BK, bcol, g, bar(full[s]));
                        else
                            for (int j = 0; j < boxes; ++j) tma_3d(b + (uint32_t)j * 8192u, &map_w, bcol + j * 64, c * BK - shift, g, bar(full[s]));
                    }
                }
            }
            if (!ok) failed = 1;
            // no copy may be in flight when the block leaves
            for (int i = max(0, it - p.stages); i < it && rank == 0; ++i)
                for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(full[i % p.stages]), (uint32_t)(i / p.stages) & 1u); ++tries) {}
        }
    } else if (warp == MMA_WARP && rank != 0) {
        // the even block issues for both
    } else if (warp == MMA_WARP) {
        const uint32_t idesc = instr_desc(std::is_same<T, __nv_bfloat16>::value, false, !TRANS, TILE_ROWS, p.NT);
        int it = 0, j = 0;
        bool ok = true;
        for (int tile = unit0; tile < total && ok; tile += units) {
            int chunks = p.nchunks, shift = 0;
            if (SHIFTED) {
                int g, row0, row1, col0;
                locate(tile, g, row0, row1, col0);
                chunks = chunks_of(row0);
                shift = shift_of(row0);
            }
            for (int first = 0; first < chunks && ok; first += DEEP ? PIECE : chunks, ++j) {
                const int buf = j & 1, end = DEEP ? min(first + PIECE, chunks) : chunks;
                bool w = mbar_wait(bar(acc_free[buf]), ((uint32_t)(j >> 1) & 1u) ^ 1u, gave_up);
                for (int c = first; c < end; ++c, ++it) {
                    const int s = it % p.stages;
                    w = w && mbar_wait(bar(full[s]), (uint32_t)(it / p.stages) & 1u, gave_up, it ? WAIT_LIMIT : QMLB_TEST_FIRST_WAIT_POLLS);
                    if (!__all_sync(QMLB_FULL_MASK, w)) { ok = false; break; }
                    if (SHIFTED && c == 0 && shift) {               // what lies in front of the rows is not theirs
                        unsigned char *rows = sp + (size_t)s * stage_bytes;
                        for (int r = lane; r < BM; r += 32)
                            for (int i = 0; i < shift; ++i) *reinterpret_cast<uint16_t *>(rows + r * 128 + ((r & 7) << 4) + i * 2) = 0;
                        fence_async_smem();
                        __syncwarp();
                    }
                    if (LOADED) fence_async_smem();                 // copies and stores of the loading threads, as seen through the barrier
                    fence_after();
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes, d = tmem + (uint32_t)buf * BUF_COLS;
                    const uint32_t al = desc_lo(a, 16), bl = desc_lo(a + A_BYTES, TRANS ? 16 : 8192);
                    constexpr uint32_t b_step = TRANS ? 2u : 128u;          // 16 deep: 32 bytes along the lines, or 16 lines
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            if (PAIR) mma_f16_pair(d, al + k * 2u, DESC_HI_SW128, bl + k * b_step, DESC_HI_SW128, idesc, (c > first || k) ? 1u : 0u);
                            else mma_f16(d, al + k * 2u, DESC_HI_SW128, bl + k * b_step, DESC_HI_SW128, idesc, (c > first || k) ? 1u : 0u);
                        }
                        if (PAIR) mma_commit_pair(bar(empty[s]));
                        else mma_commit(bar(empty[s]));
                        if (c == end - 1) {
                            if (PAIR) mma_commit_pair(bar(acc_full[buf]));
                            else mma_commit(bar(acc_full[buf]));
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) failed = 1;
        if (lane == 0) {
            if (PAIR) mma_commit_pair(bar(done));
            else mma_commit(bar(done));                         // everything issued has left the tensor pipe
        }
        __syncwarp();
        for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(done), 0u); ++tries) {}
    } else if (warp < EPI_WARP) {
        // zero rows in front of the first group and behind the last
        const int first = gr.start[0], last = max(gr.start[p.G], first);
        const int outside = first + (p.n - last);
        for (int i = blockIdx.x * 2 + (warp - 2); i < outside; i += gridDim.x * 2) {
            T *row = out + (size_t)(i < first ? i : last + (i - first)) * p.out;
            for (int c = lane; c < p.out; c += 32) row[c] = qmlb::from_f32<T>(0.f);
        }
    } else if (warp < LOAD_WARP) {
        // warps w and w + 4 share a quarter of the rows and take every other 32 columns
        const int quarter = warp & 3, c_first = ((warp - EPI_WARP) >> 2) * 32;
        unsigned char *mine = epi + (warp - EPI_WARP) * EPI_TILE;
        const size_t row_bytes = (size_t)p.out * 2, row_step = row_bytes * period;
        auto release = [&](int buf) {                           // to the block that issues
            if (PAIR) mbar_arrive_cluster(map_rank(bar(acc_free[buf]), 0));
            else mbar_arrive(bar(acc_free[buf]));
        };
        // this thread's sums of a column group: [32 columns][32 lanes] per warp and group
        float *kept = p.sums + (size_t)blockIdx.x * SUMS + (size_t)(warp - EPI_WARP) * (SUMS / EPI_WARPS) + lane;
        int j = 0;
        bool ok = true;
        for (int tile = unit0; tile < total; tile += units) {
            int g, row0, row1, col0;
            locate(tile, g, row0, row1, col0);
            const int row = row0 + quarter * 32 * period;
            const int rows = min(32, (row1 - row + period - 1) / period);
            const int pieces = DEEP ? (chunks_of(row0) + PIECE - 1) / PIECE : 1;
            for (int piece = 0; piece < pieces; ++piece, ++j) {
                const int buf = j & 1;
                ok = ok && mbar_wait(bar(acc_full[buf]), (uint32_t)(j >> 1) & 1u, gave_up);
                ok = __all_sync(QMLB_FULL_MASK, ok);
                if (!ok) failed = 1;                            // at once: the other roles stop waiting
                fence_after();
                const uint32_t from = tmem + (uint32_t)buf * BUF_COLS + ((uint32_t)(quarter * 32) << 16);
                if (ok && c_first >= p.NT) {
                    __syncwarp();
                    if (lane == 0) release(buf);
                }
                for (int c = c_first; c < p.NT; c += 64) {
                    uint32_t v[32];
                    const int left = p.NT - c;
                    if (ok) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (u * 16 < left) tmem_ld16(from + (uint32_t)(c + u * 16), v + u * 16);
                        tmem_ld_wait();
                        if (c + 64 >= p.NT) {                   // the accumulator is free once it sits in registers
                            fence_before();
                            __syncwarp();
                            if (lane == 0) release(buf);
                        }
                    } else {
#pragma unroll
                        for (int u = 0; u < 32; ++u) v[u] = 0x7fc00000u;
                    }
                    if (DEEP && pieces > 1) {
                        float *sum = kept + (size_t)(c >> 6) * 1024;
                        if (piece > 0) {
#pragma unroll
                            for (int u = 0; u < 32; ++u) v[u] = __float_as_uint(__uint_as_float(v[u]) + sum[u * 32]);
                        }
                        if (piece < pieces - 1) {
#pragma unroll
                            for (int u = 0; u < 32; ++u) sum[u * 32] = __uint_as_float(v[u]);
                            continue;
                        }
                    }
                    stage_row<T>(mine, lane, v);
                    __syncwarp();
                    const int bytes = min(min(32, left), p.out - col0 - c) * 2;
                    unsigned char *to = reinterpret_cast<unsigned char *>(out) + (size_t)row * row_bytes + (size_t)(col0 + c) * 2;
                    store_tile(mine, to, row_step, rows, bytes, lane, p.out_access);
                    __syncwarp();
                }
            }
        }
    } else if (LOADED) {
        const int t = tid - LOAD_WARP * 32;
        const unsigned char *src = reinterpret_cast<const unsigned char *>(in);
        const size_t row_bytes = (size_t)p.K * 2;
        int it = 0;
        bool ok = true;
        for (int tile = unit0; tile < total && ok; tile += units) {
            int g, row0, row1, col0;
            locate(tile, g, row0, row1, col0);
            for (int c = 0; c < p.nchunks; ++c, ++it) {
                const int s = it % p.stages;
                ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up));
                if (!ok) break;
                const uint32_t a = sbase + (uint32_t)s * stage_bytes;
                load_box<BM, LOAD_WARPS * 32>(src, row_bytes, row0, p.n, (size_t)c * BK * 2, a, t, p.in_access);
                if (p.in_access >= 4) {
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
    if (PAIR) cluster_sync();                                   // neither block leaves while the other's instructions may read it
    if (warp == MMA_WARP) {
        if (PAIR) tmem_free_pair(tmem, TMEM_COLS);
        else tmem_free(tmem, TMEM_COLS);
    }
}

// Rows of `cols` values that no 16-byte access can follow -> the same with rows padded to a multiple of 8 values, 8 per thread
template <typename T>
__global__ void __launch_bounds__(256)
pad_kernel(const T *__restrict__ in, size_t rows, int cols, int padded, T *__restrict__ to) {
    const unsigned words = (unsigned)padded / 8;
    const size_t total = rows * words;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t r = i / words;
        const int c = (int)(i - r * words) * 8;
        const T *src = in + r * cols;
        qmlb::Pack<T, 8> k;
#pragma unroll
        for (int u = 0; u < 8; ++u) k.item[u] = src[min(c + u, cols - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (c + u >= cols) k.item[u] = qmlb::from_f32<T>(0.f);
        reinterpret_cast<uint4 *>(to)[i] = k.word;
    }
}
template <typename T>
void pad_rows(const void *in, size_t rows, int cols, void *to, cudaStream_t st) {
    const int padded = (cols + 7) & ~7;
    const size_t b = (rows * (padded / 8) + 255) / 256;
    pad_kernel<T><<<(unsigned)(b < 148 * 16 ? b : 148 * 16), 256, 0, st>>>(static_cast<const T *>(in), rows, cols, padded, static_cast<T *>(to));
}

// Every offset has tiles of its own in every group, so rows in groups of few rows per offset are copied to the 16-byte boundaries first.
// 64 groups of 781 deep bf16 rows, 256 columns (eight offsets): 20 rows each 99 -> 32 us, 256 63 -> 34, 500 45 -> 49, 1,000 47 -> 83; 2,048
// columns, 16 groups of 500: 72 -> 48; 782 deep (four): 256 rows 40 -> 34, 500 28 -> 48; 780 deep (two): 100 rows 30 -> 26, 256 24 -> 34.
bool copies_rows(size_t n, int G, int depth, int transpose) {
    const int offsets = (depth & 1) ? 8 : (depth & 2) ? 4 : (depth & 4) ? 2 : 1;
    return !transpose && offsets > 1 && n / G <= (size_t)64 * offsets;
}

// a sum may begin up to seven values early
bool several_pieces(int depth) { return (depth + 7 + BK - 1) / BK > PIECE; }
size_t sums_bytes(int depth) { return several_pieces(depth) ? (size_t)MAX_BLOCKS * SUMS * 4 : 0; }
size_t padded_bytes(int G, int K, int N) { return ((size_t)G * K * ((N + 7) & ~7) * 2 + 255) & ~(size_t)255; }

bool needs_pad(const void *W, int N) { return ((uintptr_t)W & 15) != 0 || (N & 7) != 0; }

template <typename T, bool TRANS, bool LOADED, bool PAIR, bool SHIFTED, bool DEEP>
int launch_as(const RowMaps &mi, const CUtensorMap &mw, const T *in, const int *start, const Shape &p, int blocks, T *out, cudaStream_t st) {
    const size_t smem = (size_t)p.stages * (A_BYTES + p.b_bytes) + EPI_BYTES + (size_t)2 * (p.G + 1) * 4 + 1024;
    auto kernel = grouped_kernel<T, TRANS, LOADED, PAIR, SHIFTED, DEEP>;
    if (int rc = qmlb::ensure_smem(kernel, smem, "qmlb_grouped_matmul")) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(LOADED ? NTHREADS_LOADED : NTHREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = PAIR ? 2 : 1;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mi, mw, in, start, p, out);
    if (e != cudaSuccess) {
        qmlb::set_error("qmlb_grouped_matmul: %s", cudaGetErrorString(e));
        return QMLB_ERR_CUDA;
    }
    return qmlb::check_launch("qmlb_grouped_matmul");
}

template <typename T, bool TRANS, bool LOADED, bool PAIR, bool SHIFTED>
int launch(const RowMaps &mi, const CUtensorMap &mw, const T *in, const int *start, const Shape &p, int blocks, T *out, cudaStream_t st) {
    return several_pieces(p.K) ? launch_as<T, TRANS, LOADED, PAIR, SHIFTED, true>(mi, mw, in, start, p, blocks, out, st)
                               : launch_as<T, TRANS, LOADED, PAIR, SHIFTED, false>(mi, mw, in, start, p, blocks, out, st);
}

template <typename T>
int run(const void *x, const void *W, const int *start, size_t n, int G, int K, int N, int transpose, void *out, void *workspace, cudaStream_t st) {
    const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
    Shape p;
    p.n = (int)n;
    p.G = G;
    p.K = transpose ? N : K;
    p.out = transpose ? K : N;
    p.nchunks = (p.K + BK - 1) / BK;
    uint64_t row_bytes = (uint64_t)p.K * 2;
    if (copies_rows(n, G, p.K, transpose)) {
        void *copy = static_cast<unsigned char *>(workspace) + padded_bytes(G, K, N) + sums_bytes(p.K);
        pad_rows<T>(x, n, p.K, copy, st);
        x = copy;
        row_bytes = (uint64_t)((p.K + 7) & ~7) * 2;
    }
    p.in_access = qmlb::access_bytes(row_bytes, 2, x);
    p.out_access = qmlb::access_bytes((size_t)p.out * 2, 2, out);
    // Columns per tile: as many as one accumulator holds, so that the rows are read once, in equal parts; fewer when the row
    // tiles alone do not give every SM a tile.
    const long mtiles = (long)((n + BM - 1) / BM);
    const bool aligned = p.in_access == 16, shifted = !aligned && !transpose, loaded = !aligned && transpose;
    const bool pair = aligned && p.K >= PAIR_DEPTH && n / G >= PAIR_ROWS && mtiles * ((p.out + 255) / 256) >= 2 * 148;
    const int blocks_per_tile = pair ? 2 : 1;
    long nt = (p.out + 255) / 256;
    const long wanted = (148 + mtiles - 1) / mtiles, most = (p.out + 63) / 64;
    if (nt < wanted) nt = wanted < most ? wanted : most;
    const int unit = 16 * blocks_per_tile;                     // each block of a pair holds half of the columns
    p.NT = (int)(((p.out + nt - 1) / nt + unit - 1) / unit * unit);
    p.ntiles = (p.out + p.NT - 1) / p.NT;
    const int own = p.NT / blocks_per_tile;
    p.b_bytes = transpose ? (uint32_t)own * 128u : (uint32_t)((own + 63) / 64) * 8192u;
    p.b_bytes = (p.b_bytes + 1023u) & ~1023u;
    const size_t fixed = EPI_BYTES + (size_t)2 * (G + 1) * 4 + 1024 + 512;
    p.stages = (int)((SMEM_LIMIT - fixed) / (A_BYTES + p.b_bytes));
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;

    const void *Wp = W;
    int Np = N;
    if (needs_pad(W, N)) {
        Np = (N + 7) & ~7;
        pad_rows<T>(W, (size_t)G * K, N, workspace, st);
        Wp = workspace;
    }
    RowMaps mi;
    CUtensorMap mw;
    memset(&mi, 0, sizeof(mi));
    if (int rc = qmlb::encode_tiles(&mw, Wp, bf16, (uint64_t)N, (uint64_t)K, (uint64_t)G, (uint64_t)Np * 2, transpose ? (uint32_t)own : 64u,
                                    "qmlb_grouped_matmul"))
        return rc;
    p.sums = reinterpret_cast<float *>(static_cast<unsigned char *>(workspace) + padded_bytes(G, K, N));
    p.period = 1;
    if (shifted) {
        // a map's rows must not overlap: they begin up to seven elements early (offset views, and depths of 2 and 4)
        while (((row_bytes * p.period) & 15) || p.K + 7 > p.K * p.period) p.period <<= 1;
    }
    for (int q = 0; q < 8; ++q) {
        const uintptr_t at = (uintptr_t)x + q * row_bytes;
        p.shift[q] = (int)(at & 15) / 2;
        if (loaded || q >= p.period) continue;
        if ((uint64_t)q >= n) {                                // no such row: any valid map, nothing of it is stored
            mi.map[q] = mi.map[0];
            continue;
        }
        if (int rc = qmlb::encode_tiles(&mi.map[q], reinterpret_cast<const void *>(at & ~(uintptr_t)15), bf16, (uint64_t)(p.K + p.shift[q]),
                                        (n - q + p.period - 1) / p.period, 0, row_bytes * p.period, BM, "qmlb_grouped_matmul"))
            return rc;
    }
    const long rows_per_tile = (long)BM * blocks_per_tile * p.period;
    const long tiles = ((long)((n + rows_per_tile - 1) / rows_per_tile) + G) * p.period * p.ntiles * blocks_per_tile;
    const int blocks = (int)(tiles < MAX_BLOCKS ? tiles : MAX_BLOCKS);
    const T *xi = static_cast<const T *>(x);
    T *o = static_cast<T *>(out);
    if (loaded) return launch<T, true, true, false, false>(mi, mw, xi, start, p, blocks, o, st);
    if (shifted) return launch<T, false, false, false, true>(mi, mw, xi, start, p, blocks, o, st);
    if (pair)
        return transpose ? launch<T, true, false, true, false>(mi, mw, xi, start, p, blocks, o, st)
                         : launch<T, false, false, true, false>(mi, mw, xi, start, p, blocks, o, st);
    return transpose ? launch<T, true, false, false, false>(mi, mw, xi, start, p, blocks, o, st)
                     : launch<T, false, false, false, false>(mi, mw, xi, start, p, blocks, o, st);
}

}  // namespace

namespace qmlb {

size_t grouped_tc_workspace(size_t n, int G, int K, int N, int transpose) {
    const size_t copy = copies_rows(n, G, K, transpose) ? n * ((K + 7) & ~7) * 2 : 0;
    return padded_bytes(G, K, N) + sums_bytes(transpose ? N : K) + copy + 256;
}

int grouped_tc(const void *x, const void *W, const int *start, int dtype, size_t n, int G, int K, int N, int transpose, void *out,
               void *workspace, cudaStream_t st) {
    return dtype == QMLB_F16 ? run<__half>(x, W, start, n, G, K, N, transpose, out, workspace, st)
                             : run<__nv_bfloat16>(x, W, start, n, G, K, N, transpose, out, workspace, st);
}

int grouped_tc_timeouts() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace qmlb
