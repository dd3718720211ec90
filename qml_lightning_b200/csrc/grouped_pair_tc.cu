// Products of ragged groups of rows with one matrix each, float32 operands, on the 16-bit tensor cores.
//
// Arithmetic.  A stretch of 64 values along the depth (of one row or one column of an operand) is scaled by a power of two
// so that its largest lies in [2^14, 2^15), and every scaled value x is split into two fp16 numbers, x ~ h + l:
// h = fp16(x), l = fp16(x - h), off by at most 2^-22 |x| (and 2^-39 of the stretch's largest value, where l would be
// subnormal).  A product is h h' + h l' + l h' (l l' is at most 2^-22 of it), so three 16-bit products give a 32-bit one
// where bf16 parts would need six and tf32 parts three of twice the cost.  Sums: the tensor core truncates when it adds, so
// an accumulator only ever covers one stretch (4 steps: the small cross terms first, then h h'), and warps of CUDA cores add
// the stretches in registers in 32 bits, rounded, undoing both scales on the way.  Against 64 bits the results are off by
// about 2e-7 of their norm, like a float32 product, and rows and columns keep their own magnitudes.
//
// Work split.  One persistent block of 16 warps per SM takes tiles of 128 x NT (NT <= 256) results:
//   warp 0     bulk copies of the matrix operand's images (products of rows; the images are made by a packing kernel)
//   warp 1     issues tcgen05.mma, two tensor-memory accumulators in turn
//   warps 2-3  zero rows outside the groups
//   warps 4-7  load float32 rows, find the scales, split, and write the swizzled operand images to shared memory
//   warps 8-15 add the finished accumulator to their 128 x 32 registers while the next one fills, and store the tile
// Registers are moved from the first eight warps to the last eight (setmaxnreg), which hold 128 sums per thread.
//
// The gradient of the matrices is the same kernel with both operands loaded by warps 4-7: the depth runs over the rows of
// the group, so the operands' lines run across it, and the stretches are 64 rows of one column.
#include <cuda_fp16.h>
#include <string.h>

#include "grouped_rows.cuh"
#include "grouped_tc.cuh"

namespace {

using namespace qmlb::tc;

constexpr int BM = 128;
constexpr uint32_t A_HALF = BM * BK * 2;          // one image (high or low parts) of the 128-wide operand
constexpr int NTHREADS = 512;
constexpr int TMA_WARP = 0, MMA_WARP = 1, LOAD_WARP = 4, FOLD_WARP = 8;
constexpr int MAXST = 4;
constexpr uint32_t SCALE_FLOATS = 128 + 256;      // per chunk: scales of the rows and of the columns of the tile
constexpr uint32_t EPI = 8 * 2048;                // 32 rows x 16 columns per folding warp

__device__ int g_timeouts = 0;

struct Shape {
    int n, G, K, out;        // rows, groups, depth (products of rows) or columns of x (gradient), columns of the result
    int NT, ntiles, ktiles;  // ktiles: tiles of 128 columns of x (gradient)
    int nchunks;             // stretches of the depth (products of rows)
    int split;               // rows per part (gradient)
    int stages;
    uint32_t b_half;         // one image of the NT-wide operand
    int a_access, b_access, out_access;
};

// power of two that takes `m` (bits of the largest magnitude) to [2^14, 2^15), and its inverse; both normal numbers
__device__ __forceinline__ void scales(uint32_t m, float &s, float &inv) {
    const int e = min(max(268 - (int)(m >> 23), 1), 253);
    s = __uint_as_float((uint32_t)e << 23);
    inv = __uint_as_float((uint32_t)(254 - e) << 23);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// N consecutive floats of which `valid` exist
template <int N>
__device__ __forceinline__ void load_floats(const float *src, int valid, int access, float *v) {
    if (valid >= N && access == 16) {
#pragma unroll
        for (int q = 0; q < N; q += 4) {
            const float4 t = *reinterpret_cast<const float4 *>(src + q);
            v[q] = t.x; v[q + 1] = t.y; v[q + 2] = t.z; v[q + 3] = t.w;
        }
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = q < valid ? src[q] : 0.f;
    }
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void sts64(uint32_t at, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(a), "r"(b) : "memory");
}

// Products of rows: a = x [n, K], packed/pack_scales = images of the matrices, result y [n, out].
// GRAD: a = x [n, K], b = dy [n, out], result dW [G, K, out], partial = parts of split groups.
template <bool GRAD>
__global__ void __launch_bounds__(NTHREADS, 1)
pair_kernel(const float *__restrict__ a_in, const float *__restrict__ b_in, const unsigned char *__restrict__ packed,
            const float *__restrict__ pack_scales, const int *__restrict__ start, Shape p, float *__restrict__ out, float *__restrict__ partial) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[MAXST], empty[MAXST], acc_full[2], acc_free[2], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *sp = smem_raw + (sbase - smem_u32(smem_raw));
    const uint32_t stage_bytes = 2 * A_HALF + 2 * p.b_half;
    const int slots = p.stages + 2;               // scales outlive their stage until the accumulator is folded
    float *scale = reinterpret_cast<float *>(sp + (size_t)p.stages * stage_bytes);
    unsigned char *epi = reinterpret_cast<unsigned char *>(scale + (size_t)slots * SCALE_FLOATS);
    Groups gr;
    gr.start = reinterpret_cast<int *>(epi + EPI);
    gr.parts = gr.start + p.G + 1;
    gr.split = GRAD ? gr.parts + p.G + 1 : nullptr;
    auto bar = [](const uint64_t &b) { return smem_u32(&b); };

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar(full[s]), GRAD ? 4 : 5);     // the four loading warps, and the issuer of the bulk copies
            mbar_init(bar(empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(bar(acc_full[i]), 1); mbar_init(bar(acc_free[i]), 8); }
        mbar_init(bar(done), 1);
        failed = 0;
        mbar_init_fence();
    }
    if (warp == MMA_WARP) tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    fence_before();
    read_groups(gr, start, p.G, p.n, GRAD ? p.split : BM);
    fence_after();
    const uint32_t tmem = tmem_slot;
    const int tiles = GRAD ? p.ktiles * p.ntiles : p.ntiles, total = gr.parts[p.G] * tiles;
    const volatile int *gave_up = &failed;
    // unit -> group, part, rows [r0, r1), first column of x (gradient), column tile
    auto locate = [&](int unit, int &g, int &part, int &r0, int &r1, int &k0, int &nt) {
        part = unit / tiles;
        const int tile = unit - part * tiles;
        g = gr.find(p.G, part);
        const int rows = GRAD ? p.split : BM;
        r0 = gr.start[g] + (part - gr.parts[g]) * rows;
        r1 = min(r0 + rows, gr.start[g + 1]);
        nt = GRAD ? tile % p.ntiles : tile;
        k0 = GRAD ? (tile / p.ntiles) * BM : 0;
    };
    auto chunks_of = [&](int r0, int r1) { return GRAD ? (r1 - r0 + BK - 1) / BK : p.nchunks; };

    if (warp < LOAD_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == TMA_WARP) {
            if (!GRAD && lane == 0) {
                int it = 0, slot = 0;
                bool ok = true;
                for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                    int g, part, r0, r1, k0, nt;
                    locate(unit, g, part, r0, r1, k0, nt);
                    const size_t image = (size_t)(g * p.ntiles + nt) * p.nchunks;
                    for (int c = 0; c < p.nchunks; ++c, ++it) {
                        const int s = it % p.stages;
                        if (!mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up)) { ok = false; break; }
                        mbar_expect_tx(bar(full[s]), 2 * p.b_half + (uint32_t)p.NT * 4u);
                        bulk_copy(sbase + (uint32_t)s * stage_bytes + 2 * A_HALF, packed + (image + c) * (2 * p.b_half), 2 * p.b_half, bar(full[s]));
                        bulk_copy(smem_u32(scale + (size_t)slot * SCALE_FLOATS + 128), pack_scales + (image + c) * p.NT, (uint32_t)p.NT * 4u, bar(full[s]));
                        slot = slot + 1 == slots ? 0 : slot + 1;
                    }
                }
                if (!ok) failed = 1;
                for (int i = max(0, it - p.stages); i < it; ++i)          // no copy may be in flight when the block leaves
                    for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(full[i % p.stages]), (uint32_t)(i / p.stages) & 1u); ++tries) {}
            }
        } else if (warp == MMA_WARP) {
            const uint32_t idesc = instr_desc(false, GRAD, GRAD, BM, p.NT);
            constexpr uint32_t step = GRAD ? 128u : 2u, block = GRAD ? 8192u : 16u;
            int it = 0;
            bool ok = true;
            for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                int g, part, r0, r1, k0, nt;
                locate(unit, g, part, r0, r1, k0, nt);
                const int chunks = chunks_of(r0, r1), depth = GRAD ? r1 - r0 : p.K;
                for (int c = 0; c < chunks; ++c, ++it) {
                    const int s = it % p.stages, buf = it & 1;
                    bool w = mbar_wait(bar(acc_free[buf]), ((uint32_t)(it >> 1) & 1u) ^ 1u, gave_up);
                    w = w && mbar_wait(bar(full[s]), (uint32_t)(it / p.stages) & 1u, gave_up);
                    if (!__all_sync(QMLB_FULL_MASK, w)) { ok = false; break; }
                    fence_after();
                    if (lane == 0) {
                        const int steps = min(BK / 16, (depth - c * BK + 15) / 16);
                        const uint32_t a = sbase + (uint32_t)s * stage_bytes, b = a + 2 * A_HALF, d = tmem + (uint32_t)buf * BUF_COLS;
                        const uint32_t ah = desc_lo(a, block), al = desc_lo(a + A_HALF, block), bh = desc_lo(b, block), bl = desc_lo(b + p.b_half, block);
                        for (int k = 0; k < steps; ++k) {
                            mma_f16(d, ah + k * step, DESC_HI_SW128, bl + k * step, DESC_HI_SW128, idesc, k ? 1u : 0u);
                            mma_f16(d, al + k * step, DESC_HI_SW128, bh + k * step, DESC_HI_SW128, idesc, 1u);
                        }
                        for (int k = 0; k < steps; ++k) mma_f16(d, ah + k * step, DESC_HI_SW128, bh + k * step, DESC_HI_SW128, idesc, 1u);
                        mma_commit(bar(empty[s]));
                        mma_commit(bar(acc_full[buf]));
                    }
                    __syncwarp();
                }
            }
            if (!ok) failed = 1;
            if (lane == 0) mma_commit(bar(done));
            __syncwarp();
            for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(done), 0u); ++tries) {}
        } else if (!GRAD) {
            const int first = gr.start[0], last = max(gr.start[p.G], first), outside = first + (p.n - last);
            for (int i = blockIdx.x * 2 + (warp - 2); i < outside; i += gridDim.x * 2) {
                float *row = out + (size_t)(i < first ? i : last + (i - first)) * p.out;
                for (int c = lane; c < p.out; c += 32) row[c] = 0.f;
            }
        }
    } else if (warp < FOLD_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        const int w = warp - LOAD_WARP;
        int it = 0, slot = 0;
        bool ok = true;
        if (!GRAD) {
            // a row is 8 lanes of 8 values; 8 passes of 4 rows per warp
            const int lr = lane >> 3, kc = lane & 7;
            for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                int g, part, r0, r1, k0, nt;
                locate(unit, g, part, r0, r1, k0, nt);
                const int row = r0 + w * 32 + lr;
                for (int c = 0; c < p.nchunks; ++c, ++it) {
                    const int s = it % p.stages, k = c * BK + kc * 8, left = p.K - k;
                    float v[8][8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) load_floats<8>(a_in + (size_t)(row + i * 4) * p.K + k, row + i * 4 < r1 ? left : 0, p.a_access, v[i]);
                    ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up));
                    if (!ok) break;
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t m = 0;
#pragma unroll
                        for (int q = 0; q < 8; ++q) m = max(m, magnitude(v[i][q]));
#pragma unroll
                        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(QMLB_FULL_MASK, m, o));
                        float sc, inv;
                        scales(m, sc, inv);
                        const int r = w * 32 + i * 4 + lr;
                        if (kc == 0) scale[(size_t)slot * SCALE_FLOATS + r] = inv;
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) split2(v[i][q * 2] * sc, v[i][q * 2 + 1] * sc, hi[q], lo[q]);
                        const uint32_t at = a + (uint32_t)r * 128u + ((uint32_t)(kc ^ (r & 7)) << 4);
                        sts128(at, hi);
                        sts128(at + A_HALF, lo);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(full[s]));
                    slot = slot + 1 == slots ? 0 : slot + 1;
                }
            }
        } else {
            // slabs of 16 columns: 4 lanes of 4 columns, 8 lanes of rows, 8 rows each
            const int cg = lane & 3, rr = lane >> 2;
            for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                int g, part, r0, r1, k0, nt;
                locate(unit, g, part, r0, r1, k0, nt);
                const int n0 = nt * p.NT, slabs = 8 + p.NT / 16;
                for (int r = r0; r < r1; r += BK, ++it) {
                    const int s = it % p.stages;
                    float v[2][8][4];
                    auto fetch = [&](int slab, float (&t)[8][4]) {
                        const bool is_b = slab >= 8;
                        const int col = (is_b ? n0 + (slab - 8) * 16 : k0 + slab * 16) + cg * 4, width = is_b ? p.out : p.K;
                        const float *src = (is_b ? b_in : a_in) + (size_t)(r + rr) * width + col;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            load_floats<4>(src + (size_t)(i * 8) * width, r + rr + i * 8 < r1 ? width - col : 0, is_b ? p.b_access : p.a_access, t[i]);
                    };
                    fetch(w, v[0]);
                    ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), ((uint32_t)(it / p.stages) & 1u) ^ 1u, gave_up));
                    if (!ok) break;
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes;
                    auto put = [&](int slab, const float (&t)[8][4]) {
                        const bool is_b = slab >= 8;
                        const int col = (is_b ? slab - 8 : slab) * 16 + cg * 4;          // within the tile
                        float sc[4], inv[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t m = 0;
#pragma unroll
                            for (int i = 0; i < 8; ++i) m = max(m, magnitude(t[i][q]));
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) m = max(m, __shfl_xor_sync(QMLB_FULL_MASK, m, o));
                            scales(m, sc[q], inv[q]);
                        }
                        if (rr == 0)
                            *reinterpret_cast<float4 *>(scale + (size_t)slot * SCALE_FLOATS + (is_b ? 128 : 0) + col) = make_float4(inv[0], inv[1], inv[2], inv[3]);
                        const uint32_t base = a + (is_b ? 2 * A_HALF : 0) + (uint32_t)(col >> 6) * 8192u, half = is_b ? p.b_half : A_HALF;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            uint32_t h0, h1, l0, l1;
                            split2(t[i][0] * sc[0], t[i][1] * sc[1], h0, l0);
                            split2(t[i][2] * sc[2], t[i][3] * sc[3], h1, l1);
                            const uint32_t at = base + (uint32_t)(rr + i * 8) * 128u + ((uint32_t)((col & 63) * 2) ^ ((uint32_t)rr << 4));
                            sts64(at, h0, h1);
                            sts64(at + half, l0, l1);
                        }
                    };
                    for (int q = w; q < slabs; q += 8) {
                        if (q + 4 < slabs) fetch(q + 4, v[1]);
                        put(q, v[0]);
                        if (q + 8 < slabs) fetch(q + 8, v[0]);
                        if (q + 4 < slabs) put(q + 4, v[1]);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(full[s]));
                    slot = slot + 1 == slots ? 0 : slot + 1;
                }
            }
        }
        if (!ok) failed = 1;
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        const int quarter = warp & 3, h = (warp - FOLD_WARP) >> 2, half = p.NT / 2;       // rows and columns of this warp
        unsigned char *mine = epi + (warp - FOLD_WARP) * 2048;
        const uint32_t lane_field = (uint32_t)(quarter * 32) << 16;
        int it = 0, slot = 0;
        bool ok = true;
        for (int unit = blockIdx.x; unit < total; unit += gridDim.x) {
            int g, part, r0, r1, k0, nt;
            locate(unit, g, part, r0, r1, k0, nt);
            const int chunks = chunks_of(r0, r1);
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.f;
            for (int c = 0; c < chunks && ok; ++c, ++it) {
                const int buf = it & 1;
                ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(acc_full[buf]), (uint32_t)(it >> 1) & 1u, gave_up));
                if (!ok) break;
                fence_after();
                const float *sc = scale + (size_t)slot * SCALE_FLOATS;
                const float mine_scale = sc[quarter * 32 + lane];
                const float *cols = sc + 128 + h * half;
                const uint32_t from = tmem + (uint32_t)buf * BUF_COLS + lane_field + (uint32_t)(h * half);
#pragma unroll
                for (int cc = 0; cc < 128; cc += 8) {
                    if (cc < half) {
                        uint32_t t[8];
                        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                     : "=r"(t[0]), "=r"(t[1]), "=r"(t[2]), "=r"(t[3]), "=r"(t[4]), "=r"(t[5]), "=r"(t[6]), "=r"(t[7])
                                     : "r"(from + (uint32_t)cc));
                        const float4 f0 = *reinterpret_cast<const float4 *>(cols + cc), f1 = *reinterpret_cast<const float4 *>(cols + cc + 4);
                        tmem_ld_wait();
                        acc[cc] = fmaf(__uint_as_float(t[0]), f0.x * mine_scale, acc[cc]);
                        acc[cc + 1] = fmaf(__uint_as_float(t[1]), f0.y * mine_scale, acc[cc + 1]);
                        acc[cc + 2] = fmaf(__uint_as_float(t[2]), f0.z * mine_scale, acc[cc + 2]);
                        acc[cc + 3] = fmaf(__uint_as_float(t[3]), f0.w * mine_scale, acc[cc + 3]);
                        acc[cc + 4] = fmaf(__uint_as_float(t[4]), f1.x * mine_scale, acc[cc + 4]);
                        acc[cc + 5] = fmaf(__uint_as_float(t[5]), f1.y * mine_scale, acc[cc + 5]);
                        acc[cc + 6] = fmaf(__uint_as_float(t[6]), f1.z * mine_scale, acc[cc + 6]);
                        acc[cc + 7] = fmaf(__uint_as_float(t[7]), f1.w * mine_scale, acc[cc + 7]);
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(acc_free[buf]));
                slot = slot + 1 == slots ? 0 : slot + 1;
            }
            if (!ok) {
                failed = 1;                                     // at once: the other roles stop waiting
#pragma unroll
                for (int i = 0; i < 128; ++i) acc[i] = __int_as_float(0x7fc00000);
            }
            // where the tile goes: rows of y, of dW, or of a part
            const int col0 = nt * p.NT + h * half;
            float *to;
            size_t row_floats;
            int rows, width, access;
            if (!GRAD) {
                row_floats = (size_t)p.out;
                to = out + (size_t)(r0 + quarter * 32) * row_floats + col0;
                rows = min(32, r1 - r0 - quarter * 32);
                width = p.out - col0;
                access = p.out_access;
            } else {
                rows = min(32, p.K - k0 - quarter * 32);
                if (gr.parts[g + 1] - gr.parts[g] == 1) {
                    row_floats = (size_t)p.out;
                    to = out + ((size_t)g * p.K + k0 + quarter * 32) * row_floats + col0;
                    width = p.out - col0;
                    access = p.out_access;
                } else {
                    const size_t part_slot = (size_t)(gr.split[g] + part - gr.parts[g]);
                    row_floats = (size_t)p.ntiles * p.NT;
                    to = partial + (part_slot * p.K + k0 + quarter * 32) * row_floats + col0;
                    width = half;
                    access = 16;
                }
            }
            width = min(width, half);
#pragma unroll
            for (int cc = 0; cc < 128; cc += 16) {
                if (cc < half) {
                    // 32 rows x 16 columns through shared memory: 64-byte pieces of rows
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<float4 *>(mine + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) =
                            make_float4(acc[cc + q * 4], acc[cc + q * 4 + 1], acc[cc + q * 4 + 2], acc[cc + q * 4 + 3]);
                    __syncwarp();
                    const int cols = min(16, width - cc);
                    if (access == 16) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2), q = lane & 3;
                            const float4 t = *reinterpret_cast<const float4 *>(mine + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
                            if (r < rows && q * 4 < cols) *reinterpret_cast<float4 *>(to + (size_t)r * row_floats + cc + q * 4) = t;
                        }
                    } else {
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            const int r = i * 2 + (lane >> 4), q = lane & 15;
                            const float t = *reinterpret_cast<const float *>(mine + r * 64 + (((q >> 2) ^ ((r >> 1) & 3)) << 4) + (q & 3) * 4);
                            if (r < rows && q < cols) to[(size_t)r * row_floats + cc + q] = t;
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (tid == 0 && failed) atomicAdd(&g_timeouts, 1);
    if (warp == MMA_WARP) tmem_free(tmem, TMEM_COLS);
}

// Images of the matrices: per group, column tile and stretch of 64 along the depth NT lines of 64 high parts and NT lines of
// low parts, swizzled as the kernel's shared memory wants them, and NT inverse scales.  One block: 64 columns of one stretch.
template <bool TRANS>
__global__ void __launch_bounds__(256)
pack_kernel(const float *__restrict__ W, Shape p, int N, unsigned char *__restrict__ packed, float *__restrict__ pack_scales) {
    __shared__ uint32_t most[4][64];
    const int g = blockIdx.z, c = blockIdx.x;
    const int kq = TRANS ? threadIdx.x & 3 : threadIdx.x >> 6, cl = TRANS ? threadIdx.x >> 2 : threadIdx.x & 63;
    const int col = blockIdx.y * 64 + cl;
    const float *Wg = W + (size_t)g * p.K * p.out;
    float v[16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int k = c * BK + kq * 16 + i;
        v[i] = (col < p.out && k < p.K) ? (TRANS ? Wg[(size_t)col * N + k] : Wg[(size_t)k * N + col]) : 0.f;
        m = max(m, magnitude(v[i]));
    }
    most[kq][cl] = m;
    __syncthreads();
    m = max(max(most[0][cl], most[1][cl]), max(most[2][cl], most[3][cl]));
    if (col >= p.ntiles * p.NT) return;
    float s, inv;
    scales(m, s, inv);
    const int tile = col / p.NT, in = col - tile * p.NT;
    const size_t image = ((size_t)(g * p.ntiles + tile)) * p.nchunks + c;
    if (kq == 0) pack_scales[image * p.NT + in] = inv;
    unsigned char *line = packed + image * (2 * p.b_half) + (size_t)in * 128;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split2(v[q * 8 + i * 2] * s, v[q * 8 + i * 2 + 1] * s, hi[i], lo[i]);
        const int at = ((kq * 2 + q) ^ (in & 7)) << 4;
        *reinterpret_cast<uint4 *>(line + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(line + p.b_half + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// shared memory of a block, or the largest column tile that fits
size_t smem_of(const Shape &p, int arrays) {
    return (size_t)p.stages * (2 * A_HALF + 2 * p.b_half) + (size_t)(p.stages + 2) * SCALE_FLOATS * 4 + EPI + (size_t)arrays * (p.G + 1) * 4 + 1024;
}

void tile_columns(Shape &p, int out, bool grad, int arrays) {
    for (int limit = 256;; limit -= 64) {                      // many groups leave less shared memory for the stages
        const int nt = (out + limit - 1) / limit;
        p.NT = ((out + nt - 1) / nt + 15) / 16 * 16;
        p.ntiles = (out + p.NT - 1) / p.NT;
        p.b_half = grad ? (uint32_t)((p.NT + 63) / 64) * 8192u : (uint32_t)p.NT * 128u;
        p.stages = MAXST;
        while (p.stages > 2 && smem_of(p, arrays) > SMEM_LIMIT - 512) --p.stages;
        if (smem_of(p, arrays) <= SMEM_LIMIT - 512 || limit == 64) return;
    }
}

Shape product_shape(size_t n, int G, int K, int N, int transpose) {
    Shape p;
    memset(&p, 0, sizeof(p));
    p.n = (int)n;
    p.G = G;
    p.K = transpose ? N : K;
    p.out = transpose ? K : N;
    p.nchunks = (p.K + BK - 1) / BK;
    tile_columns(p, p.out, false, 2);
    return p;
}

}  // namespace

namespace qmlb {

size_t grouped_pair_workspace(size_t n, int G, int K, int N, int transpose) {
    const Shape p = product_shape(n, G, K, N, transpose);
    const size_t images = (size_t)G * p.ntiles * p.nchunks;
    return images * (2 * p.b_half + (size_t)p.NT * 4) + 256;
}

int grouped_pair(const float *x, const float *W, const int *start, size_t n, int G, int K, int N, int transpose, float *out, void *workspace,
                 cudaStream_t st) {
    Shape p = product_shape(n, G, K, N, transpose);
    p.a_access = access_bytes((size_t)p.K * 4, 4, x);
    p.out_access = access_bytes((size_t)p.out * 4, 4, out);
    unsigned char *packed = static_cast<unsigned char *>(workspace);
    const size_t images = (size_t)G * p.ntiles * p.nchunks;
    float *pack_scales = reinterpret_cast<float *>(packed + images * (2 * p.b_half));
    const dim3 pg((unsigned)p.nchunks, (unsigned)((p.ntiles * p.NT + 63) / 64), (unsigned)G);
    if (transpose) pack_kernel<true><<<pg, 256, 0, st>>>(W, p, N, packed, pack_scales);
    else pack_kernel<false><<<pg, 256, 0, st>>>(W, p, N, packed, pack_scales);
    const long units = ((long)((n + BM - 1) / BM) + G) * p.ntiles;
    const size_t smem = smem_of(p, 2);
    if (int rc = ensure_smem(pair_kernel<false>, smem, "qmlb_grouped_matmul")) return rc;
    pair_kernel<false><<<(unsigned)(units < 148 ? units : 148), NTHREADS, smem, st>>>(x, nullptr, packed, pack_scales, start, p, out, nullptr);
    return check_launch("qmlb_grouped_matmul");
}

int grouped_wgrad_pair(const float *x, const float *dy, const int *start, size_t n, int G, int K, int N, float *dW, void *workspace,
                       cudaStream_t st) {
    Shape p;
    memset(&p, 0, sizeof(p));
    p.n = (int)n;
    p.G = G;
    p.K = K;
    p.out = N;
    tile_columns(p, N, true, 3);
    p.ktiles = (K + BM - 1) / BM;
    p.split = wgrad_split(n, G, p.ktiles, p.ntiles);
    p.a_access = access_bytes((size_t)K * 4, 4, x);
    p.b_access = access_bytes((size_t)N * 4, 4, dy);
    p.out_access = access_bytes((size_t)N * 4, 4, dW);
    const long units = ((long)(n / p.split) + G) * p.ktiles * p.ntiles;
    const size_t smem = smem_of(p, 3);
    float *partial = static_cast<float *>(workspace);
    if (int rc = ensure_smem(pair_kernel<true>, smem, "qmlb_grouped_matmul_wgrad")) return rc;
    pair_kernel<true><<<(unsigned)(units < 148 ? units : 148), NTHREADS, smem, st>>>(x, dy, nullptr, nullptr, start, p, dW, partial);
    return wgrad_join(dW, QMLB_F32, start, n, G, K, N, p.split, p.ntiles * p.NT, partial, st);
}

size_t grouped_wgrad_pair_workspace(size_t n, int G, int K, int N) {
    Shape p;
    memset(&p, 0, sizeof(p));
    p.G = G;
    tile_columns(p, N, true, 3);
    return wgrad_slots(n, G, wgrad_split(n, G, (K + BM - 1) / BM, p.ntiles)) * K * p.ntiles * p.NT * 4 + 256;
}

int grouped_pair_timeouts() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace qmlb
