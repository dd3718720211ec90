// Products of ragged groups of rows with one matrix each, float32 operands, on the 16-bit tensor cores.
//
// Arithmetic.  A value x is the sum of three bf16 numbers, x = a + b + c: a = bf16(x), b = bf16(x - a), c = x - a - b, each rounded to
// nearest, 8 + 8 + 8 bits, |b| <= 2^-9 |x|, |c| <= 2^-18 |x|.  A product is a a' + a b' + b a' + b b' + a c' + c a'; the other three are
// less than 2^-25 of it.  bf16 has the exponents of float32, so this holds for every value by itself, whatever stands beside it
// (two fp16 parts on a common scale would take three products, but lose the small values of a stretch that holds large ones).  The
// parts of values below 2^-110 would leave the range, so all values are multiplied by 2^10 on their way in, and sums by 2^-20 on
// their way out: numbers above 2^-120 enter exactly, smaller ones are off by at most 2^-144, and values may reach 2^117 and sums 2^108
// before they overflow (see below; room for masks of 1e30).  Sums: the tensor core
// truncates when it adds, so an accumulator only ever covers one stretch of 64 values (the small products first, then a a'), and
// warps of CUDA cores add the stretches in registers in 32 bits, rounded.  Against 64 bits the results are off by about 1e-7 of
// their norm, a float32 product by 3e-7.
//
// Work split.  One persistent block per SM takes tiles of 128 x NT results:
//   warp 0          bulk copies of the matrix operand's images (products of rows; a packing kernel makes the images), one of the
//                   three parts at a time: a part's place is free again once the products that need it are issued and done
//   warp 1          issues tcgen05.mma, several tensor-memory accumulators in turn
//   warps 2-3       zero rows outside the groups, zero matrices of groups without rows
//   loading warps   load float32 rows, split, and write the swizzled operand images to shared memory
//   folding warps   (eight) add the finished accumulators to their registers, and store the tile
// Products of rows: NT <= 256, 4 loading warps, 128 sums per folding thread.  Gradient of the matrices: both operands are loaded
// by the loading warps (the depth runs over the rows of the group, the operands' lines run across it), and NT <= 128 leaves
// registers for eight of them, two per scheduler, and room for two stages (six parts of 128 are 96 KB; of 128 and 256 144 KB).
// 210,000 x (336, 256): products of rows 232 us, transposed 256 us (the six products alone take 132 us at the rate of a library
// product), gradient 386 us.  60,000 x 1,024 x 1,024 of 32 groups: 815, 820 and 1,092 us (461 us).  Of 5,600 cycles per stretch the
// issuing warp spends 2,500 issuing, 1,300 waiting for a part of the matrix, 900 for an accumulator while a tile is stored (11,000
// cycles per tile, of which two stretches hide half) and 850 for the rows; with smaller copies of the parts nothing changes.
// Registers are moved between the warps by setmaxnreg.
//
// Results that are not finite.  An infinity times the zero low part of another number is NaN, and scaled sums leave the range before
// their results do.  So a folding warp remembers its tiles with such results and, when no other warp waits for it any
// more, forms these results again as plain sums of fused multiply-adds over the operands as they are: they come out as a product in
// 32 bits gives them.  Finite tiles pay one packed multiply-add per two results for the test.
#include <cuda_bf16.h>
#include <string.h>

#include "grouped_rows.cuh"
#include "grouped_tc.cuh"

namespace {

using namespace qmlb::tc;

constexpr int BM = 128;
constexpr uint32_t A_IMAGE = BM * BK * 2;         // one part of the 128-wide operand
constexpr float SCALE = 1024.f, UNSCALE = 1.f / (SCALE * SCALE);
constexpr int TMA_WARP = 0, MMA_WARP = 1, LOAD_WARP = 4;
constexpr int MAXST = 4, MAXSLOT = 6;
template <bool GRAD>
struct Config {
    static constexpr int LOADERS = GRAD ? 8 : 4, FOLD_WARP = LOAD_WARP + LOADERS, THREADS = (FOLD_WARP + 8) * 32;
    static constexpr int NT = GRAD ? 128 : 256;   // widest tile
    static constexpr int ACCS = 512 / NT;         // accumulators in tensor memory
    // registers: launched with, then in the first warpgroup, the loading and the folding warps; their sum over the warpgroups
    // does not exceed what the block was launched with
    static constexpr int R_LAUNCH = GRAD ? 96 : 128, R_FIRST = 40, R_LOAD = 112, R_FOLD = GRAD ? 104 : 176;
    static_assert(R_FIRST * 4 + R_LOAD * LOADERS + R_FOLD * 8 <= R_LAUNCH * (4 + LOADERS + 8), "register split");
};
constexpr int PART_COST = 384;                    // of a part of a sum through scratch, in rows
constexpr int AHEAD = 4;                          // stretches by which rows are asked into L2 in front of their loads
constexpr uint32_t EPI = 8 * 2048;                // 32 rows x 16 columns per folding warp

__device__ int g_timeouts = 0;

struct Shape {
    int n, G, K, out;        // rows, groups, depth (products of rows) or columns of x (gradient), columns of the result
    int NT, ntiles, ktiles;  // ktiles: tiles of 128 columns of x (gradient)
    int nchunks;             // stretches of the depth (products of rows)
    int split;               // rows per part (gradient)
    int stages;              // of the 128-wide operand's three parts (gradient: and the other's)
    int slots;               // of one part of the NT-wide operand (products of rows)
    uint32_t b_image;        // one part of the NT-wide operand
    int a_access, b_access, out_access;
    size_t w_depth, w_col;   // steps of the matrix as it is, along the depth and along the columns (products of rows)
};

// the three parts of two values
__device__ __forceinline__ void split2(float2 x, uint32_t (&part)[3]) {
    x = __fmul2_rn(x, make_float2(SCALE, SCALE));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const __nv_bfloat162 h = __float22bfloat162_rn(x);
        part[i] = *reinterpret_cast<const uint32_t *>(&h);
        // minus the part: its bits are the upper halves of two floats
        x = __fadd2_rn(x, make_float2(__uint_as_float((part[i] << 16) ^ 0x80000000u), __uint_as_float((part[i] & 0xffff0000u) ^ 0x80000000u)));
    }
}
// Four consecutive floats, of which the first `valid` exist (the others become zeros).  Predicated loads without a branch: behind
// a branch the compiler waits for each load before the next.
__device__ __forceinline__ void load4(const float *src, bool wanted, float2 (&v)[2]) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.f32 %0, 0f00000000;\n\tmov.f32 %1, 0f00000000;\n\tmov.f32 %2, 0f00000000;\n\tmov.f32 %3, 0f00000000;\n\t"
        "@p ld.global.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&f"(v[0].x), "=&f"(v[0].y), "=&f"(v[1].x), "=&f"(v[1].y)
        : "l"(__cvta_generic_to_global(src)), "r"((int)wanted));
}
__device__ __forceinline__ void load1(const float *src, bool wanted, float &v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.global.f32 %0, [%1];\n\t}"
                 : "=&f"(v)
                 : "l"(__cvta_generic_to_global(src)), "r"((int)wanted));
}
__device__ __forceinline__ void load4_narrow(const float *src, int valid, float2 (&v)[2]) {
    load1(src, valid > 0, v[0].x);
    load1(src + 1, valid > 1, v[0].y);
    load1(src + 2, valid > 2, v[1].x);
    load1(src + 3, valid > 3, v[1].y);
}
__device__ __forceinline__ void prefetch_l2(const void *src) { asm volatile("prefetch.global.L2 [%0];" ::"l"(__cvta_generic_to_global(src)) : "memory"); }
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

// sum of a[d * a_step] * b[d * b_step] over the depth in 32 bits, by all lanes of a warp; only `wanted` ones go on for the others
__device__ __forceinline__ float plain_sum(const float *__restrict__ a, size_t a_step, const float *__restrict__ b, size_t b_step, int depth, bool wanted) {
    float s = 0.f;
    for (int d0 = 0; d0 < depth && __any_sync(QMLB_FULL_MASK, wanted && !isnan(s)); d0 += 8) {      // NaN stays
        float u[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {                    // addresses are clamped instead of tested: all loads are in flight together
            const size_t d = (size_t)min(d0 + i, depth - 1);
            u[i] = a[d * a_step];
            v[i] = b[d * b_step];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (d0 + i < depth) s = fmaf(u[i], v[i], s);
    }
    return s;
}

// Products of rows: a = x [n, K], b = the matrices, packed = their images, result y [n, out].
// GRAD: a = x [n, K], b = dy [n, out], result dW [G, K, out], partial = parts of split groups.
template <bool GRAD>
__global__ void __launch_bounds__(Config<GRAD>::THREADS, 1)
pair_kernel(const float *__restrict__ a_in, const float *__restrict__ b_in, const unsigned char *__restrict__ packed,
            const int *__restrict__ start, Shape p, float *__restrict__ out, float *__restrict__ partial) {
    using C = Config<GRAD>;
    constexpr int NACC = C::ACCS, NT_MAX = C::NT, FOLD_WARP = C::FOLD_WARP, HALF = C::NT / 2;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[MAXST], empty[MAXST], b_full[MAXSLOT], b_empty[MAXSLOT], acc_full[NACC], acc_free[NACC], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char *sp = smem_raw + (sbase - smem_u32(smem_raw));
    const uint32_t stage_bytes = 3 * A_IMAGE + (GRAD ? 3 * p.b_image : 0u);
    const uint32_t b_ring = sbase + (uint32_t)p.stages * stage_bytes;                 // products of rows
    unsigned char *epi = sp + (size_t)p.stages * stage_bytes + (GRAD ? 0u : (size_t)p.slots * p.b_image);
    Groups gr;
    gr.start = reinterpret_cast<int *>(epi + EPI);
    gr.parts = gr.start + p.G + 1;
    gr.split = GRAD ? gr.parts + p.G + 1 : nullptr;
    auto bar = [](const uint64_t &b) { return smem_u32(&b); };

    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar(full[s]), C::LOADERS);
            mbar_init(bar(empty[s]), 1);
        }
        for (int s = 0; s < p.slots; ++s) { mbar_init(bar(b_full[s]), 1); mbar_init(bar(b_empty[s]), 1); }
        for (int i = 0; i < NACC; ++i) { mbar_init(bar(acc_full[i]), 1); mbar_init(bar(acc_free[i]), 8); }
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
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_FIRST));
        if (warp == TMA_WARP) {
            if (!GRAD && lane == 0) {
                int it = 0;
                bool ok = true;
                for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                    int g, part, r0, r1, k0, nt;
                    locate(unit, g, part, r0, r1, k0, nt);
                    const unsigned char *image = packed + (size_t)(g * p.ntiles + nt) * p.nchunks * (3 * p.b_image);
                    for (int c = 0; c < p.nchunks * 3; ++c, ++it) {           // c, b, a of every stretch
                        const int s = it % p.slots;
                        if (!mbar_wait(bar(b_empty[s]), ((uint32_t)(it / p.slots) & 1u) ^ 1u, gave_up)) { ok = false; break; }
                        mbar_expect_tx(bar(b_full[s]), p.b_image);
                        bulk_copy(b_ring + (uint32_t)s * p.b_image, image + (size_t)c * p.b_image, p.b_image, bar(b_full[s]));
                    }
                }
                if (!ok) failed = 1;
                for (int i = max(0, it - p.slots); i < it; ++i)           // no copy may be in flight when the block leaves
                    for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(b_full[i % p.slots]), (uint32_t)(i / p.slots) & 1u); ++tries) {}
            }
        } else if (warp == MMA_WARP) {
            const uint32_t idesc = instr_desc(true, GRAD, GRAD, BM, p.NT);
            constexpr uint32_t step = GRAD ? 128u : 2u, block = GRAD ? 8192u : 16u;
            int it = 0, bt = 0;
            bool ok = true;
            for (int unit = blockIdx.x; unit < total && ok; unit += gridDim.x) {
                int g, part, r0, r1, k0, nt;
                locate(unit, g, part, r0, r1, k0, nt);
                const int chunks = chunks_of(r0, r1), depth = GRAD ? r1 - r0 : p.K;
                for (int c = 0; c < chunks && ok; ++c, ++it) {
                    const int s = it % p.stages, buf = it % NACC;
                    bool w = mbar_wait(bar(acc_free[buf]), ((uint32_t)(it / NACC) & 1u) ^ 1u, gave_up);
                    w = w && mbar_wait(bar(full[s]), (uint32_t)(it / p.stages) & 1u, gave_up, it ? WAIT_LIMIT : QMLB_TEST_FIRST_WAIT_POLLS);
                    if (!__all_sync(QMLB_FULL_MASK, w)) { ok = false; break; }
                    fence_after();
                    const int steps = min(BK / 16, (depth - c * BK + 15) / 16);
                    const uint32_t a = sbase + (uint32_t)s * stage_bytes, d = tmem + (uint32_t)buf * NT_MAX;
                    // part i of the one operand times the part at `b` of the other
                    auto multiply = [&](int i, uint32_t b, bool first) {
                        const uint32_t al = desc_lo(a + (uint32_t)i * A_IMAGE, block), bl = desc_lo(b, block);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            if (k >= steps) break;
                            mma_f16(d, al + k * step, DESC_HI_SW128, bl + k * step, DESC_HI_SW128, idesc, first && k == 0 ? 0u : 1u);
                        }
                    };
                    if (GRAD) {
                        const uint32_t b = a + 3 * A_IMAGE;
                        if (elect_one()) {
                            multiply(0, b + 2 * p.b_image, true);
                            multiply(2, b, false);
                            multiply(1, b + p.b_image, false);
                            multiply(0, b + p.b_image, false);
                            multiply(1, b, false);
                            multiply(0, b, false);
                            mma_commit(bar(empty[s]));
                            mma_commit(bar(acc_full[buf]));
                        }
                        __syncwarp();
                    } else {
#pragma unroll 1
                        for (int j = 2; j >= 0; --j, ++bt) {                  // parts c, b, a of the matrix
                            const int slot = bt % p.slots;
                            w = mbar_wait(bar(b_full[slot]), (uint32_t)(bt / p.slots) & 1u, gave_up);
                            if (!__all_sync(QMLB_FULL_MASK, w)) { ok = false; break; }
                            const uint32_t b = b_ring + (uint32_t)slot * p.b_image;
                            if (elect_one()) {
                                if (j == 0) multiply(2, b, false);
                                if (j <= 1) multiply(1, b, false);
                                multiply(0, b, j == 2);
                                mma_commit(bar(b_empty[slot]));
                                if (j == 0) {
                                    mma_commit(bar(empty[s]));
                                    mma_commit(bar(acc_full[buf]));
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
            }
            if (!ok) failed = 1;
            if (lane == 0) mma_commit(bar(done));
            __syncwarp();
            for (int tries = 0; tries < WAIT_LIMIT && !mbar_try(bar(done), 0u); ++tries) {}
        } else if (GRAD) {
            zero_empty_groups(gr, p.G, reinterpret_cast<unsigned char *>(out), (size_t)p.K * p.out * 4, p.out_access, blockIdx.x * 2 + warp - 2, gridDim.x * 2, lane);
        } else {
            const int first = gr.start[0], last = max(gr.start[p.G], first), outside = first + (p.n - last);
            for (int i = blockIdx.x * 2 + (warp - 2); i < outside; i += gridDim.x * 2) {
                float *row = out + (size_t)(i < first ? i : last + (i - first)) * p.out;
                for (int c = lane; c < p.out; c += 32) row[c] = 0.f;
            }
        }
    } else if (warp < FOLD_WARP) {
        if constexpr (C::R_LOAD < C::R_LAUNCH) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_LOAD));
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_LOAD));
        const int w = warp - LOAD_WARP;
        bool ok = true;
        if (!GRAD) {
            // A row is 8 lanes of 8 values, a pass 4 rows per warp.  Two halves of 4 passes each: while one is split and stored,
            // the loads of the other are in flight.
            const int lr = lane >> 3, kc = lane & 7;
            float2 v[2][4][4];
            int unit = blockIdx.x, c = 0, row = 0, end = 0;          // what is loaded next
            auto place = [&]() {
                int g, part, r0, r1, k0, nt;
                if (unit < total) {
                    locate(unit, g, part, r0, r1, k0, nt);
                    row = r0 + w * 32 + lr;
                    end = r1;
                }
            };
            auto fetch = [&](int h, float2 (&t)[4][4]) {
                if (unit >= total) return;
                const int k = c * BK + kc * 8, left = p.K - k;
                const float *src = a_in + (size_t)(row + h * 16) * p.K + k;
                if (p.a_access == 16) {                              // a depth that is a multiple of 4: all four exist, or none
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool in = row + (h * 4 + i) * 4 < end;
                        load4(src + (size_t)(i * 4) * p.K, in && left > 0, reinterpret_cast<float2(&)[2]>(t[i][0]));
                        load4(src + (size_t)(i * 4) * p.K + 4, in && left > 4, reinterpret_cast<float2(&)[2]>(t[i][2]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int valid = row + (h * 4 + i) * 4 < end ? left : 0;
                        load4_narrow(src + (size_t)(i * 4) * p.K, valid, reinterpret_cast<float2(&)[2]>(t[i][0]));
                        load4_narrow(src + (size_t)(i * 4) * p.K + 4, valid - 4, reinterpret_cast<float2(&)[2]>(t[i][2]));
                    }
                }
            };
            auto next = [&]() {
                if (++c == p.nchunks) {
                    c = 0;
                    unit += gridDim.x;
                    place();
                }
            };
            // Rows on their way into L2, AHEAD stretches in front: the registers hold too few loads in flight for the latency of
            // the memory, but enough for that of the cache.
            int pu = blockIdx.x, pc = 0, prow = 0, pend = 0;
            auto pplace = [&]() {
                int g, part, r0, k0, nt;
                if (pu < total) {
                    locate(pu, g, part, r0, pend, k0, nt);
                    prow = r0 + w * 32 + lane;
                }
            };
            auto prefetch = [&]() {
                if (pu >= total) return;
                if (prow < pend) {
                    const float *src = a_in + (size_t)prow * p.K + pc * BK;
                    prefetch_l2(src);
                    if (pc * BK + 32 < p.K) prefetch_l2(src + 32);
                }
                if (++pc == p.nchunks) {
                    pc = 0;
                    pu += gridDim.x;
                    pplace();
                }
            };
            pplace();
            for (int i = 0; i < AHEAD; ++i) prefetch();
            place();
            fetch(0, v[0]);
            fetch(1, v[1]);
            int s = 0;
            uint32_t phase = 1;
            while (unit < total) {
                ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), phase, gave_up));
                if (!ok) break;
                const uint32_t a = sbase + (uint32_t)s * stage_bytes;
                auto put = [&](int h, const float2 (&t)[4][4]) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = w * 32 + (h * 4 + i) * 4 + lr;
                        uint32_t v[3][4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t u[3];
                            split2(t[i][q], u);
                            v[0][q] = u[0];
                            v[1][q] = u[1];
                            v[2][q] = u[2];
                        }
                        const uint32_t at = a + (uint32_t)r * 128u + ((uint32_t)(kc ^ (r & 7)) << 4);
#pragma unroll
                        for (int e = 0; e < 3; ++e) sts128(at + (uint32_t)e * A_IMAGE, v[e]);
                    }
                };
                prefetch();
                put(0, v[0]);
                next();
                fetch(0, v[0]);
                put(1, v[1]);
                fetch(1, v[1]);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(full[s]));
                if (++s == p.stages) { s = 0; phase ^= 1u; }
            }
        } else {
            // Slabs of 16 columns: 4 lanes of 4 columns, 8 lanes of rows, 8 rows each.  A warp takes one slab of x and one of dy.
            const int cg = lane & 3, rr = lane >> 2, col = w * 16 + cg * 4;
            const bool has_b = w * 16 < p.NT;
            float2 v[2][8][2];
            struct Cursor { int unit, r, r1, k0, n0; };
            auto place = [&](Cursor &u) {
                if (u.unit >= total) return;
                int g, part, nt;
                locate(u.unit, g, part, u.r, u.r1, u.k0, nt);
                u.n0 = nt * p.NT;
            };
            auto advance = [&](Cursor &u) {
                u.r += BK;
                if (u.r < u.r1) return;
                u.unit += gridDim.x;
                place(u);
            };
            auto fetch = [&](const Cursor &u, const float *in, int first, int width, int access, float2 (&t)[8][2]) {
                if (u.unit >= total) return;
                const int rows = u.r1 - u.r - rr;
                const float *src = in + (size_t)(u.r + rr) * width + first + col;
                if (access == 16) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) load4(src + (size_t)(i * 8) * width, i * 8 < rows && first + col < width, t[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) load4_narrow(src + (size_t)(i * 8) * width, i * 8 < rows ? width - first - col : 0, t[i]);
                }
            };
            Cursor at{(int)blockIdx.x, 0, 0, 0, 0};
            place(at);
            fetch(at, a_in, at.k0, p.K, p.a_access, v[0]);
            if (has_b) fetch(at, b_in, at.n0, p.out, p.b_access, v[1]);
            int s = 0;
            uint32_t phase = 1;
            auto store = [&](const float2 (&t)[8][2], uint32_t to, uint32_t image) {
                to += (uint32_t)(col >> 6) * 8192u + (uint32_t)rr * 128u + ((uint32_t)((col & 63) * 2) ^ ((uint32_t)rr << 4));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t u[3], v[3];
                    split2(t[i][0], u);
                    split2(t[i][1], v);
#pragma unroll
                    for (int e = 0; e < 3; ++e) sts64(to + (uint32_t)e * image + (uint32_t)i * 1024u, u[e], v[e]);
                }
            };
            while (at.unit < total) {
                if (!(ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(empty[s]), phase, gave_up)))) break;
                const uint32_t stage = sbase + (uint32_t)s * stage_bytes;
                Cursor next = at;
                advance(next);
                store(v[0], stage, A_IMAGE);
                fetch(next, a_in, next.k0, p.K, p.a_access, v[0]);
                if (has_b) {
                    store(v[1], stage + 3 * A_IMAGE, p.b_image);
                    fetch(next, b_in, next.n0, p.out, p.b_access, v[1]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(full[s]));
                if (++s == p.stages) { s = 0; phase ^= 1u; }
                at = next;
            }
        }
        if (!ok) failed = 1;
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_FOLD));
        const int quarter = warp & 3, h = (warp - FOLD_WARP) >> 2, half = p.NT / 2;       // rows and columns of this warp
        unsigned char *mine = epi + (warp - FOLD_WARP) * 2048;
        const uint32_t lane_field = (uint32_t)(quarter * 32) << 16;
        int it = 0;
        bool ok = true;
        // where a tile goes: rows of y, of dW, or of a part
        auto target = [&](int g, int part, int r0, int r1, int k0, int nt, size_t &row_floats, int &rows, int &width, int &access) {
            const int col0 = nt * p.NT + h * half;
            float *to;
            row_floats = (size_t)p.out;
            width = p.out - col0;
            access = p.out_access;
            if (!GRAD) {
                to = out + (size_t)(r0 + quarter * 32) * row_floats + col0;
                rows = min(32, r1 - r0 - quarter * 32);
            } else {
                rows = min(32, p.K - k0 - quarter * 32);
                if (gr.parts[g + 1] - gr.parts[g] == 1) {
                    to = out + ((size_t)g * p.K + k0 + quarter * 32) * row_floats + col0;
                } else {
                    const size_t part_slot = (size_t)(gr.split[g] + part - gr.parts[g]);
                    row_floats = (size_t)p.ntiles * p.NT;
                    to = partial + (part_slot * p.K + k0 + quarter * 32) * row_floats + col0;
                    width = half;
                    access = 16;
                }
            }
            width = min(width, half);
            return to;
        };
        unsigned long long odd = 0;                             // units with results that are not finite (the last bit: all from the 64th on)
        for (int unit = blockIdx.x, nth = 0; unit < total; unit += gridDim.x, ++nth) {
            int g, part, r0, r1, k0, nt;
            locate(unit, g, part, r0, r1, k0, nt);
            const int chunks = chunks_of(r0, r1);
            float2 acc[HALF / 2];
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) acc[i] = make_float2(0.f, 0.f);
            for (int c = 0; c < chunks && ok; ++c, ++it) {
                const int buf = it % NACC;
                ok = __all_sync(QMLB_FULL_MASK, mbar_wait(bar(acc_full[buf]), (uint32_t)(it / NACC) & 1u, gave_up));
                if (!ok) break;
                fence_after();
                const uint32_t from = tmem + (uint32_t)buf * NT_MAX + lane_field + (uint32_t)(h * half);
                // 16 columns at a time, the next 16 on their way from tensor memory meanwhile
                uint32_t t[2][16];
                tmem_ld16(from, t[0]);
#pragma unroll
                for (int cc = 0; cc < HALF; cc += 16) {
                    if (cc < half) {
                        tmem_ld_wait();
                        if (cc + 16 < half) tmem_ld16(from + (uint32_t)cc + 16u, t[(cc / 16 + 1) & 1]);
                        const uint32_t(&u)[16] = t[(cc / 16) & 1];
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            acc[cc / 2 + q] = __fadd2_rn(make_float2(__uint_as_float(u[q * 2]), __uint_as_float(u[q * 2 + 1])), acc[cc / 2 + q]);
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(acc_free[buf]));
            }
            if (!ok) {
                failed = 1;                                     // at once: the other roles stop waiting
#pragma unroll
                for (int i = 0; i < HALF / 2; ++i) acc[i] = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
            }
            size_t row_floats;
            int rows, width, access;
            float *to = target(g, part, r0, r1, k0, nt, row_floats, rows, width, access);
            float2 test = make_float2(0.f, 0.f);                // stays zero while all results are finite
#pragma unroll
            for (int cc = 0; cc < HALF; cc += 16) {
                if (cc < half) {
                    // 32 rows x 16 columns through shared memory: 64-byte pieces of rows
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float2 unscale = make_float2(UNSCALE, UNSCALE);
                        const float2 lo = __fmul2_rn(acc[cc / 2 + q * 2], unscale), hi = __fmul2_rn(acc[cc / 2 + q * 2 + 1], unscale);
                        if (cc + q * 4 < half) {                // (what lies behind is no result of this warp)
                            test = __ffma2_rn(lo, make_float2(0.f, 0.f), test);
                            test = __ffma2_rn(hi, make_float2(0.f, 0.f), test);
                        }
                        *reinterpret_cast<float4 *>(mine + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = make_float4(lo.x, lo.y, hi.x, hi.y);
                    }
                    __syncwarp();
                    const int left = min(16, width - cc);
                    if (access == 16) {
                        float *at = to + (size_t)(lane >> 2) * row_floats + cc + (lane & 3) * 4;
                        uint4 t[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = i * 8 + (lane >> 2);
                            t[i] = *reinterpret_cast<const uint4 *>(mine + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            store_if(at, t[i], i * 8 + (lane >> 2) < rows && (lane & 3) * 4 < left);
                            at += 8 * row_floats;
                        }
                    } else {
                        float *at = to + (size_t)(lane >> 4) * row_floats + cc + (lane & 15);
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            const int r = i * 2 + (lane >> 4), q = lane & 15;
                            const uint32_t t = *reinterpret_cast<const uint32_t *>(mine + r * 64 + (((q >> 2) ^ ((r >> 1) & 3)) << 4) + (q & 3) * 4);
                            store_if(at, t, r < rows && q < left);
                            at += 2 * row_floats;
                        }
                    }
                    __syncwarp();
                }
            }
            if (__any_sync(QMLB_FULL_MASK, test.x + test.y != 0.f)) odd |= 1ull << min(nth, 63);
        }
        // what is not finite, as a product in 32 bits gives it (nobody waits for this warp any more)
        for (int unit = blockIdx.x, nth = 0; unit < total && odd && ok; unit += gridDim.x, ++nth) {
            if (!((odd >> min(nth, 63)) & 1)) continue;
            int g, part, r0, r1, k0, nt, rows, width, access;
            locate(unit, g, part, r0, r1, k0, nt);
            size_t row_floats;
            float *to = target(g, part, r0, r1, k0, nt, row_floats, rows, width, access);
            width = min(width, p.out - nt * p.NT - h * half);   // a part's row has room for columns that do not exist
            for (int r = 0; r < rows; ++r) {
                for (int cc = 0; cc < width; cc += 32) {
                    const int c = min(cc + lane, width - 1), col = nt * p.NT + h * half + c;
                    float *at = to + (size_t)r * row_floats + c;
                    const bool wanted = cc + lane < width && !isfinite(*at);
                    if (!__any_sync(QMLB_FULL_MASK, wanted)) continue;
                    float v;
                    if (GRAD) {
                        v = plain_sum(a_in + (size_t)r0 * p.K + k0 + quarter * 32 + r, (size_t)p.K, b_in + (size_t)r0 * p.out + col, (size_t)p.out, r1 - r0, wanted);
                    } else {
                        v = plain_sum(a_in + (size_t)(r0 + quarter * 32 + r) * p.K, 1, b_in + (size_t)g * p.K * p.out + (size_t)col * p.w_col, p.w_depth, p.K, wanted);
                    }
                    if (wanted) *at = v;
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

// Images of the matrices: per group, column tile and stretch of 64 along the depth the parts c, b and a, NT lines of 64 values each,
// swizzled as the kernel's shared memory wants them.  One block: 16 columns of one group, two stretches at a time.
template <bool TRANS>
__global__ void __launch_bounds__(256)
pack_kernel(const float *__restrict__ W, Shape p, int N, unsigned char *__restrict__ packed) {
    const int g = blockIdx.y;
    // neighbouring threads read neighbouring addresses: along the columns, or along the depth of the transposed matrix
    const int cl = TRANS ? threadIdx.x >> 4 : threadIdx.x & 15, kl = TRANS ? threadIdx.x & 15 : threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + cl;
    const float *Wg = W + (size_t)g * p.K * p.out;
    const int inside = min(col, p.out - 1);              // addresses are clamped instead of tested: the loads are in flight together
    const float *base = TRANS ? Wg + (size_t)inside * N : Wg + inside;
    const size_t step = TRANS ? 1 : (size_t)N;
    const int tile = col / p.NT, in = col - tile * p.NT;               // the grid covers whole tiles
    const size_t image = (size_t)(g * p.ntiles + tile) * p.nchunks;
#pragma unroll 2
    for (int c0 = (int)blockIdx.z * 2; c0 < p.nchunks; c0 += (int)gridDim.z * 2) {      // 16 threads of 8 values per column
        const int c = c0 + (kl >> 3), k0 = c0 * BK + kl * 8;
        if (c >= p.nchunks) continue;
        float t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = base[(size_t)min(k0 + i, p.K - 1) * step];
        uint32_t v[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = make_float2(col < p.out && k0 + i * 2 < p.K ? t[i * 2] : 0.f, col < p.out && k0 + i * 2 + 1 < p.K ? t[i * 2 + 1] : 0.f);
            uint32_t u[3];
            split2(x, u);
            v[0][i] = u[0];
            v[1][i] = u[1];
            v[2][i] = u[2];
        }
        unsigned char *line = packed + (image + c) * (3 * p.b_image) + (size_t)in * 128 + (((kl & 7) ^ (in & 7)) << 4);
#pragma unroll
        for (int e = 0; e < 3; ++e) *reinterpret_cast<uint4 *>(line + (size_t)(2 - e) * p.b_image) = make_uint4(v[e][0], v[e][1], v[e][2], v[e][3]);
    }
}

template <bool GRAD>
size_t smem_of(const Shape &p) {
    const size_t operands = GRAD ? (size_t)p.stages * 3 * (A_IMAGE + p.b_image) : (size_t)p.stages * 3 * A_IMAGE + (size_t)p.slots * p.b_image;
    return operands + EPI + (size_t)(GRAD ? 3 : 2) * (p.G + 1) * 4 + 1024;
}

// Columns per tile and stages.  Many groups leave less shared memory for the stages: then the tiles get narrower.  Products of rows:
// three slots let a part of the matrix arrive while the products of the two others run; a third stage of the rows comes before more.
template <bool GRAD>
void tile_columns(Shape &p, int out) {
    const size_t limit = SMEM_LIMIT - 512;
    for (int widest = Config<GRAD>::NT;; widest -= 64) {
        const int nt = (out + widest - 1) / widest;
        p.NT = ((out + nt - 1) / nt + 15) / 16 * 16;
        p.ntiles = (out + p.NT - 1) / p.NT;
        p.b_image = GRAD ? (uint32_t)((p.NT + 63) / 64) * 8192u : (uint32_t)p.NT * 128u;
        p.slots = GRAD ? 0 : 3;
        p.stages = GRAD ? MAXST : 3;
        while (p.stages > 2 && smem_of<GRAD>(p) > limit) --p.stages;
        const bool fits = smem_of<GRAD>(p) <= limit;
        while (!GRAD && fits && p.slots < MAXSLOT) {
            ++p.slots;
            if (smem_of<GRAD>(p) > limit) { --p.slots; break; }
        }
        if (fits || widest == 64) return;
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
    tile_columns<false>(p, p.out);
    return p;
}

}  // namespace

namespace qmlb {

size_t grouped_pair_workspace(size_t n, int G, int K, int N, int transpose) {
    const Shape p = product_shape(n, G, K, N, transpose);
    const size_t images = (size_t)G * p.ntiles * p.nchunks;
    return images * (3 * p.b_image) + 256;
}

int grouped_pair(const float *x, const float *W, const int *start, size_t n, int G, int K, int N, int transpose, float *out, void *workspace,
                 cudaStream_t st) {
    Shape p = product_shape(n, G, K, N, transpose);
    p.a_access = access_bytes((size_t)p.K * 4, 4, x);
    p.out_access = access_bytes((size_t)p.out * 4, 4, out);
    p.w_depth = transpose ? 1 : (size_t)N;
    p.w_col = transpose ? (size_t)N : 1;
    unsigned char *packed = static_cast<unsigned char *>(workspace);
    const unsigned pairs = (unsigned)(p.nchunks + 1) / 2;
    const dim3 pg((unsigned)(p.ntiles * p.NT / 16), (unsigned)G, pairs < 64 ? pairs : 64);
    if (transpose) pack_kernel<true><<<pg, 256, 0, st>>>(W, p, N, packed);
    else pack_kernel<false><<<pg, 256, 0, st>>>(W, p, N, packed);
    const long units = ((long)((n + BM - 1) / BM) + G) * p.ntiles;
    const size_t smem = smem_of<false>(p);
    if (int rc = ensure_smem(pair_kernel<false>, smem, "qmlb_grouped_matmul")) return rc;
    pair_kernel<false><<<(unsigned)(units < 148 ? units : 148), Config<false>::THREADS, smem, st>>>(x, W, packed, start, p, out, nullptr);
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
    tile_columns<true>(p, N);
    p.ktiles = (K + BM - 1) / BM;
    p.split = wgrad_split(n, G, p.ktiles, p.ntiles, PART_COST);
    p.a_access = access_bytes((size_t)K * 4, 4, x);
    p.b_access = access_bytes((size_t)N * 4, 4, dy);
    p.out_access = access_bytes((size_t)N * 4, 4, dW);
    const long units = ((long)(n / p.split) + G) * p.ktiles * p.ntiles;
    const size_t smem = smem_of<true>(p);
    float *partial = static_cast<float *>(workspace);
    if (int rc = ensure_smem(pair_kernel<true>, smem, "qmlb_grouped_matmul_wgrad")) return rc;
    pair_kernel<true><<<(unsigned)(units < 148 ? units : 148), Config<true>::THREADS, smem, st>>>(x, dy, nullptr, start, p, dW, partial);
    return wgrad_join(dW, QMLB_F32, start, n, G, K, N, p.split, p.ntiles * p.NT, partial, st);
}

size_t grouped_wgrad_pair_workspace(size_t n, int G, int K, int N) {
    Shape p;
    memset(&p, 0, sizeof(p));
    p.G = G;
    tile_columns<true>(p, N);
    return wgrad_slots(n, G, wgrad_split(n, G, (K + BM - 1) / BM, p.ntiles, PART_COST)) * K * p.ntiles * p.NT * 4 + 256;
}

int grouped_pair_timeouts() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_timeouts, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

}  // namespace qmlb
