// Device helpers shared by the tensor-core kernels of the grouped products: group lookup, the epilogue's padded tile, and
// loads of rows that TMA cannot follow.
#pragma once

#include "tcgen.cuh"
#include "typed.cuh"

namespace qmlb {
namespace tc {

constexpr int BK = 64;                           // depth per stage: one 128-byte line of 16-bit elements
constexpr int MAX_STAGES = 8;
constexpr int EPI_WARPS = 8;                     // warps that drain an accumulator: two per quarter of its rows
constexpr int EPI_TILE = 2048;                   // a warp's epilogue tile: 32 rows of 64 bytes
constexpr uint32_t EPI_BYTES = EPI_WARPS * EPI_TILE;
constexpr uint32_t TMEM_COLS = 512, BUF_COLS = 256;
constexpr size_t SMEM_LIMIT = 227 * 1024;

struct Groups {              // in shared memory
    int *start;              // [G + 1] clamped bounds
    int *parts;              // [G + 1] parts (row tiles, or splits of the sum) before group g
    int *split;              // null, or [G + 1]: parts before group g that belong to groups of several parts
    __device__ __forceinline__ int rows(int g) const { return max(start[g + 1] - start[g], 0); }
    // group that holds part `i`
    __device__ __forceinline__ int find(int G, int i) const {
        int lo = 0, hi = G - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (parts[mid] <= i) lo = mid; else hi = mid - 1;
        }
        return lo;
    }
};

// Fill `start` (all threads) and `parts` (warp 0): a group of r rows has ceil(r / part_rows) parts.  Bounds that descend, which
// no caller should pass, are raised to the largest before them: the groups never hold more than n rows, for which tiles and
// scratch were counted.  Ends with a barrier.
__device__ __forceinline__ void read_groups(const Groups &s, const int *__restrict__ start, int G, int n, int part_rows) {
    for (int g = threadIdx.x; g <= G; g += blockDim.x) s.start[g] = min(max(start[g], 0), n);
    __syncthreads();
    bool down = false;
    for (int g = threadIdx.x; g < G; g += blockDim.x) down |= s.start[g + 1] < s.start[g];
    if (__syncthreads_or(down)) {
        if (threadIdx.x == 0)
            for (int g = 0; g < G; ++g) s.start[g + 1] = max(s.start[g + 1], s.start[g]);
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        for (int pass = 0; pass < (s.split ? 2 : 1); ++pass) {
            int *to = pass ? s.split : s.parts;
            int before = 0;
            for (int g0 = 0; g0 < G; g0 += 32) {
                const int g = g0 + lane;
                int t = g < G ? (s.rows(g) + part_rows - 1) / part_rows : 0;
                if (pass && t == 1) t = 0;
                int inc = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(QMLB_FULL_MASK, inc, o);
                    if (lane >= o) inc += v;
                }
                if (g < G) to[g] = before + inc - t;
                before += __shfl_sync(QMLB_FULL_MASK, inc, 31);
            }
            if (lane == 0) to[G] = before;
        }
    }
    __syncthreads();
}

// Predicated global stores: without a branch the loads in front of them are issued together.
__device__ __forceinline__ void store_if(void *p, uint4 v, bool wanted) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p st.global.v4.b32 [%0], {%1, %2, %3, %4};\n\t}" ::"l"(__cvta_generic_to_global(p)),
                 "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"((int)wanted)
                 : "memory");
}
__device__ __forceinline__ void store_if(void *p, uint2 v, bool wanted) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t@p st.global.v2.b32 [%0], {%1, %2};\n\t}" ::"l"(__cvta_generic_to_global(p)), "r"(v.x),
                 "r"(v.y), "r"((int)wanted)
                 : "memory");
}
__device__ __forceinline__ void store_if(void *p, uint32_t v, bool wanted) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.global.b32 [%0], %1;\n\t}" ::"l"(__cvta_generic_to_global(p)), "r"(v), "r"((int)wanted)
                 : "memory");
}
__device__ __forceinline__ void store_if(void *p, uint16_t v, bool wanted) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.global.b16 [%0], %1;\n\t}" ::"l"(__cvta_generic_to_global(p)), "h"(v), "r"((int)wanted)
                 : "memory");
}

// Zeros into the matrices [K][row_bytes] of the groups without rows, by warp `i` of `count`; a row is a multiple of `access` bytes.
__device__ __forceinline__ void zero_empty_groups(const Groups &s, int G, unsigned char *out, size_t matrix_bytes, int access, int i, int count, int lane) {
    const size_t first = (size_t)i * 32 + lane, step = (size_t)count * 32;
    for (int g = 0; g < G; ++g) {
        if (s.parts[g + 1] != s.parts[g]) continue;
        unsigned char *to = out + (size_t)g * matrix_bytes;
        if (access == 16)
            for (size_t k = first; k < matrix_bytes / 16; k += step) reinterpret_cast<uint4 *>(to)[k] = make_uint4(0, 0, 0, 0);
        else if (access >= 4)
            for (size_t k = first; k < matrix_bytes / 4; k += step) reinterpret_cast<uint32_t *>(to)[k] = 0;
        else
            for (size_t k = first; k < matrix_bytes / 2; k += step) reinterpret_cast<uint16_t *>(to)[k] = 0;
    }
}

// Byte `c` of row `r` in a warp's epilogue tile: 16-byte pieces in an order that changes every two rows, so that neither the
// writes by rows nor the reads along rows collide in the banks.
__device__ __forceinline__ int tile_at(int r, int c) { return r * 64 + (((c >> 4) ^ ((r >> 1) & 3)) << 4) + (c & 15); }

// Store one warp's tile (32 rows of up to 64 bytes) from shared memory, W bytes per access.
template <int W>
__device__ __forceinline__ void store_rows(const unsigned char *tile, unsigned char *out, size_t row_bytes, int rows, int bytes, int lane) {
    constexpr int LANES = 64 / W, ROWS = 32 / LANES, BATCH = 32 / ROWS < 8 ? 32 / ROWS : 8;      // lanes per row, rows per access
    using V = typename Word<W>::type;
    const int r0 = lane / LANES, c = (lane % LANES) * W;
    unsigned char *to = out + (size_t)r0 * row_bytes + c;
#pragma unroll 1
    for (int b = 0; b < 32 / ROWS; b += BATCH) {
        V t[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) t[i] = *reinterpret_cast<const V *>(tile + tile_at(r0 + (b + i) * ROWS, c));
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            store_if(to, t[i], r0 + (b + i) * ROWS < rows && c < bytes);
            to += (size_t)ROWS * row_bytes;
        }
    }
}
__device__ __forceinline__ void store_tile(const unsigned char *tile, unsigned char *out, size_t row_bytes, int rows, int bytes, int lane, int access) {
    if (access == 16) store_rows<16>(tile, out, row_bytes, rows, bytes, lane);
    else if (access == 8) store_rows<8>(tile, out, row_bytes, rows, bytes, lane);
    else if (access == 4) store_rows<4>(tile, out, row_bytes, rows, bytes, lane);
    else store_rows<2>(tile, out, row_bytes, rows, bytes, lane);
}

// 32 accumulator columns of this thread's row, rounded to the result type, into the warp's tile
template <typename T>
__device__ __forceinline__ void stage_row(unsigned char *tile, int lane, const uint32_t (&v)[32]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        Pack<T, 8> k;
#pragma unroll
        for (int q = 0; q < 8; ++q) k.item[q] = from_f32<T>(__uint_as_float(v[u * 8 + q]));
        *reinterpret_cast<uint4 *>(tile + tile_at(lane, u * 16)) = k.word;
    }
}
// 16 of them as they are
__device__ __forceinline__ void stage_row_f32(unsigned char *tile, int lane, const uint32_t *v) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
        *reinterpret_cast<uint4 *>(tile + tile_at(lane, u * 16)) = make_uint4(v[u * 4], v[u * 4 + 1], v[u * 4 + 2], v[u * 4 + 3]);
}

// LINES lines of 128 bytes (64 elements) of consecutive rows into a swizzled box, W bytes per access (2: through registers),
// by THREADS threads.  Rows from `end` on and bytes behind the row's end become zeros.
template <int W, int LINES, int THREADS>
__device__ __forceinline__ void load_lines(const unsigned char *in, size_t row_bytes, int row0, int end, size_t byte0, uint32_t dst, int t) {
    constexpr int PER_ROW = 128 / W, ROWS = THREADS / PER_ROW;       // rows per round
    static_assert(THREADS % PER_ROW == 0 && LINES % ROWS == 0, "whole rounds");
    const int r0 = t / PER_ROW, c = (t % PER_ROW) * W;
    const bool in_row = byte0 + c < row_bytes;
    const unsigned char *src = in + (size_t)(row0 + r0) * row_bytes + byte0 + c;
#pragma unroll 8
    for (int i = 0; i < LINES / ROWS; ++i) {
        const int r = r0 + i * ROWS;
        const bool wanted = in_row && row0 + r < end;
        const uint32_t to = dst + (uint32_t)r * 128u + ((uint32_t)c ^ ((uint32_t)(r & 7) << 4));      // the 128-byte swizzle
        if (W >= 4) {
            cp_async<W >= 4 ? W : 4>(to, wanted ? src : in, wanted);
        } else {
            const uint16_t v = wanted ? *reinterpret_cast<const uint16_t *>(src) : (uint16_t)0;
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(v) : "memory");
        }
        src += (size_t)ROWS * row_bytes;
    }
}
template <int LINES, int THREADS>
__device__ __forceinline__ void load_box(const unsigned char *in, size_t row_bytes, int row0, int end, size_t byte0, uint32_t dst, int t, int access) {
    if (access >= 8) load_lines<8, LINES, THREADS>(in, row_bytes, row0, end, byte0, dst, t);
    else if (access == 4) load_lines<4, LINES, THREADS>(in, row_bytes, row0, end, byte0, dst, t);
    else load_lines<2, LINES, THREADS>(in, row_bytes, row0, end, byte0, dst, t);
}

}  // namespace tc
}  // namespace qmlb
