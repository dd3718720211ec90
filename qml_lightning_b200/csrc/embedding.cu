// Table lookup with scaling, and the gradient of the table by ordered keys.
//
//   out[i, :]    = scale * table[index[i], :]                  (a zero row for an index outside the table)
//   dtable[v, :] = scale * sum over i with index[i] = v of dout[i, :]
//
// Both are bound by memory: the lookup writes n rows and reads the table rows that occur, the gradient reads n rows and
// writes the table.  The gradient walks the rows in key order (order[] from qmlb_group_by_key), so every table row is a
// sum over consecutive positions and no atomic is needed: the result does not depend on scheduling.  Sums are 32-bit.
//
// Work split of the gradient: positions are cut into blocks of equal size whatever the keys are, because one key may hold
// most positions (3 elements, 210,000 atoms) or almost none (a large vocabulary).  Inside a block R row groups of TC
// column threads walk equal runs of positions.  A key whose positions lie inside one run is written by it; the pieces of
// the others meet in shared memory, and what crosses a block's border goes to scratch as at most two pieces per block (the
// head, of a key begun before, and the tail, of a key that goes on), which a second kernel adds in block order.
#include "typed.cuh"

namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ int64_t index_at(const void *index, int bits, size_t i) {
    return bits == 32 ? (int64_t) reinterpret_cast<const int32_t *>(index)[i] : reinterpret_cast<const int64_t *>(index)[i];
}

// one access of VEC elements per thread and step; `chunks` accesses per row
template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS)
lookup_kernel(const void *__restrict__ index, int bits, const T *__restrict__ table, size_t n, int64_t rows, int chunks, float scale,
              T *__restrict__ out) {
    const size_t total = n * (size_t)chunks;
    const size_t step = (size_t)gridDim.x * THREADS;
    for (size_t t = (size_t)blockIdx.x * THREADS + threadIdx.x; t < total; t += step) {
        const size_t i = t / (unsigned)chunks;
        const int c = (int)(t - i * (unsigned)chunks);
        const int64_t v = index_at(index, bits, i);
        float x[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) x[q] = 0.f;
        if (v >= 0 && v < rows) {
            qmlb::load_f32<T, VEC>(table + ((size_t)v * chunks + c) * VEC, x);
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[q] *= scale;
        }
        qmlb::store_f32<T, VEC>(out + t * VEC, x);
    }
}

// Rows that accesses of 8 bytes cannot follow: the result is written flat, 16 bytes per thread (they end in the next row at most, for
// widths of at least UNITS elements), and read element by element.  200,000 rows of 301 float32: 86 us, with single elements 141;
// 100,000 rows of 1,001 fp16: 109 against 256; 300,000 of 17: 12 against 20.  Where 8 bytes can follow the rows they are faster (50,000
// rows of 1,028 bf16: 51 against 59 us; of 1,026 float32 88 against 80).
template <typename T, int UNITS>
__global__ void __launch_bounds__(THREADS)
lookup_flat_kernel(const void *__restrict__ index, int bits, const T *__restrict__ table, size_t n, int64_t rows, int width, float scale,
                   T *__restrict__ out) {
    const size_t total = n * (size_t)width, step = (size_t)gridDim.x * THREADS * UNITS;
    for (size_t e = ((size_t)blockIdx.x * THREADS + threadIdx.x) * UNITS; e < total; e += step) {
        const size_t i = e / (unsigned)width;
        const int c = (int)(e - i * (unsigned)width), here = width - c;        // elements of this row
        const int64_t v0 = index_at(index, bits, i), v1 = index_at(index, bits, i + 1 < n ? i + 1 : i);
        const bool in0 = v0 >= 0 && v0 < rows, in1 = v1 >= 0 && v1 < rows;
        const T *p0 = table + (in0 ? (size_t)v0 * width : 0) + c, *p1 = table + (in1 ? (size_t)v1 * width : 0) - here;
        T x[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) x[u] = (u < here ? p0 : p1)[u];        // a row of the table always: row 0 for an index outside
        float f[UNITS];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) f[u] = (u < here ? in0 : in1) ? qmlb::to_f32(x[u]) * scale : 0.f;
        if (e + UNITS <= total) qmlb::store_f32<T, UNITS>(out + e, f);
        else
            for (int u = 0; e + u < total; ++u) out[e + u] = qmlb::from_f32<T>(f[u]);
    }
}

// ---- gradient -----------------------------------------------------------------------------------------------------
struct GradPlan {
    int vec, chunks;          // elements per access, accesses per row
    int tc, r, run;           // column threads, row groups (tc * r <= THREADS), positions per row group
    int block;                // positions per block = r * run
    unsigned blocks, col_blocks, zero_blocks;
    size_t bytes;
};

GradPlan make_grad_plan(size_t n, int nkeys, int width, int dtype, const void *dout, const void *dtable) {
    GradPlan p;
    const int es = qmlb::dtype_size(dtype);
    p.vec = qmlb::access_bytes((size_t)width * es, es, dout, dtable) / es;
    p.chunks = width / p.vec;
    // all accesses of a row in one block where 128 threads suffice, in equal parts otherwise
    p.col_blocks = (unsigned)((p.chunks + 127) / 128);
    p.tc = (p.chunks + (int)p.col_blocks - 1) / (int)p.col_blocks;
    p.r = THREADS / p.tc;
    // runs long enough that the pieces stay few and all blocks run at once, short enough that there is a block for every SM
    p.run = 8;
    while (p.run < 128 && p.r * p.run < 2048 && n / ((size_t)p.r * p.run) * p.col_blocks > 148 * 4) p.run <<= 1;
    p.block = p.r * p.run;
    p.blocks = (unsigned)((n + p.block - 1) / p.block);
    // rows of keys that do not occur are zeroed by blocks of their own
    const size_t table_blocks = ((size_t)nkeys + p.r * 16 - 1) / (p.r * 16);
    p.zero_blocks = (unsigned)(table_blocks < 148 * 8 ? table_blocks : 148 * 8);
    // per block: key of the tail, then head and tail pieces
    p.bytes = (((size_t)p.blocks * 4 + 255) & ~(size_t)255) + (size_t)p.blocks * 2 * width * 4 + 512;
    return p;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_scaled(T *p, const float (&v)[VEC], float scale) {
    float s[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) s[q] = v[q] * scale;
    qmlb::store_f32<T, VEC>(p, s);
}

// Dynamic shared memory: order int[block], key int[block + 2] (keys of the positions, with the neighbours of the block at
// both ends), then pieces float[r][2][tc * VEC].
template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS)
grad_kernel(const T *__restrict__ dout, const void *__restrict__ index, int bits, const int *__restrict__ order,
            const int *__restrict__ start, unsigned n, int nkeys, int chunks, int tc, int run, unsigned blocks, float scale, T *__restrict__ dtable,
            int *__restrict__ tail_key, float *__restrict__ pieces) {
    extern __shared__ int sm[];
    const int r = THREADS / tc, block = r * run, width = chunks * VEC;
    int *ord = sm, *key = sm + block + 1;                  // key[-1] .. key[block]
    float *piece = reinterpret_cast<float *>(sm + ((2 * block + 2 + 3) & ~3));
    const size_t p0 = (size_t)blockIdx.x * block;
    const int col = blockIdx.y * tc + threadIdx.x % tc;    // access within the row
    const int g = threadIdx.x / tc;
    if (blockIdx.x >= blocks) {                            // zero rows of keys without positions
        if (g >= r || col >= chunks) return;
        float z[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) z[q] = 0.f;
        const int64_t step = (int64_t)(gridDim.x - blocks) * r;
        for (int64_t v = (int64_t)(blockIdx.x - blocks) * r + g; v < nkeys; v += 4 * step) {
            bool empty[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {                  // addresses are clamped instead of tested: all loads are in flight together
                const int64_t at = v + i * step < nkeys ? v + i * step : nkeys - 1;
                empty[i] = start[at] == start[at + 1];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v + i * step < nkeys && empty[i]) qmlb::store_f32<T, VEC>(dtable + ((size_t)(v + i * step) * chunks + col) * VEC, z);
        }
        return;
    }
    // keys of the positions p0 - 1 .. p0 + block; a position without a valid row has key -1 and adds nothing
    for (int i0 = (int)threadIdx.x - 1; i0 <= block; i0 += 4 * THREADS) {
        int o[4], k[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t p = (int64_t)p0 + i0 + u * THREADS;
            o[u] = order[p < 0 ? 0 : p < (int64_t)n ? p : (int64_t)n - 1];
            if (p < 0 || p >= (int64_t)n || o[u] < 0 || (unsigned)o[u] >= n) o[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t v = index_at(index, bits, (size_t)max(o[u], 0));
            k[u] = o[u] >= 0 && v >= 0 && v < nkeys ? (int)v : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * THREADS;
            if (i >= 0 && i < block) ord[i] = max(o[u], 0);
            if (i <= block) key[i] = k[u];
        }
    }
    __syncthreads();
    const bool mine = g < r, active = mine && col < chunks;         // threads beyond r * tc only fetch keys
    const int a = mine ? g * run : 0, b = mine ? a + run : 0;
    float acc[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
    // the piece of a key that began before this run is the head, one that goes on behind it the tail; a key that covers the
    // whole run is its head
    float *head = piece + ((size_t)(g * 2) * tc + threadIdx.x % tc) * VEC, *tail = head + (size_t)tc * VEC;
    bool from_before = key[a - 1] == key[a];
    constexpr int U = 8;
    for (int i = a; i < b; i += U) {
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            qmlb::load_f32<T, VEC>(dout + ((size_t)ord[i + u] * chunks + (active ? col : 0)) * VEC, x[u]);      // always: see above
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = key[i + u];
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += k >= 0 ? x[u][q] : 0.f;
            const bool ends = key[i + u + 1] != k, last = i + u == b - 1;
            if (k >= 0 && (ends || last)) {
                if (ends && !from_before) {
                    if (active) store_scaled<T, VEC>(dtable + ((size_t)k * chunks + col) * VEC, acc, scale);
                } else {
                    float *to = from_before ? head : tail;
#pragma unroll
                    for (int q = 0; q < VEC; ++q) to[q] = acc[q];
                }
            }
            if (ends) {
                from_before = false;
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
            }
        }
    }
    __syncthreads();
    // join the pieces of the block: the group whose run holds the beginning of a key (or group 0, for the key that began
    // before the block) adds the heads that follow
    if (!mine) return;
    const int ka = key[a], kb = key[b - 1];
    const bool whole = ka == kb;                                    // one key fills the run
    const bool opens = kb >= 0 && key[b] == kb && !(whole && key[a - 1] == ka);   // a key begins here and goes on
    float *block_head = pieces + (size_t)blockIdx.x * 2 * width + (size_t)col * VEC, *block_tail = block_head + width;
    if (g == 0 && ka >= 0 && key[-1] == ka) {
        float s[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) s[q] = head[q];
        for (int j = 1; j < r && key[j * run] == ka && key[j * run - 1] == ka; ++j) {
            const float *h = head + (size_t)j * 2 * tc * VEC;
#pragma unroll
            for (int q = 0; q < VEC; ++q) s[q] += h[q];
        }
        if (active) {
#pragma unroll
            for (int q = 0; q < VEC; ++q) block_head[q] = s[q];
        }
    }
    int my_tail = -1;
    if (opens) {
        float s[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) s[q] = tail[q];
        int j = g + 1;
        for (; j < r && key[j * run] == kb; ++j) {
            const float *h = head + (size_t)(j - g) * 2 * tc * VEC;
#pragma unroll
            for (int q = 0; q < VEC; ++q) s[q] += h[q];
        }
        const bool leaves = key[block - 1] == kb && key[block] == kb;      // goes on behind the block
        if (leaves) {
            my_tail = kb;
            if (active) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) block_tail[q] = s[q];
            }
        } else if (active) {
            store_scaled<T, VEC>(dtable + ((size_t)kb * chunks + col) * VEC, s, scale);
        }
        if (leaves && blockIdx.y == 0 && threadIdx.x % tc == 0) tail_key[blockIdx.x] = my_tail;
    }
    // no key leaves this block, or the one that does began before it
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        const int k = key[block - 1];
        const bool leaves = k >= 0 && key[block] == k;
        if (!leaves || (key[0] == k && key[-1] == k)) tail_key[blockIdx.x] = -1;
    }
}

// Keys that cross block borders: block b whose tail opens such a key adds the heads of the blocks behind it, in an order that
// depends on their number alone.  Few pieces: every thread adds its columns.  Many (one key may hold most positions): JOIN_LANES
// row lanes of 32 column threads take every JOIN_LANES-th piece, and blockIdx.y shares the columns.
constexpr int JOIN_LANES = 16, JOIN_THREADS = 32 * JOIN_LANES;
template <typename T, int VEC>
__global__ void __launch_bounds__(JOIN_THREADS)
join_kernel(const int *__restrict__ tail_key, const float *__restrict__ pieces, const int *__restrict__ start, unsigned blocks, int block,
            int width, float scale, T *__restrict__ dtable) {
    __shared__ float part[JOIN_LANES][32 * VEC];
    const unsigned b = blockIdx.x;
    const int k = tail_key[b];
    if (k < 0) return;
    const int end = start[k + 1];                                   // one past the key's last position
    unsigned last = end > 0 ? (unsigned)(end - 1) / (unsigned)block : 0u;
    if (last >= blocks) last = blocks - 1;
    auto load = [&](unsigned j, int c, float (&v)[VEC]) { qmlb::load_f32<float, VEC>(pieces + ((size_t)j * 2 + (j == b)) * width + c, v); };
    auto store = [&](int c, const float (&s)[VEC]) {
#pragma unroll
        for (int q = 0; q < VEC; ++q) dtable[(size_t)k * width + c + q] = qmlb::from_f32<T>(s[q] * scale);
    };
    if (last < b + JOIN_LANES) {
        if (blockIdx.y) return;
        for (int c = (int)threadIdx.x * VEC; c < width; c += JOIN_THREADS * VEC) {
            float s[VEC], v[4][VEC];
            load(b, c, s);
            for (unsigned j = b + 1; j <= last; j += 4) {        // addresses are clamped instead of tested: the loads are in flight together
#pragma unroll
                for (unsigned u = 0; u < 4; ++u) load(min(j + u, last), c, v[u]);
#pragma unroll
                for (unsigned u = 0; u < 4; ++u)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) s[q] += j + u <= last ? v[u][q] : 0.f;
            }
            store(c, s);
        }
        return;
    }
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int c0 = blockIdx.y * 32 * VEC; c0 < width; c0 += gridDim.y * 32 * VEC) {
        const int c = c0 + lane * VEC;
        float s[VEC], v[8][VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) s[q] = 0.f;
        if (c < width) {
            for (unsigned j = b + (unsigned)w; j <= last; j += 8 * JOIN_LANES) {
#pragma unroll
                for (unsigned u = 0; u < 8; ++u) load(min(j + u * JOIN_LANES, last), c, v[u]);
#pragma unroll
                for (unsigned u = 0; u < 8; ++u)
#pragma unroll
                    for (int q = 0; q < VEC; ++q) s[q] += j + u * JOIN_LANES <= last ? v[u][q] : 0.f;
            }
        }
#pragma unroll
        for (int q = 0; q < VEC; ++q) part[w][lane * VEC + q] = s[q];
        __syncthreads();
        for (int i = threadIdx.x; i < 32 * VEC; i += JOIN_THREADS) {
            float t = 0.f;
#pragma unroll
            for (int q = 0; q < JOIN_LANES; ++q) t += part[q][i];
            if (c0 + i < width) dtable[(size_t)k * width + c0 + i] = qmlb::from_f32<T>(t * scale);
        }
        __syncthreads();
    }
}

template <typename T, int VEC>
int run_lookup(const void *index, int bits, const T *table, size_t n, int64_t rows, int width, float scale, T *out, cudaStream_t st) {
    const int chunks = width / VEC;
    const size_t need = (n * (size_t)chunks + THREADS - 1) / THREADS;
    const unsigned blocks = (unsigned)(need < 148 * 64 ? need : 148 * 64);
    lookup_kernel<T, VEC><<<blocks, THREADS, 0, st>>>(index, bits, table, n, rows, chunks, scale, out);
    return qmlb::check_launch("qmlb_embedding");
}

template <typename T>
int lookup_typed(const void *index, int bits, const void *table, size_t n, int64_t rows, int width, float scale, void *out, cudaStream_t st) {
    const T *t = static_cast<const T *>(table);
    T *o = static_cast<T *>(out);
    const int access = qmlb::access_bytes((size_t)width * sizeof(T), sizeof(T), table, out);
    constexpr int UNITS = 16 / (int)sizeof(T);
    if (access < 8 && width >= UNITS && ((uintptr_t)out & 15) == 0 && rows > 0) {          // rows: an index outside reads row 0
        const size_t need = (n * (size_t)width + THREADS * UNITS - 1) / (THREADS * UNITS);
        lookup_flat_kernel<T, UNITS><<<(unsigned)(need < 148 * 64 ? need : 148 * 64), THREADS, 0, st>>>(index, bits, t, n, rows, width, scale, o);
        return qmlb::check_launch("qmlb_embedding");
    }
    switch (access) {
        case 16: return run_lookup<T, 16 / (int)sizeof(T)>(index, bits, t, n, rows, width, scale, o, st);
        case 8: return run_lookup<T, 8 / (int)sizeof(T)>(index, bits, t, n, rows, width, scale, o, st);
        case 4: return run_lookup<T, 4 / (int)sizeof(T)>(index, bits, t, n, rows, width, scale, o, st);
        default: return run_lookup<T, 1>(index, bits, t, n, rows, width, scale, o, st);
    }
}

template <typename T, int VEC>
int run_grad(const GradPlan &p, const T *dout, const void *index, int bits, const int *order, const int *start, size_t n, int nkeys, int width,
             float scale, T *dtable, unsigned char *scratch, cudaStream_t st) {
    int *tail_key = reinterpret_cast<int *>(scratch);
    float *pieces = reinterpret_cast<float *>(scratch + (((size_t)p.blocks * 4 + 255) & ~(size_t)255));
    const size_t smem = (size_t)((2 * p.block + 2 + 3) & ~3) * 4 + (size_t)p.r * 2 * p.tc * VEC * 4;
    dim3 grid(p.blocks + p.zero_blocks, p.col_blocks);
    if (int rc = qmlb::ensure_smem(grad_kernel<T, VEC>, smem, "qmlb_embedding_grad")) return rc;
    grad_kernel<T, VEC><<<grid, THREADS, smem, st>>>(dout, index, bits, order, start, (unsigned)n, nkeys, p.chunks, p.tc, p.run, p.blocks, scale, dtable,
                                                    tail_key, pieces);
    if (p.blocks > 1) {
        const bool wide = (width & 3) == 0;
        const unsigned cb = (unsigned)((width + (wide ? 127 : 31)) / (wide ? 128 : 32));
        const dim3 jg(p.blocks - 1, cb < 4 ? cb : 4);
        if (wide) join_kernel<T, 4><<<jg, JOIN_THREADS, 0, st>>>(tail_key, pieces, start, p.blocks, p.block, width, scale, dtable);
        else join_kernel<T, 1><<<jg, JOIN_THREADS, 0, st>>>(tail_key, pieces, start, p.blocks, p.block, width, scale, dtable);
    }
    return qmlb::check_launch("qmlb_embedding_grad");
}

template <typename T>
int grad_typed(const GradPlan &p, const void *dout, const void *index, int bits, const int *order, const int *start, size_t n, int nkeys,
               int width, float scale, void *dtable, unsigned char *scratch, cudaStream_t st) {
    const T *d = static_cast<const T *>(dout);
    T *t = static_cast<T *>(dtable);
    switch (p.vec * (int)sizeof(T)) {
        case 16: return run_grad<T, 16 / (int)sizeof(T)>(p, d, index, bits, order, start, n, nkeys, width, scale, t, scratch, st);
        case 8: return run_grad<T, 8 / (int)sizeof(T)>(p, d, index, bits, order, start, n, nkeys, width, scale, t, scratch, st);
        case 4: return run_grad<T, 4 / (int)sizeof(T)>(p, d, index, bits, order, start, n, nkeys, width, scale, t, scratch, st);
        default: return run_grad<T, 1>(p, d, index, bits, order, start, n, nkeys, width, scale, t, scratch, st);
    }
}

}  // namespace

extern "C" int qmlb_embedding(const void *index, int index_bits, const void *table, int dtype, size_t n, int64_t rows, int width, float scale,
                              void *out, qmlb_stream_t stream) {
    QMLB_REQUIRE((index && out) || n == 0, "qmlb_embedding: null tensor");
    QMLB_REQUIRE(table || rows == 0, "qmlb_embedding: null table");
    QMLB_REQUIRE(index_bits == 32 || index_bits == 64, "qmlb_embedding: indices must have 32 or 64 bits");
    QMLB_REQUIRE(qmlb::dtype_size(dtype) != 0, "qmlb_embedding: unknown element type %d", dtype);
    QMLB_REQUIRE(width > 0 && rows >= 0, "qmlb_embedding: bad sizes");
    if (n == 0) return QMLB_OK;
    cudaStream_t st = qmlb::as_stream(stream);
    if (dtype == QMLB_F32) return lookup_typed<float>(index, index_bits, table, n, rows, width, scale, out, st);
    if (dtype == QMLB_F16) return lookup_typed<__half>(index, index_bits, table, n, rows, width, scale, out, st);
    return lookup_typed<__nv_bfloat16>(index, index_bits, table, n, rows, width, scale, out, st);
}

extern "C" size_t qmlb_embedding_grad_scratch_bytes(size_t n, int rows, int width) {
    if (n == 0 || n >= (size_t)1 << 31 || rows <= 0 || width <= 0) return 256;
    // the widest need over the access widths that the pointers may allow
    size_t most = 0;
    for (int dtype = QMLB_F32; dtype <= QMLB_BF16; ++dtype)
        for (uintptr_t at = 1; at <= 16; at <<= 1) {
            const size_t b = make_grad_plan(n, rows, width, dtype, reinterpret_cast<const void *>(at), nullptr).bytes;
            if (b > most) most = b;
        }
    return most;
}

extern "C" int qmlb_embedding_grad(const void *dout, int dtype, const void *index, int index_bits, const int *order, const int *group_start,
                                   size_t n, int rows, int width, float scale, void *dtable, void *scratch, size_t scratch_bytes,
                                   qmlb_stream_t stream) {
    QMLB_REQUIRE(dtable && group_start && ((dout && index && order && scratch) || n == 0), "qmlb_embedding_grad: null tensor");
    QMLB_REQUIRE(index_bits == 32 || index_bits == 64, "qmlb_embedding_grad: indices must have 32 or 64 bits");
    const int es = qmlb::dtype_size(dtype);
    QMLB_REQUIRE(es != 0, "qmlb_embedding_grad: unknown element type %d", dtype);
    QMLB_REQUIRE(rows > 0 && rows < INT32_MAX && width > 0 && n < (size_t)1 << 31, "qmlb_embedding_grad: bad sizes");
    cudaStream_t st = qmlb::as_stream(stream);
    if (n == 0) {
        if (cudaMemsetAsync(dtable, 0, (size_t)rows * width * es, st) != cudaSuccess) return qmlb::check_launch("qmlb_embedding_grad(memset)");
        return QMLB_OK;
    }
    const GradPlan p = make_grad_plan(n, rows, width, dtype, dout, dtable);
    QMLB_REQUIRE(scratch_bytes >= p.bytes, "qmlb_embedding_grad: scratch too small");
    QMLB_REQUIRE(((uintptr_t)scratch & 15) == 0, "qmlb_embedding_grad: scratch must be 16-byte aligned");
    unsigned char *sc = static_cast<unsigned char *>(scratch);
    if (dtype == QMLB_F32) return grad_typed<float>(p, dout, index, index_bits, order, group_start, n, rows, width, scale, dtable, sc, st);
    if (dtype == QMLB_F16) return grad_typed<__half>(p, dout, index, index_bits, order, group_start, n, rows, width, scale, dtable, sc, st);
    return grad_typed<__nv_bfloat16>(p, dout, index, index_bits, order, group_start, n, rows, width, scale, dtable, sc, st);
}
