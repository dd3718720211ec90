// Stable order of integer keys: order[] lists the positions of the keys by ascending key, equal keys in their original
// order, and group_start[v] = number of valid keys below v.  Keys outside [0, nkeys) (the -1 of a padded slot) count as
// the key nkeys: they come behind all groups, in their original order.
//
// Least-significant-digit radix sort with digits of at most RADIX_BITS bits in separate launches, C_BITS in a cluster, so up to 1,023 keys
// (in a cluster 511; every element or species numbering) take ONE pass and 1,048,575 (262,143) take two.  A pass over blocks of 1,024
// or 2,048 keys:
//   1. histogram : counts[digit][block]
//   2. scan      : one block per digit turns its row into an exclusive prefix over the blocks and writes the digit's total
//   3. scatter   : every block ranks its keys again (the same order, so the result never depends on scheduling) and
//                  writes position and key to base(digit) + counts[digit][block] + rank
// Rank inside a block: each warp owns a contiguous run of its keys; the lanes that hold the same digit find one another
// by ballots or a match, and the warp's running count per digit stays in shared memory.  What bounds a pass is
// latency and the scattered writes, not arithmetic: 8 + 8 bytes per key and pass.
// With one pass the digit totals are the group sizes; with more, group_start is read off the sorted keys.
// Up to CLUSTER_KEYS keys (PORTABLE_KEYS where the device runs no clusters of sixteen blocks) take one launch of one thread-block
// cluster: the same passes, with the digit totals read from the neighbours' shared memory and cluster barriers between the steps.
// (Separate launches took 20 us for one pass and 57 us for two whatever the number of keys; most of it the launches and the few
// busy SMs.)
#include <cooperative_groups.h>

#include <atomic>

#include "typed.cuh"

namespace {

constexpr int RADIX_BITS = 10;                 // widest digit
constexpr int THREADS = 256, WARPS = THREADS / 32;
// keys per thread: few while the blocks do not fill the device (3.3 million keys of 5: 27.5 us with 8, 31.6 with 16, 37 with 32)
constexpr int FEW = 4, MANY = 8;
inline int items_for(size_t n) { return n < (size_t)148 * 8 * THREADS * FEW ? FEW : MANY; }

__host__ __device__ inline int bits_for(unsigned nkeys) {   // digits of the values 0 .. nkeys (nkeys = "outside")
    int b = 1;
    while (b < 32 && (nkeys >> b)) ++b;
    return b;
}

template <typename K>
__device__ __forceinline__ uint32_t clamp_key(K k, uint32_t nkeys) {
    return (k >= 0 && (unsigned long long)k < (unsigned long long)nkeys) ? (uint32_t)k : nkeys;
}

// lanes that hold the same digit as mine (all lanes of the warp take part; lanes with `in` = false match nobody that has it
// true).  Few digits: one match instruction, whose time grows with the number of distinct values; many: one ballot per bit.
__device__ __forceinline__ unsigned same_digit(uint32_t d, int nbits, bool in) {
    if (nbits <= 4) return __match_any_sync(QMLB_FULL_MASK, in ? d : 0xffffffffu);
    unsigned m = __ballot_sync(QMLB_FULL_MASK, in);
    if (!in) m = ~m;
#pragma unroll
    for (int b = 0; b < RADIX_BITS; ++b) {
        if (b >= nbits) break;
        const bool one = (d >> b) & 1u;
        const unsigned v = __ballot_sync(QMLB_FULL_MASK, one);
        m &= one ? v : ~v;
    }
    return m;
}

// Long runs of keys that do not occur have one start, which the warp that finds the run stores 512 bytes at a time (at most 20 us).
// From FAR_KEYS keys on it leaves the whole segments of SEGMENT keys in the run to gap_kernel, a launch of 4 to 6 us.  (All keys equal:
// 131,072 keys of 300,000: 451 -> 69 us, 300,000 of 2,000,000: 2,830 -> 57 us, against 32 starts at a time.)
constexpr uint32_t SEGMENT = 4096, FAR_KEYS = 524288, LONG_RUN = 256;

// group_start[from .. end - 1] = value, by a warp, 16 bytes per lane
__device__ __forceinline__ void fill_run(int *__restrict__ group_start, uint32_t from, uint32_t end, int value) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t head = min(end, from + (uint32_t)(((16 - ((uintptr_t)(group_start + from) & 15)) & 15) / 4));
    if (from + lane < head) group_start[from + lane] = value;
    const uint32_t words = (end - head) / 4;
    int4 *to4 = reinterpret_cast<int4 *>(group_start + head);
    for (uint32_t i = lane; i < words; i += 32) to4[i] = make_int4(value, value, value, value);
    if (head + words * 4 + lane < end) group_start[head + words * 4 + lane] = value;
}

// group_start[v] = first position whose sorted key is not below v, for the v that the 32 positions p0 .. p0 + 31 answer: those
// above the key in front of them and not above their last one (positions behind the end count as the key nkeys).  `key`: the key
// of position p0 + lane, `front`: the key of position p0 - 1, or -1.  All lanes of the warp take part; writes are whole lines.
__device__ __forceinline__ void write_starts(uint32_t key, int64_t front, uint32_t p0, uint32_t nkeys, int *__restrict__ group_start) {
    const uint32_t last = __shfl_sync(QMLB_FULL_MASK, key, 31);
    for (int64_t v0 = front + 1; v0 <= (int64_t)last; v0 += 32) {
        const uint32_t v = (uint32_t)v0 + (threadIdx.x & 31);
        int below = 0;                                           // lanes with a smaller key
#pragma unroll
        for (int step = 16; step; step >>= 1)
            if (__shfl_sync(QMLB_FULL_MASK, key, below + step - 1) < v) below += step;
        const int first = __shfl_sync(QMLB_FULL_MASK, below, 0);
        const uint32_t end = __shfl_sync(QMLB_FULL_MASK, key, first);          // of the run of absent keys that v0 lies in
        if (end - (uint32_t)v0 >= LONG_RUN) {
            uint32_t from = (uint32_t)v0, to = end + 1;
            const uint32_t a = (from + SEGMENT - 1) / SEGMENT * SEGMENT, b = to / SEGMENT * SEGMENT;
            const bool parts = nkeys >= FAR_KEYS && a < b;       // [from, a) and [b, to)
            if (parts) to = a;
#pragma unroll 1
            for (int i = 0; i < (parts ? 2 : 1); ++i, from = b, to = end + 1)
                if (from < to) fill_run(group_start, from, to, (int)(p0 + first));
            v0 = (int64_t)end + 1 - 32;
            continue;
        }
        if (v <= last) group_start[v] = (int)(p0 + below);
    }
}

// first position whose sorted key is not below v, by a warp: 32 probes at a time
__device__ __forceinline__ uint32_t warp_lower_bound(const uint32_t *__restrict__ sorted, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t lane = threadIdx.x & 31, at = lo + (uint32_t)(((uint64_t)(hi - lo) * lane) >> 5);
        const int below = __popc(__ballot_sync(QMLB_FULL_MASK, sorted[at] < v));
        if (below == 0) break;
        const uint32_t next = __shfl_sync(QMLB_FULL_MASK, at, below & 31);
        lo = __shfl_sync(QMLB_FULL_MASK, at, below - 1) + 1;
        if (below < 32) hi = next;
    }
    return lo;
}

// FIRST: keys come from the caller's tensor; else from the pairs of the previous pass
template <typename K, bool FIRST, int ITEMS>
__global__ void __launch_bounds__(THREADS)
histogram_kernel(const K *__restrict__ keys, const uint32_t *__restrict__ pair_keys, uint32_t n, uint32_t nkeys, int shift, int nbits,
                 uint32_t *__restrict__ counts) {
    extern __shared__ uint32_t hist[];
    const int nd = 1 << nbits;
    for (int d = threadIdx.x; d < nd; d += THREADS) hist[d] = 0;
    __syncthreads();
    const uint32_t base = blockIdx.x * (uint32_t)(THREADS * ITEMS);
    uint32_t key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {                // addresses are clamped instead of tested: all loads are in flight together
        const uint32_t in = min(base + i * THREADS + threadIdx.x, n - 1);
        key[i] = FIRST ? clamp_key(keys[in], nkeys) : pair_keys[in];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool in = base + i * THREADS + threadIdx.x < n;
        const uint32_t d = (key[i] >> shift) & (uint32_t)(nd - 1);
        // few distinct digits: one shared-memory add per distinct digit and warp instead of 32 colliding ones
        const unsigned m = same_digit(d, nbits, in);
        if (in && (threadIdx.x & 31) == __ffs(m) - 1) atomicAdd(&hist[d], (uint32_t)__popc(m));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < nd; d += THREADS) counts[(size_t)d * gridDim.x + blockIdx.x] = hist[d];
}

// exclusive prefix of a value over the block's threads; total in *sum
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *warp_sums, uint32_t *sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(QMLB_FULL_MASK, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    const uint32_t own = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;      // every warp adds the warps' sums up
    uint32_t upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(QMLB_FULL_MASK, upto, o);
        if (lane >= o) upto += t;
    }
    *sum = __shfl_sync(QMLB_FULL_MASK, upto, 31);
    return __shfl_sync(QMLB_FULL_MASK, upto - own, warp) + inc - v;
}

constexpr int SCAN_THREADS = 1024;
__global__ void __launch_bounds__(SCAN_THREADS)
scan_kernel(uint32_t *__restrict__ counts, uint32_t nblocks, uint32_t *__restrict__ totals) {
    __shared__ uint32_t warp_sums[SCAN_THREADS / 32];
    uint32_t *row = counts + (size_t)blockIdx.x * nblocks;
    uint32_t carry = 0;
    for (uint32_t b = 0; b < nblocks; b += SCAN_THREADS) {
        const uint32_t at = b + threadIdx.x;
        const uint32_t v = at < nblocks ? row[at] : 0;
        uint32_t sum;
        const uint32_t ex = block_prefix(v, warp_sums, &sum);
        if (at < nblocks) row[at] = carry + ex;
        carry += sum;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// LAST: writes order[] (and, when START, group_start from the digit totals: one-pass sorts)
template <typename K, bool FIRST, bool LAST, int ITEMS>
__global__ void __launch_bounds__(THREADS)
scatter_kernel(const K *__restrict__ keys, const uint32_t *__restrict__ pair_keys, const uint32_t *__restrict__ pair_pos, uint32_t n,
               uint32_t nkeys, int shift, int nbits, const uint32_t *__restrict__ counts, const uint32_t *__restrict__ totals,
               uint32_t *__restrict__ out_keys, uint32_t *__restrict__ out_pos, int *__restrict__ group_start) {
    extern __shared__ uint32_t sm[];           // [nd] digit bases, then [WARPS][nd] running counts
    __shared__ uint32_t warp_sums[WARPS];
    const int nd = 1 << nbits;
    uint32_t *base = sm, *run = sm + nd;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < WARPS * nd; i += THREADS) run[i] = 0;
    // digit bases: exclusive prefix over the totals (every block computes the same)
    uint32_t carry = 0;
    for (int d0 = 0; d0 < nd; d0 += THREADS) {
        const int d = d0 + threadIdx.x;
        uint32_t sum;
        const uint32_t t = d < nd ? totals[d] : 0;
        const uint32_t ex = block_prefix(t, warp_sums, &sum);
        if (d < nd) base[d] = carry + ex;
        if (FIRST && LAST && blockIdx.x == 0 && d <= (int)nkeys) group_start[d] = (int)(carry + ex);
        carry += sum;
    }
    __syncthreads();
    // pass over the warp's run: digit and rank of every key
    const uint32_t w0 = blockIdx.x * (uint32_t)(THREADS * ITEMS) + warp * (uint32_t)(32 * ITEMS);
    uint32_t key[ITEMS], pos[ITEMS];
    uint16_t rank[ITEMS];
    uint32_t *mine = run + warp * nd;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const uint32_t at = w0 + i * 32 + lane, in = min(at, n - 1);
        key[i] = FIRST ? clamp_key(keys[in], nkeys) : pair_keys[in];
        pos[i] = FIRST ? at : pair_pos[in];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const bool in = w0 + i * 32 + lane < n;
        const uint32_t d = (key[i] >> shift) & (uint32_t)(nd - 1);
        const unsigned m = same_digit(d, nbits, in);
        const uint32_t before = in ? mine[d] : 0;
        __syncwarp();
        rank[i] = (uint16_t)(before + __popc(m & ((1u << lane) - 1u)));
        if (in && lane == __ffs(m) - 1) mine[d] = before + __popc(m);
        __syncwarp();
    }
    __syncthreads();
    // first place of every (warp, digit) of this block
    for (int d = threadIdx.x; d < nd; d += THREADS) {
        uint32_t at = base[d] + counts[(size_t)d * gridDim.x + blockIdx.x];
        for (int w = 0; w < WARPS; ++w) {
            const uint32_t c = run[w * nd + d];
            run[w * nd + d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (w0 + i * 32 + lane < n) {
            const uint32_t to = mine[(key[i] >> shift) & (uint32_t)(nd - 1)] + rank[i];
            out_pos[to] = pos[i];
            if (!(FIRST && LAST)) out_keys[to] = key[i];
        }
    }
}

// the same from all positions, 32 per warp
__global__ void __launch_bounds__(THREADS)
fill_kernel(const uint32_t *__restrict__ sorted, uint32_t n, uint32_t nkeys, int *__restrict__ group_start) {
    const uint32_t p0 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * 32, p = p0 + (threadIdx.x & 31);
    if (p0 > n) return;
    const uint32_t key = p < n ? sorted[p] : nkeys;
    write_starts(key, p0 == 0 ? -1 : (int64_t)sorted[p0 - 1], p0, nkeys, group_start);
}

// segments of keys of which none but the last occurs, one warp each: the others are written by the positions around them
__global__ void __launch_bounds__(THREADS)
gap_kernel(const uint32_t *__restrict__ sorted, uint32_t n, uint32_t segments, int *__restrict__ group_start) {
    for (uint32_t i = blockIdx.x * WARPS + (threadIdx.x >> 5); i < segments; i += gridDim.x * WARPS) {
        const uint32_t from = i * SEGMENT, to = from + SEGMENT - 1, start = warp_lower_bound(sorted, n, from);
        if (start == n || sorted[start] >= to) fill_run(group_start, from, to + 1, (int)start);
    }
}
void fill_gaps(const uint32_t *sorted, size_t n, int nkeys, int *group_start, cudaStream_t st) {
    if ((uint32_t)nkeys < FAR_KEYS) return;
    const uint32_t segments = ((uint32_t)nkeys + 1) / SEGMENT, blocks = (segments + WARPS - 1) / WARPS;
    gap_kernel<<<blocks < 1184 ? blocks : 1184, THREADS, 0, st>>>(sorted, (uint32_t)n, segments, group_start);
}

// the same by a search per key: many more keys than positions would leave wide gaps to few warps
__global__ void __launch_bounds__(THREADS)
start_kernel(const uint32_t *__restrict__ sorted, uint32_t n, uint32_t nkeys, int *__restrict__ group_start) {
    for (uint32_t v = blockIdx.x * THREADS + threadIdx.x; v <= nkeys; v += gridDim.x * THREADS) {
        uint32_t lo = 0, hi = n;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (sorted[mid] < v) lo = mid + 1; else hi = mid;
        }
        group_start[v] = (int)lo;
    }
}

__global__ void empty_kernel(uint32_t nkeys, int *__restrict__ group_start) {
    for (uint32_t v = blockIdx.x * THREADS + threadIdx.x; v <= nkeys; v += gridDim.x * THREADS) group_start[v] = 0;
}

// ---- one cluster ----------------------------------------------------------------------------------------------------
constexpr int C_THREADS = 1024, C_WARPS = 32, C_ITEMS = 8, C_BITS = 9, C_MAX = 16;
constexpr uint32_t CLUSTER_KEYS = C_MAX * C_THREADS * C_ITEMS, PORTABLE_KEYS = 8 * C_THREADS * C_ITEMS;      // 131,072 and 65,536

// `items` keys per thread; pairs: scratch of two buffers of n keys and two of n positions
template <typename K>
__global__ void __launch_bounds__(C_THREADS)
cluster_kernel(const K *__restrict__ keys, uint32_t n, uint32_t nkeys, int passes, int nbits, int items, int *__restrict__ order,
               int *__restrict__ group_start, uint32_t *__restrict__ pairs, uint32_t row, int fill) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ uint32_t sm[];
    __shared__ uint32_t warp_sums[C_WARPS];
    const int nd = 1 << nbits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t *totals = sm;                                       // [2][nd], read by the other blocks (two: passes take turns)
    uint32_t *base = sm + 2 * nd;                                // [nd] first place of this block's keys of a digit
    uint32_t *inside = sm + 3 * nd;                              // [nd] the same within the block
    uint16_t *run = reinterpret_cast<uint16_t *>(sm + 4 * nd);   // [C_WARPS][nd]
    // Many digits: the block's keys are first put in order here and leave in runs of one digit; scattered one by one they would
    // cost a store each on the few SMs of the cluster.
    const bool gather = nbits > 5;
    uint32_t *own_key = sm + 4 * nd + C_WARPS * nd / 2, *own_pos = own_key + C_THREADS * items;
    const int rank_of_block = (int)cluster.block_rank(), blocks = (int)cluster.num_blocks();
    const uint32_t w0 = ((uint32_t)rank_of_block * C_WARPS + warp) * (uint32_t)(32 * items);
    uint32_t *bk[2] = {pairs, pairs + row}, *bp[2] = {pairs + 2 * row, pairs + 3 * row};
    for (int pass = 0; pass < passes; ++pass) {
        const bool first = pass == 0, last = pass == passes - 1;
        const int shift = pass * nbits;
        const uint32_t *ik = bk[(pass + 1) & 1], *ip = bp[(pass + 1) & 1];
        uint32_t *ok = bk[pass & 1], *op = last ? reinterpret_cast<uint32_t *>(order) : bp[pass & 1];
        uint32_t key[C_ITEMS], pos[C_ITEMS];
        uint16_t rank[C_ITEMS];
#pragma unroll
        for (int i = 0; i < C_ITEMS; ++i) {
            // addresses are clamped instead of tested: all loads are in flight together
            const uint32_t at = w0 + i * 32 + lane, in = min(at, n - 1);
            key[i] = first ? clamp_key(keys[in], nkeys) : ik[in];
            pos[i] = first ? at : ip[in];
        }
        for (int i = threadIdx.x; i < C_WARPS * nd / 2; i += C_THREADS) reinterpret_cast<uint32_t *>(run)[i] = 0;
        __syncthreads();
        uint16_t *mine = run + warp * nd;
#pragma unroll
        for (int i = 0; i < C_ITEMS; ++i) {
            if (i < items && w0 + i * 32 < n) {                  // the same for the whole warp
                const bool in = w0 + i * 32 + lane < n;
                const uint32_t d = (key[i] >> shift) & (uint32_t)(nd - 1);
                const unsigned m = same_digit(d, nbits, in);
                const uint32_t before = in ? mine[d] : 0;
                __syncwarp();
                rank[i] = (uint16_t)(before + __popc(m & ((1u << lane) - 1u)));
                if (in && lane == __ffs(m) - 1) mine[d] = (uint16_t)(before + __popc(m));
                __syncwarp();
            }
        }
        __syncthreads();
        uint32_t *tot = totals + (pass & 1) * nd;
        if ((int)threadIdx.x < nd) {                             // warps' counts -> prefix over the warps, block total
            const int d = threadIdx.x;
            uint32_t sum = 0;
            uint16_t c[C_WARPS];
#pragma unroll
            for (int w = 0; w < C_WARPS; ++w) c[w] = run[w * nd + d];
#pragma unroll
            for (int w = 0; w < C_WARPS; ++w) {
                run[w * nd + d] = (uint16_t)sum;
                sum += c[w];
            }
            tot[d] = sum;
        }
        cluster.sync();
        uint32_t before = 0, all = 0;
        if ((int)threadIdx.x < nd)
        {
            uint32_t t[C_MAX];
#pragma unroll
            for (int q = 0; q < C_MAX; ++q) t[q] = *cluster.map_shared_rank(tot + threadIdx.x, min(q, blocks - 1));
#pragma unroll
            for (int q = 0; q < C_MAX; ++q) {
                if (q < rank_of_block) before += t[q];
                if (q < blocks) all += t[q];
            }
        }
        uint32_t whole;
        const uint32_t start = block_prefix(all, warp_sums, &whole);
        uint32_t local = 0;
        if (gather) local = block_prefix((int)threadIdx.x < nd ? tot[threadIdx.x] : 0u, warp_sums, &whole);
        if ((int)threadIdx.x < nd) {
            base[threadIdx.x] = start + before - local;          // (modulo 2^32)
            inside[threadIdx.x] = local;
            if (passes == 1 && rank_of_block == 0 && threadIdx.x <= nkeys) group_start[threadIdx.x] = (int)start;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < C_ITEMS; ++i) {
            if (i < items && w0 + i * 32 + lane < n) {
                const uint32_t d = (key[i] >> shift) & (uint32_t)(nd - 1), to = (gather ? inside[d] : base[d]) + mine[d] + rank[i];
                if (gather) {
                    own_key[to] = key[i];
                    own_pos[to] = pos[i];
                } else {
                    op[to] = pos[i];
                    if (passes > 1) ok[to] = key[i];
                }
            }
        }
        if (gather) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < whole; i += C_THREADS) {
                const uint32_t k = own_key[i], to = base[(k >> shift) & (uint32_t)(nd - 1)] + i;
                op[to] = own_pos[i];
                if (passes > 1) ok[to] = k;
            }
        }
        cluster.sync();                                          // pairs written; nobody reads a block's totals after it has left
    }
    if (!fill) return;
    // group_start[v] = first position whose key is not below v: position p writes the v above its predecessor's key
    const uint32_t *sorted = bk[(passes - 1) & 1];
    uint32_t here[C_ITEMS], left[C_ITEMS];
#pragma unroll
    for (int i = 0; i < C_ITEMS; ++i) {
        const uint32_t p0 = w0 + i * 32;
        here[i] = sorted[min(p0 + lane, n - 1)];
        left[i] = sorted[min(max(p0, 1u) - 1, n - 1)];
    }
#pragma unroll
    for (int i = 0; i < C_ITEMS; ++i) {
        const uint32_t p0 = w0 + i * 32;
        if (i < items && p0 <= n) write_starts(p0 + lane < n ? here[i] : nkeys, p0 == 0 ? -1 : (int64_t)left[i], p0, nkeys, group_start);
    }
    if (w0 + (uint32_t)(32 * items) == n) write_starts(nkeys, sorted[n - 1], n, nkeys, group_start);      // nobody's positions lie behind the end
}

// Two keys per thread, then more; sixteen blocks, where the device runs such clusters, only where ranking counts.
struct ClusterPlan {
    int passes, nbits, blocks, items;
    size_t smem;
};
ClusterPlan plan_cluster(size_t n, int nkeys, bool wide) {
    ClusterPlan p;
    const int bits = bits_for((unsigned)nkeys), most = wide && (bits > C_BITS || n > PORTABLE_KEYS) ? C_MAX : 8;
    p.passes = (bits + C_BITS - 1) / C_BITS;
    p.nbits = (bits + p.passes - 1) / p.passes;
    p.blocks = 1;
    while (p.blocks < most && (size_t)p.blocks * C_THREADS * 2 < n) p.blocks <<= 1;
    p.items = (int)((n + (size_t)p.blocks * C_THREADS - 1) / ((size_t)p.blocks * C_THREADS));
    p.smem = ((size_t)16 << p.nbits) + ((size_t)C_WARPS * 2 << p.nbits) + (p.nbits > 5 ? (size_t)8 * C_THREADS * p.items : 0);
    return p;
}

cudaLaunchConfig_t cluster_config(const ClusterPlan &p, cudaLaunchAttribute *at, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.blocks);
    cfg.blockDim = dim3(C_THREADS);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    at->id = cudaLaunchAttributeClusterDimension;
    at->val.clusterDim.x = (unsigned)p.blocks;
    at->val.clusterDim.y = at->val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cfg;
}

// Whether the current device runs clusters of sixteen blocks, which is more than every device promises; asked once per device.
template <typename K>
bool wide_clusters() {
#ifdef QMLB_TEST_NO_WIDE_CLUSTERS
    return false;                                                // for a test of the way without
#else
    constexpr int DEVICES = 64;
    static std::atomic<signed char> known[DEVICES];              // 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (dev < DEVICES)
        if (const signed char k = known[dev].load(std::memory_order_relaxed)) return k > 0;
    const ClusterPlan p = plan_cluster(CLUSTER_KEYS, (1 << C_BITS) - 1, true);       // the largest launch
    cudaLaunchAttribute at;
    const cudaLaunchConfig_t cfg = cluster_config(p, &at, nullptr);
    int clusters = 0;
    const bool yes = qmlb::ensure_smem(cluster_kernel<K>, p.smem, "qmlb_group_by_key") == QMLB_OK &&
                     cudaFuncSetAttribute(cluster_kernel<K>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                     cudaOccupancyMaxActiveClusters(&clusters, cluster_kernel<K>, &cfg) == cudaSuccess && clusters > 0;
    if (!yes) cudaGetLastError();                                // a refusal is an answer
    if (dev < DEVICES) known[dev].store(yes ? 1 : -1, std::memory_order_relaxed);
    return yes;
#endif
}

template <typename K>
int run_cluster(const ClusterPlan &p, const K *keys, size_t n, int nkeys, int *order, int *group_start, unsigned char *scratch, cudaStream_t st) {
    const int passes = p.passes;
    // many more keys than positions: the gaps are wide, and a search per key on all SMs fills them sooner
    const bool fill = passes > 1 && (size_t)nkeys <= 16 * n;
    const uint32_t row = (uint32_t)(((n * 4 + 255) & ~(size_t)255) / 4);
    uint32_t *pairs = reinterpret_cast<uint32_t *>(scratch);
    cudaLaunchAttribute at;
    const cudaLaunchConfig_t cfg = cluster_config(p, &at, st);
    if (p.blocks > 8 && cudaFuncSetAttribute(cluster_kernel<K>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return qmlb::check_launch("qmlb_group_by_key(cluster size)");
    // (1 KB more: the kernel's own variables count towards the 48 KB that need no opting in)
    if (int rc = qmlb::ensure_smem(cluster_kernel<K>, p.smem + 1024, "qmlb_group_by_key")) return rc;
    if (cudaLaunchKernelEx(&cfg, cluster_kernel<K>, keys, (uint32_t)n, (uint32_t)nkeys, passes, p.nbits, p.items, order, group_start, pairs, row,
                           (int)fill) != cudaSuccess)
        return qmlb::check_launch("qmlb_group_by_key");
    const uint32_t *sorted = pairs + ((passes - 1) & 1) * row;
    if (passes > 1 && !fill) {
        const uint32_t sb = ((uint32_t)nkeys + THREADS) / THREADS;
        start_kernel<<<sb < 1184 ? sb : 1184, THREADS, 0, st>>>(sorted, (uint32_t)n, (uint32_t)nkeys, group_start);
    }
    if (fill) fill_gaps(sorted, n, nkeys, group_start, st);
    return qmlb::check_launch("qmlb_group_by_key");
}

struct Plan {
    uint32_t blocks;
    int passes, nbits;       // digit width
    size_t counts, totals, keys, pos, bytes;      // offsets in scratch: counts, totals, two (keys, positions) pairs
};

Plan make_plan(size_t n, int nkeys) {
    Plan p;
    const int bits = bits_for((unsigned)nkeys);
    p.passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
    p.nbits = (bits + p.passes - 1) / p.passes;
    const size_t tile = (size_t)THREADS * items_for(n);
    p.blocks = (uint32_t)((n + tile - 1) / tile);
    auto round = [](size_t v) { return (v + 255) & ~(size_t)255; };
    const size_t row = round(n * 4);
    p.counts = 0;
    p.totals = round(((size_t)p.blocks << p.nbits) * 4);
    p.keys = p.totals + round((size_t)4 << p.nbits);
    // a one-pass sort needs no pairs; two passes: pair A, and the sorted keys of the last pass; more: pairs A and B
    p.pos = p.keys + (p.passes > 1 ? 2 * row : 0);
    p.bytes = p.pos + (p.passes > 2 ? 2 * row : p.passes > 1 ? row : 0);
    return p;
}

template <typename K, int ITEMS>
int run_sort(const K *keys, size_t n, int nkeys, int *order, int *group_start, unsigned char *scratch, cudaStream_t st) {
    const Plan p = make_plan(n, nkeys);
    uint32_t *counts = reinterpret_cast<uint32_t *>(scratch + p.counts), *totals = reinterpret_cast<uint32_t *>(scratch + p.totals);
    const size_t row = (n * 4 + 255) & ~(size_t)255;
    uint32_t *pk[2] = {reinterpret_cast<uint32_t *>(scratch + p.keys), reinterpret_cast<uint32_t *>(scratch + p.keys + row)};
    uint32_t *pp[2] = {reinterpret_cast<uint32_t *>(scratch + p.pos), reinterpret_cast<uint32_t *>(scratch + p.pos + row)};
    const size_t hist_smem = (size_t)4 << p.nbits, scat_smem = ((size_t)4 << p.nbits) * (1 + WARPS);
    const uint32_t un = (uint32_t)n, uk = (uint32_t)nkeys;
    uint32_t *pos_out = reinterpret_cast<uint32_t *>(order);
    for (int i = 0; i < p.passes; ++i) {
        const bool first = i == 0, last = i == p.passes - 1;
        const int shift = i * p.nbits;
        const uint32_t *ik = first ? nullptr : pk[(i - 1) & 1], *ip = first ? nullptr : pp[(i - 1) & 1];
        uint32_t *ok = pk[i & 1], *op = last ? pos_out : pp[i & 1];
        auto histogram = first ? histogram_kernel<K, true, ITEMS> : histogram_kernel<K, false, ITEMS>;
        auto scatter = first ? (last ? scatter_kernel<K, true, true, ITEMS> : scatter_kernel<K, true, false, ITEMS>)
                             : (last ? scatter_kernel<K, false, true, ITEMS> : scatter_kernel<K, false, false, ITEMS>);
        histogram<<<p.blocks, THREADS, hist_smem, st>>>(keys, ik, un, uk, shift, p.nbits, counts);
        scan_kernel<<<1 << p.nbits, SCAN_THREADS, 0, st>>>(counts, p.blocks, totals);
        scatter<<<p.blocks, THREADS, scat_smem, st>>>(keys, ik, ip, un, uk, shift, p.nbits, counts, totals, ok, op, group_start);
        if (last && !first) {
            const uint32_t sb = (uk + THREADS) / THREADS;
            if ((size_t)nkeys <= 16 * n) {
                fill_kernel<<<un / (WARPS * 32) + 1, THREADS, 0, st>>>(ok, un, uk, group_start);
                fill_gaps(ok, n, nkeys, group_start, st);
            } else start_kernel<<<sb < 1184 ? sb : 1184, THREADS, 0, st>>>(ok, un, uk, group_start);
        }
    }
    return qmlb::check_launch("qmlb_group_by_key");
}

template <typename K>
int run(const void *keys, size_t n, int nkeys, int *order, int *group_start, unsigned char *scratch, cudaStream_t st) {
    const K *k = static_cast<const K *>(keys);
    if (n <= CLUSTER_KEYS) {
        // a wide cluster has to be asked for only where one would be used
        ClusterPlan p = plan_cluster(n, nkeys, true);
        const bool wide = p.blocks <= 8 || wide_clusters<K>();
        if (!wide) p = plan_cluster(n, nkeys, false);
        if (wide || n <= PORTABLE_KEYS) return run_cluster(p, k, n, nkeys, order, group_start, scratch, st);
    }
    return items_for(n) == FEW ? run_sort<K, FEW>(k, n, nkeys, order, group_start, scratch, st)
                               : run_sort<K, MANY>(k, n, nkeys, order, group_start, scratch, st);
}

}  // namespace

extern "C" size_t qmlb_group_by_key_scratch_bytes(size_t n, int nkeys) {
    if (n == 0 || n >= (size_t)1 << 31 || nkeys <= 0 || nkeys == INT32_MAX) return 0;
    const size_t cluster = bits_for((unsigned)nkeys) <= C_BITS ? 0 : 4 * ((n * 4 + 255) & ~(size_t)255);
    if (n <= PORTABLE_KEYS) return cluster;
    const size_t launches = make_plan(n, nkeys).bytes;
    return n <= CLUSTER_KEYS && cluster > launches ? cluster : launches;
}

extern "C" int qmlb_group_by_key(const void *keys, int key_bits, size_t n, int nkeys, int *order, int *group_start, void *scratch,
                                 size_t scratch_bytes, qmlb_stream_t stream) {
    QMLB_REQUIRE(group_start && ((keys && order) || n == 0), "qmlb_group_by_key: null tensor");
    QMLB_REQUIRE(key_bits == 32 || key_bits == 64, "qmlb_group_by_key: keys must have 32 or 64 bits");
    QMLB_REQUIRE(n < (size_t)1 << 31, "qmlb_group_by_key: fewer than 2^31 keys supported");
    QMLB_REQUIRE(nkeys > 0 && nkeys < INT32_MAX, "qmlb_group_by_key: bad number of keys");
    cudaStream_t st = qmlb::as_stream(stream);
    if (n == 0) {
        empty_kernel<<<((unsigned)nkeys + THREADS) / THREADS < 1184 ? ((unsigned)nkeys + THREADS) / THREADS : 1184, THREADS, 0, st>>>((uint32_t)nkeys, group_start);
        return qmlb::check_launch("qmlb_group_by_key");
    }
    const size_t need = qmlb_group_by_key_scratch_bytes(n, nkeys);
    QMLB_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), "qmlb_group_by_key: scratch too small");
    QMLB_REQUIRE(need == 0 || ((uintptr_t)scratch & 3) == 0, "qmlb_group_by_key: scratch must be 4-byte aligned");
    unsigned char *sc = static_cast<unsigned char *>(scratch);
    return key_bits == 32 ? run<int32_t>(keys, n, nkeys, order, group_start, sc, st) : run<int64_t>(keys, n, nkeys, order, group_start, sc, st);
}
