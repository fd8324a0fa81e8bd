// Rows sorted by group: the plan that the ragged products (grouped_linear.hip) read.
//
//   order   = the rows 0..R-1 sorted stably by key, key(r) = ids[r] if 0 <= ids[r] < G, else G (no group: last)
//   offsets = offsets[g] = number of rows with key < g, g = 0..G
//
// A stable counting sort.  The rows are cut into chunks, one wave each, with counters of their own in LDS; a wave walks its chunk 64
// rows at a time and finds the lanes that hold the same key by one ballot per key bit (match_key), so the rank of a row among its
// equals is a popcount.  Waves share no counter and a wave's LDS operations run in order: the result is a function of the ids alone.
//   one workgroup   (R <= kOneRows): count, scan and place in one launch - a mini-batch costs one launch latency.
//   three launches  (otherwise): count -> counts[key][chunk]; scan each key's row over the chunks; place.
// Bound: the ids are read twice and order written once, 2 x 8 + 4 bytes per row with 64-bit ids; the second read of the ids
// mostly hits the last-level cache.  3.65M rows x 32 groups: 30 us a call (count 9, scan 7, place 16: the 60 vector
// instructions a slab that find equal keys, and the scattered writes) against 8 us for reading the ids and writing the order once at
// 5.4 TB/s; up to 8,192 rows 8.5-10 us, the launch and its Python.
#include "common.hpp"

namespace mcmc {

namespace {

constexpr int kOneWaves = 16;           // waves of the one-workgroup kernel
constexpr int kWaves = 4;               // waves per workgroup of count / place: their four chunks are one int4 of counts
constexpr int64_t kOneRows = 8192;
constexpr int kOneKeys = 1024;          // LDS of the one-workgroup kernel: 16 waves x keys x 4 B
constexpr int kFewBits = 3;              // up to 8 keys counting by match_key beats 64 LDS additions to few addresses
constexpr int kMostChunks = 8192;       // eight waves per SIMD (2,048 chunks: 53 us at 3.65M rows x 32 groups, 4,096: 31, 8,192: 30)
constexpr int kBatch = 4;               // 64-row slabs whose ids are in flight together (2, 4, 8: the same within 1 us)

struct Plan {
    int64_t chunk_rows;  // rows per wave, a multiple of 64
    int chunks;          // a multiple of kWaves
};
// as many chunks as keep the chip busy, but no more counters than half the rows (they are written, scanned and read: at 3.65M rows
// and 1,000 groups a quarter takes 97 us, half 72, all 77)
Plan plan_of(int64_t rows, int G) {
    int64_t most = rows / (2 * ((int64_t)G + 1));
    most = most < 256 ? 256 : most > kMostChunks ? kMostChunks : most;
    int64_t per = (rows + most - 1) / most;
    if (per < 512) per = 512;
    per = (per + 63) / 64 * 64;
    int64_t n = (rows + per - 1) / per;
    n = n < 1 ? kWaves : (n + kWaves - 1) / kWaves * kWaves;  // no rows: one workgroup that writes the offsets
    return Plan{per, (int)n};
}

template <typename Id>
__device__ __forceinline__ int key_of(const Id* ids, int64_t r, int G) {
    const Id v = ids[r];
    return v >= 0 && v < (Id)G ? (int)v : G;
}

// lanes of the wave with this lane's key (`live` lanes only); bits = bits of the largest key
__device__ __forceinline__ uint64_t match_key(int key, bool live, int bits) {
    uint64_t m = __ballot(live);
    uint32_t lo = (uint32_t)m, hi = (uint32_t)(m >> 32);
    for (int b = 0; b < bits; ++b) {
        const uint64_t one = __ballot((key >> b) & 1);
        const uint32_t mine = (uint32_t)((key << (31 - b)) >> 31);  // all ones where the bit is set
        lo &= ~((uint32_t)one ^ mine);
        hi &= ~((uint32_t)(one >> 32) ^ mine);
    }
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ int rank_below(uint64_t m, int lane) { return __popcll(m & ((1ull << lane) - 1)); }

// One wave over rows [r0, r1): `run[key]` (LDS, this wave's own) advances by the number of rows of that key; PLACE also writes
// order[run[key] + rank] = row.  The first lane of each key adds the key's rows of a slab in one LDS operation and hands the old value
// to the others; a wave's LDS operations complete in order, so the slabs of a batch need no wait between them.
template <bool PLACE, typename Id>
__device__ __forceinline__ void walk(const Id* __restrict__ ids, int64_t r0, int64_t r1, int G, int bits, int* run, int* __restrict__ order) {
    const int lane = threadIdx.x & 63;
    for (int64_t base = r0; base < r1; base += 64 * kBatch) {
        int key[kBatch], old[kBatch];
        uint64_t same[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int64_t r = base + 64 * i + lane;
            key[i] = r < r1 ? key_of(ids, r, G) : G;
        }
        if (!PLACE && bits > kFewBits) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (base + 64 * i + lane < r1) atomicAdd(run + key[i], 1);
            continue;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            same[i] = match_key(key[i], base + 64 * i + lane < r1, bits);
            if (same[i] && rank_below(same[i], lane) == 0 && base + 64 * i + lane < r1) {
                const int n = __popcll(same[i]);
                if (PLACE) old[i] = atomicAdd(run + key[i], n);
                else atomicAdd(run + key[i], n);
            }
        }
        if (PLACE)
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int64_t r = base + 64 * i + lane;
                const int at = __shfl(old[i], same[i] ? __ffsll((unsigned long long)same[i]) - 1 : 0);
                if (r < r1) order[at + rank_below(same[i], lane)] = (int)r;
            }
    }
}

// exclusive sum over the workgroup (`part`: one int of LDS per wave); every thread gets its own, the last one's end is *total
template <int NTHREADS>
__device__ __forceinline__ int block_exclusive(int v, int* part, int* total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 63) part[wv] = inc;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NTHREADS / 64; ++w) {
        const int p = part[w];
        before += w < wv ? p : 0;
        sum += p;
    }
    __syncthreads();
    *total = sum;
    return before + inc - v;
}

// ---- one workgroup ---------------------------------------------------------------------------------------------------------
template <typename Id>
__global__ __launch_bounds__(64 * kOneWaves) void group_rows_one_kernel(const Id* __restrict__ ids, int64_t rows, int G, int bits,
                                                                        int* __restrict__ order, int* __restrict__ offsets) {
    extern __shared__ int lds[];  // [16 waves][keys], then 16 ints
    const int keys = G + 1, t = threadIdx.x, wv = t >> 6;
    int* part = lds + kOneWaves * keys;
    for (int i = t; i < kOneWaves * keys; i += 64 * kOneWaves) lds[i] = 0;
    __syncthreads();
    const int64_t per = ((rows + kOneWaves - 1) / kOneWaves + 63) / 64 * 64;
    const int64_t r0 = wv * per < rows ? wv * per : rows, r1 = r0 + per < rows ? r0 + per : rows;
    walk<false>(ids, r0, r1, G, bits, lds + wv * keys, nullptr);
    __syncthreads();
    // thread t owns key t (keys <= 1024): its rows over the waves, then its start among the keys
    int sum = 0;
    if (t < keys)
        for (int w = 0; w < kOneWaves; ++w) {
            const int c = lds[w * keys + t];
            lds[w * keys + t] = sum;  // exclusive over the waves
            sum += c;
        }
    int total;
    const int base = block_exclusive<64 * kOneWaves>(t < keys ? sum : 0, part, &total);
    if (t < keys) {
        offsets[t] = base;
        for (int w = 0; w < kOneWaves; ++w) lds[w * keys + t] += base;
    }
    __syncthreads();
    walk<true>(ids, r0, r1, G, bits, lds + wv * keys, order);
}

// ---- three launches --------------------------------------------------------------------------------------------------------
template <typename Id>
__global__ __launch_bounds__(64 * kWaves) void group_rows_count_kernel(const Id* __restrict__ ids, int64_t rows, int G, int bits, int64_t per,
                                                                       int chunks, int* __restrict__ counts) {
    extern __shared__ int lds[];  // [keys][kWaves] is written out; the walk wants [wave][keys]
    const int keys = G + 1, t = threadIdx.x, wv = t >> 6;
    for (int i = t; i < kWaves * keys; i += 64 * kWaves) lds[i] = 0;
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * kWaves + wv;
    const int64_t r0 = c * per < rows ? c * per : rows, r1 = r0 + per < rows ? r0 + per : rows;
    walk<false>(ids, r0, r1, G, bits, lds + wv * keys, nullptr);
    __syncthreads();
    for (int k = t; k < keys; k += 64 * kWaves)
        *reinterpret_cast<int4*>(counts + (int64_t)k * chunks + (int64_t)blockIdx.x * kWaves) =
            int4{lds[k], lds[keys + k], lds[2 * keys + k], lds[3 * keys + k]};
}

// one workgroup per key: counts[key][*] -> exclusive sums over the chunks, totals[key] = the key's rows
__global__ __launch_bounds__(256) void group_rows_scan_kernel(int chunks, int* __restrict__ counts, int* __restrict__ totals) {
    __shared__ int part[4];
    int* row = counts + (int64_t)blockIdx.x * chunks;
    int carry = 0;
    for (int c0 = 0; c0 < chunks; c0 += 1024) {
        const int c = c0 + 4 * threadIdx.x;  // chunks is a multiple of four
        int4 v = c < chunks ? *reinterpret_cast<const int4*>(row + c) : int4{0, 0, 0, 0};
        int total;
        const int e = carry + block_exclusive<256>(v.x + v.y + v.z + v.w, part, &total);
        if (c < chunks) *reinterpret_cast<int4*>(row + c) = int4{e, e + v.x, e + v.x + v.y, e + v.x + v.y + v.z};
        carry += total;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename Id>
__global__ __launch_bounds__(64 * kWaves) void group_rows_place_kernel(const Id* __restrict__ ids, int64_t rows, int G, int bits, int64_t per,
                                                                       int chunks, const int* __restrict__ counts,
                                                                       const int* __restrict__ totals, int* __restrict__ order,
                                                                       int* __restrict__ offsets) {
    extern __shared__ int lds[];  // [wave][keys]
    __shared__ int part[kWaves];
    const int keys = G + 1, t = threadIdx.x, wv = t >> 6;
    int carry = 0;
    for (int k0 = 0; k0 < keys; k0 += 64 * kWaves) {
        const int k = k0 + t;
        int total;
        const int base = carry + block_exclusive<64 * kWaves>(k < keys ? totals[k] : 0, part, &total);
        if (k < keys) {
            const int4 c = *reinterpret_cast<const int4*>(counts + (int64_t)k * chunks + (int64_t)blockIdx.x * kWaves);
            lds[k] = base + c.x;
            lds[keys + k] = base + c.y;
            lds[2 * keys + k] = base + c.z;
            lds[3 * keys + k] = base + c.w;
            if (blockIdx.x == 0) offsets[k] = base;
        }
        carry += total;
    }
    __syncthreads();
    const int64_t c = (int64_t)blockIdx.x * kWaves + wv;
    const int64_t r0 = c * per < rows ? c * per : rows, r1 = r0 + per < rows ? r0 + per : rows;
    walk<true>(ids, r0, r1, G, bits, lds + wv * keys, order);
}

bool one_workgroup(int64_t rows, int G) { return rows <= kOneRows && G + 1 <= kOneKeys; }

template <typename Id>
int launch(const Id* ids, int64_t rows, int G, int* order, int* offsets, void* ws, hipStream_t s) {
    const int keys = G + 1;
    int bits = 1;
    while ((G >> bits) != 0) ++bits;  // the largest key is G
    if (one_workgroup(rows, G)) {
        const size_t lds = (kOneWaves * (size_t)keys + kOneWaves) * sizeof(int);
        if (int rc = ensure_dyn_lds((const void*)group_rows_one_kernel<Id>, lds, "group_rows_one_kernel")) return rc;
        group_rows_one_kernel<Id><<<1, 64 * kOneWaves, lds, s>>>(ids, rows, G, bits, order, offsets);
        return check_launch("group_rows_one_kernel");
    }
    const Plan p = plan_of(rows, G);
    const size_t lds = kWaves * (size_t)keys * sizeof(int);
    if (int rc = ensure_dyn_lds((const void*)group_rows_count_kernel<Id>, lds, "group_rows_count_kernel")) return rc;
    if (int rc = ensure_dyn_lds((const void*)group_rows_place_kernel<Id>, lds, "group_rows_place_kernel")) return rc;
    int* counts = static_cast<int*>(ws);
    int* totals = counts + (int64_t)keys * p.chunks;
    const int blocks = p.chunks / kWaves;
    group_rows_count_kernel<Id><<<blocks, 64 * kWaves, lds, s>>>(ids, rows, G, bits, p.chunk_rows, p.chunks, counts);
    if (int rc = check_launch("group_rows_count_kernel")) return rc;
    group_rows_scan_kernel<<<keys, 256, 0, s>>>(p.chunks, counts, totals);
    if (int rc = check_launch("group_rows_scan_kernel")) return rc;
    group_rows_place_kernel<Id><<<blocks, 64 * kWaves, lds, s>>>(ids, rows, G, bits, p.chunk_rows, p.chunks, counts, totals, order, offsets);
    return check_launch("group_rows_place_kernel");
}

}  // namespace

int64_t group_rows_workspace_bytes(int64_t rows, int G) {
    if (one_workgroup(rows, G)) return 0;
    return ((int64_t)(G + 1) * plan_of(rows, G).chunks + G + 1) * 4;
}

int launch_group_rows(const void* ids, int id_bytes, int64_t rows, int G, int* order, int* offsets, void* ws, hipStream_t s) {
    return id_bytes == 8 ? launch(static_cast<const int64_t*>(ids), rows, G, order, offsets, ws, s)
                         : launch(static_cast<const int32_t*>(ids), rows, G, order, offsets, ws, s);
}

}  // namespace mcmc
