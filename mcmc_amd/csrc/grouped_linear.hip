// One linear layer per group over ragged groups of rows, and its gradients.
//
//   y[r]  = W[g] x[r] + b[g]                      g = the group of row r; rows of no group: 0
//   dx[r] = W[g]^T dy[r]                          rows of no group: 0
//   dW[g] = sum_{r in g} dy[r] x[r]^T,  db[g] = sum_{r in g} dy[r]      a group without rows: 0
//
// All three are one tile product  O[p][q] = sum_c P(p, c) Q(q, c)  with q contiguous in the output:
//            p             q              c              P(p, c)           Q(q, c)
//   forward  row           out feature    in feature     x[row p][c]       W[g][q][c]
//   dx       row           in feature     out feature    dy[row p][c]      W[g][c][q]
//   dW       out feature   in feature     row            dy[row c][p]      x[row c][q]
// The rows of group g are order[offsets[g]] .. order[offsets[g+1] - 1] (order NULL: the rows themselves).  Only the device knows
// the offsets, so a launch has as many row tiles as any offsets could need and each workgroup looks its tile up (find_tile).
#include <type_traits>

#include "common.hpp"
#include "lds_dma.hpp"

namespace mcmc {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Product { kForward, kGradInput, kGradWeight };

struct Args {
    const void* p;  // x (forward), dy (dx, dW): rows of ld_p elements
    const void* q;  // W (forward, dx), x (dW): rows of ld_q elements; W: [G][n_out][n_in]
    const void* bias;
    void* out;      // y, dx, dW
    void* dbias;
    float* part;    // dW in chunks: [chunk][n_out][n_in] then [chunk][n_out]
    const int* order;
    const int* offsets;
    int64_t ld_p, ld_q, rows;
    int G, n_in, n_out;
    int chunk_rows;  // dW: rows per partial sum (0: a group is one sum, written to `out`)
    int chunks;      // dW: partial sums there is room for
};

// ---- matrix instructions: 16 x 16 outputs, kc contraction elements per fragment --------------------------------------------
// lane l holds row (l & 15) and kv consecutive elements from kv * (l >> 4); D: lane l holds column l & 15, rows 4 (l >> 4) + i
template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
    typedef bf16x8 V;
    static constexpr int kv = 8;
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0); }
};
template <>
struct Frag<_Float16> {
    typedef f16x8 V;
    static constexpr int kv = 8;
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, d, 0, 0, 0); }
};
template <>
struct Frag<float> {
    typedef f32x4 V;
    static constexpr int kv = 4;
    // four 16x16x4 steps; step i takes element i of every lane: the same contraction index on both sides, in another order
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], d, 0, 0, 0);
        return d;
    }
};

// ---- tiles -----------------------------------------------------------------------------------------------------------------
struct Tile {
    int g;             // G: rows of no group;  -1: past the last tile
    int first, last;   // positions in `order`
};
__device__ __forceinline__ int clamp_pos(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// A group's run count, group g's first and last position; G: the rows of no group.  Offsets outside 0..rows are clamped: no
// offset leads out of the arrays.
__device__ __forceinline__ int runs_of(const int* __restrict__ offsets, int G, int rows, int g, int per, int& first, int& last) {
    first = last = 0;
    if (g > G) return 0;
    first = clamp_pos(offsets[g], 0, rows);
    last = g < G ? clamp_pos(offsets[g + 1], first, rows) : rows;
    return (int)(((int64_t)last - first + per - 1) / per);
}
__device__ __forceinline__ int wave_inclusive(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
// runs of the groups before g
__device__ __forceinline__ int runs_before(const int* __restrict__ offsets, int G, int g, int rows, int per) {
    int n = 0, b, e;
    for (int i = threadIdx.x & 63; i < g; i += 64) n += runs_of(offsets, G, rows, i, per, b, e);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
    return n;
}
// The `tile`-th run of at most `per` rows, group after group (each group starts a run of its own), then the rows of no group.
// A wave looks at 64 groups at a time: their run counts, a prefix sum over the lanes, the lane whose group holds the tile.
__device__ __forceinline__ Tile find_tile(const int* __restrict__ offsets, int G, int rows, int tile, int per) {
    int before = 0;
    for (int g0 = 0; g0 <= G; g0 += 64) {
        int b, e;
        const int n = runs_of(offsets, G, rows, g0 + (threadIdx.x & 63), per, b, e), inc = wave_inclusive(n);
        const uint64_t hit = __ballot(before + inc > tile);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            const int start = __shfl(b, l), end = __shfl(e, l), mine = tile - before - (__shfl(inc, l) - __shfl(n, l));
            const int64_t first = (int64_t)start + (int64_t)mine * per;
            return Tile{g0 + l, (int)first, (int)(first + per < end ? first + per : end)};
        }
        before += __shfl(inc, 63);
    }
    return Tile{-1, 0, 0};
}

__device__ __forceinline__ int row_at(const Args& a, int pos) {
    const int r = a.order ? a.order[pos] : pos;
    return (unsigned)r < (unsigned)a.rows ? r : -1;  // an index out of range reads as an empty row and is not written
}

constexpr int kThreads = 256;
constexpr int BP = 64, BQ = 64;

// 64 x 64 outputs per workgroup, 32 x 32 per wave; operands go through LDS with the contraction index contiguous
template <typename T, int PRODUCT>
__global__ __launch_bounds__(kThreads) void grouped_product_kernel(Args a) {
    typedef Frag<T> F;
    constexpr int BC = sizeof(T) == 2 ? 64 : 32, S = BC + 16 / (int)sizeof(T);
    __shared__ T lp[BP * S], lq[BQ * S];
    __shared__ int rows_p[BP], rows_c[BC];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int n_q = PRODUCT == kForward ? a.n_out : a.n_in, q_tiles = (n_q + BQ - 1) / BQ;
    const int q0 = (int)(blockIdx.x % q_tiles) * BQ;
    int run = blockIdx.x / q_tiles;  // row tile; dW: the group or chunk
    int p0 = 0;                      // first output row of the tile
    Tile tl;
    if (PRODUCT == kGradWeight) {
        const int p_tiles = (a.n_out + BP - 1) / BP;
        p0 = run % p_tiles * BP;
        run /= p_tiles;
        if (a.chunk_rows) {
            tl = find_tile(a.offsets, a.G, (int)a.rows, run, a.chunk_rows);
            if (tl.g < 0 || tl.g >= a.G) return;
        } else {
            const int b = clamp_pos(a.offsets[run], 0, (int)a.rows);
            tl = Tile{run, b, clamp_pos(a.offsets[run + 1], b, (int)a.rows)};
        }
    } else {
        tl = find_tile(a.offsets, a.G, (int)a.rows, run, BP);
        if (tl.g < 0) return;
        if (t < BP) rows_p[t] = tl.first + t < tl.last ? row_at(a, tl.first + t) : -1;
    }
    const int n_p = PRODUCT == kGradWeight ? a.n_out : BP;
    const int n_c = PRODUCT == kForward ? a.n_in : PRODUCT == kGradInput ? a.n_out : tl.last - tl.first;
    const bool none = PRODUCT != kGradWeight && tl.g == a.G;
    const T* P = static_cast<const T*>(a.p);
    const T* Q = static_cast<const T*>(a.q);
    if (PRODUCT != kGradWeight && !none) Q += (int64_t)tl.g * a.n_in * a.n_out;
    f32x4 acc[2][2] = {}, accb[2] = {};
    const int pw = 32 * (wv & 1), qw = 32 * (wv >> 1), fr = lane & 15, fk = F::kv * (lane >> 4);
    typename F::V ones;
#pragma unroll
    for (int i = 0; i < F::kv; ++i) ones[i] = (T)1.0f;
    __syncthreads();
    for (int c0 = 0; c0 < (none ? 0 : n_c); c0 += BC) {
        if (PRODUCT == kGradWeight) {
            if (t < BC) rows_c[t] = c0 + t < n_c ? row_at(a, tl.first + c0 + t) : -1;
            __syncthreads();
            for (int i = t; i < BP * BC; i += kThreads) {
                const int p = i % BP, c = i / BP, r = rows_c[c];
                lp[p * S + c] = r >= 0 && p0 + p < n_p ? P[(int64_t)r * a.ld_p + p0 + p] : (T)0.0f;
                lq[p * S + c] = r >= 0 && q0 + p < n_q ? Q[(int64_t)r * a.ld_q + q0 + p] : (T)0.0f;
            }
        } else {
            for (int i = t; i < BP * BC; i += kThreads) {
                const int c = i % BC, p = i / BC, r = rows_p[p];
                lp[p * S + c] = r >= 0 && c0 + c < n_c ? P[(int64_t)r * a.ld_p + c0 + c] : (T)0.0f;
            }
            for (int i = t; i < BQ * BC; i += kThreads) {
                if (PRODUCT == kForward) {
                    const int c = i % BC, q = i / BC;
                    lq[q * S + c] = q0 + q < n_q && c0 + c < n_c ? Q[(int64_t)(q0 + q) * a.ld_q + c0 + c] : (T)0.0f;
                } else {
                    const int q = i % BQ, c = i / BQ;
                    lq[q * S + c] = q0 + q < n_q && c0 + c < n_c ? Q[(int64_t)(c0 + c) * a.ld_q + q0 + q] : (T)0.0f;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BC; k += 4 * F::kv) {
            typename F::V fp[2], fq[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fp[i] = *reinterpret_cast<const typename F::V*>(lp + (pw + 16 * i + fr) * S + k + fk);
                fq[i] = *reinterpret_cast<const typename F::V*>(lq + (qw + 16 * i + fr) * S + k + fk);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = F::mfma(fq[j], fp[i], acc[i][j]);
            if (PRODUCT == kGradWeight && a.dbias && q0 == 0)
#pragma unroll
                for (int i = 0; i < 2; ++i) accb[i] = F::mfma(ones, fp[i], accb[i]);
        }
        __syncthreads();
    }
    // lane: output row p = fr of fragment i, four consecutive q
    const T* bias = PRODUCT == kForward && a.bias && !none ? static_cast<const T*>(a.bias) + (int64_t)tl.g * a.n_out : nullptr;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int p = pw + 16 * i + fr;
        int64_t at;
        if (PRODUCT == kGradWeight) {
            if (p0 + p >= n_p) continue;
            at = ((int64_t)run * a.n_out + p0 + p) * a.n_in;
        } else {
            if (rows_p[p] < 0) continue;
            at = (int64_t)rows_p[p] * n_q;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int q = q0 + qw + 16 * j + 4 * (lane >> 4) + e;
                if (q >= n_q) continue;
                float v = acc[i][j][e];
                if (bias) v += (float)bias[q];
                if (PRODUCT == kGradWeight && a.chunk_rows) a.part[at + q] = v;
                else static_cast<T*>(a.out)[at + q] = (T)v;
            }
        if (PRODUCT == kGradWeight && a.dbias && q0 == 0 && qw == 0 && lane < 16) {
            if (a.chunk_rows) a.part[(int64_t)a.chunks * a.n_out * a.n_in + (int64_t)run * a.n_out + p0 + p] = accb[i][0];
            else static_cast<T*>(a.dbias)[(int64_t)tl.g * a.n_out + p0 + p] = (T)accb[i][0];
        }
    }
}

// ---- 16-bit types: large tiles, operands by LDS-DMA ------------------------------------------------------------------------
// BP x BQ outputs per workgroup of WP x WQ waves, 64 contraction elements a step, two LDS stages: the loads of step t+1 run while
// step t is multiplied, one barrier a step.  The tiles lie in LDS as they lie in memory, in 16-byte pieces:
//   "rows"    [BP or BQ][64 c]   operands whose contraction index is contiguous (x, dy; W in the forward pass); fragments by
//             ds_read_b128.  Piece s of row r holds chunk s ^ (r & 7): the eight lanes of a pass, eight rows, hit all banks.
//   "columns" [64 c][BP or BQ]   operands whose output index is contiguous (W in dx; both in dW); fragments by ds_read_b64_tr_b16,
//             which hands each lane a column of four rows.  The 32-byte chunks of row c are permuted by spread(c): the eight rows a
//             pass touches ({0-3, 8-11} + 4n) hit all banks.
// DMA: every row starts on 16 bytes and holds whole 8-element chunks: the pieces go global -> LDS directly (the permutation is
// on the global side, a wave-instruction fills 1 KiB of LDS in order), 16 zero bytes stand in for what lies past the contraction's
// end.  Otherwise they pass through registers, element by element where a chunk crosses the end of a row.
__device__ const uint4 kZeros = {0, 0, 0, 0};
constexpr int kSegment = 1024;  // dW: row numbers in LDS, two segments, the next one loaded while one is used

template <int B>
__device__ __forceinline__ int spread(int c) {  // bytes to xor: bits 5.. of the offset in row c
    if (B >= 128) return ((c & 3) | ((c >> 1) & 4)) << 5;
    if (B == 64) return (((c >> 1) & 1) | ((c >> 2) & 2)) << 5;
    return 0;
}

__device__ __forceinline__ uint4 load_piece(const void* p, int n) {  // n of its eight 2-byte elements exist
    union { uint4 v; uint16_t h[8]; } u;
    if (n >= 8) {
        __builtin_memcpy(&u.v, p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) u.h[i] = i < n ? static_cast<const uint16_t*>(p)[i] : (uint16_t)0;
    }
    return u.v;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename V>
__device__ __forceinline__ V columns_frag(const char* p, int four_rows) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + four_rows));
    return __builtin_bit_cast(V, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

// workgroup id -> tile id: ids go round the eight XCDs, each XCD gets a contiguous run of tiles (its L2 sees neighbours)
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t n) {
    const int64_t x = id & 7, i = id >> 3, q = n >> 3, r = n & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

template <typename T, int PRODUCT, int BP, int BQ, int WP, int WQ, bool DMA>
__global__ __launch_bounds__(64 * WP * WQ, 2) void grouped_tile_kernel(Args a) {
    typedef Frag<T> F;
    constexpr int BC = 64, NW = WP * WQ, NT = 64 * NW;
    constexpr bool kPCols = PRODUCT == kGradWeight, kQCols = PRODUCT != kForward;
    constexpr int kPBytes = BP * BC * 2, kQBytes = BQ * BC * 2, kStage = kPBytes + kQBytes;
    constexpr int NP = kPBytes / 1024 / NW, NQ = kQBytes / 1024 / NW;  // 1-KiB pieces of a stage each wave loads
    constexpr int FP = BP / WP / 16, FQ = BQ / WQ / 16;
    static_assert(NP >= 1 && NQ >= 1 && FP >= 1 && FQ >= 1, "every wave loads and multiplies");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* const rows_lds = reinterpret_cast<int*>(smem + 2 * kStage);  // dW: [2][kSegment] row numbers; else [BP]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rows = (int)a.rows;
    const int n_q = PRODUCT == kForward ? a.n_out : a.n_in, n_p = PRODUCT == kGradWeight ? a.n_out : BP;
    const int q_tiles = (n_q + BQ - 1) / BQ;
    // ---- which tile: bands of eight row tiles (dW: eight tiles of one group), q outside, so that the workgroups that run
    // together share both operands
    constexpr int kBand = 8;
    int64_t id;
    int run = 0, p0 = 0, q0;
    Tile tl;
    if (PRODUCT == kGradWeight) {
        const int p_tiles = (a.n_out + BP - 1) / BP, per_run = p_tiles * q_tiles;
        int64_t runs = a.G;
        if (a.chunk_rows) {
            runs = runs_before(a.offsets, a.G, a.G, rows, a.chunk_rows);
            runs = runs < a.chunks ? runs : a.chunks;  // (offsets that decrease could ask for more)
        }
        if ((int64_t)blockIdx.x >= runs * per_run) return;
        id = xcd_order(blockIdx.x, runs * per_run);
        run = (int)(id / per_run);
        const int in = (int)(id % per_run), band = in / (kBand * q_tiles), high = p_tiles - band * kBand < kBand ? p_tiles - band * kBand : kBand;
        const int at = in - band * kBand * q_tiles;
        p0 = (band * kBand + at % high) * BP;
        q0 = at / high * BQ;
        if (a.chunk_rows) {
            tl = find_tile(a.offsets, a.G, rows, run, a.chunk_rows);
        } else {
            tl.g = run;
            runs_of(a.offsets, a.G, rows, run, 1, tl.first, tl.last);
        }
    } else {
        const int64_t tiles = runs_before(a.offsets, a.G, a.G + 1, rows, BP);
        if ((int64_t)blockIdx.x >= tiles * q_tiles) return;
        id = xcd_order(blockIdx.x, tiles * q_tiles);
        const int64_t band = id / (kBand * q_tiles), left = tiles - band * kBand, high = left < kBand ? left : kBand;
        const int64_t at = id - band * kBand * q_tiles;
        tl = find_tile(a.offsets, a.G, rows, (int)(band * kBand + at % high), BP);
        q0 = (int)(at / high) * BQ;
        for (int i = t; i < BP; i += NT) rows_lds[i] = tl.first + i < tl.last ? row_at(a, tl.first + i) : -1;
        __syncthreads();
    }
    const bool none = PRODUCT != kGradWeight && tl.g == a.G;
    const int n_c = none ? 0 : PRODUCT == kForward ? a.n_in : PRODUCT == kGradInput ? a.n_out : tl.last - tl.first;
    const int steps = (n_c + BC - 1) / BC;
    const T* const P = static_cast<const T*>(a.p);
    const T* const Q = static_cast<const T*>(a.q) + (PRODUCT != kGradWeight && !none ? (int64_t)tl.g * a.n_in * a.n_out : 0);
    const T* const zeros = reinterpret_cast<const T*>(&kZeros);

    // ---- where this lane's pieces come from: an address at step 0, and the first contraction index it needs
    const T *src_p[NP], *src_q[NQ];
    int c_p[NP], c_q[NQ];  // "columns": row of the tile; "rows": first element of the chunk
    int w_p[NP], w_q[NQ];  // !DMA, "columns": elements of the chunk that exist
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int piece = (wave * NP + n) * 64 + lane;
        if (kPCols) {
            c_p[n] = piece / (BP / 8);
            const int col = p0 + 8 * ((piece % (BP / 8)) ^ (spread<BP>(c_p[n]) >> 4));
            w_p[n] = n_p - col;
            src_p[n] = P + (DMA ? (col + 8 <= n_p ? col : 0) : (w_p[n] > 0 ? col : 0));  // columns past the end: any, not stored
        } else {
            const int r = piece >> 3, row = rows_lds[r] < 0 ? 0 : rows_lds[r];  // rows past the end: any, not stored
            c_p[n] = 8 * ((piece & 7) ^ (r & 7));
            src_p[n] = P + (int64_t)row * a.ld_p + c_p[n];
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int piece = (wave * NQ + n) * 64 + lane;
        if (kQCols) {
            c_q[n] = piece / (BQ / 8);
            const int col = q0 + 8 * ((piece % (BQ / 8)) ^ (spread<BQ>(c_q[n]) >> 4));
            w_q[n] = n_q - col;
            src_q[n] = Q + (DMA ? (col + 8 <= n_q ? col : 0) : (w_q[n] > 0 ? col : 0));
            if (PRODUCT == kGradInput) src_q[n] += (int64_t)c_q[n] * a.ld_q;
        } else {
            const int r = piece >> 3, row = q0 + r < n_q ? q0 + r : n_q - 1;
            c_q[n] = 8 * ((piece & 7) ^ (r & 7));
            src_q[n] = Q + (int64_t)row * a.ld_q + c_q[n];
        }
    }
    // dW: row numbers of the run's positions 1024 s .. 1024 s + 1023 -> LDS
    auto fetch_segment = [&](int s) {
        if (PRODUCT != kGradWeight || !a.order) return;
        for (int i = wave; i < kSegment / 64; i += NW) {
            int pos = tl.first + s * kSegment + 64 * i;
            if (pos >= tl.last) break;
            pos += lane;
            glds4(a.order + (pos < tl.last ? pos : tl.last - 1), __builtin_amdgcn_readfirstlane(lds_address(rows_lds + (s & 1) * kSegment + 64 * i)));
        }
    };
    auto row_of = [&](int c) {  // dW: the row at position c of the run, -1 past its end
        if (c >= n_c) return -1;
        const int r = a.order ? rows_lds[c & (2 * kSegment - 1)] : tl.first + c;
        return (unsigned)r < (unsigned)rows ? r : -1;
    };
    uint4 hold_p[DMA ? 1 : NP], hold_q[DMA ? 1 : NQ];
    auto load = [&](int step, int stage) {  // DMA: into LDS; otherwise into hold_*
        const int c0 = step * BC;
        const unsigned to_p = lds_address(smem + stage * kStage) + wave * NP * 1024, to_q = lds_address(smem + stage * kStage + kPBytes) + wave * NQ * 1024;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const T* p;
            int have;  // elements of the chunk inside the contraction
            if (kPCols) {
                const int r = row_of(c0 + c_p[n]);
                have = r >= 0 ? (DMA ? 8 : w_p[n]) : 0;
                p = src_p[n] + (int64_t)r * a.ld_p;
            } else {
                have = n_c - c0 - c_p[n];
                p = src_p[n] + c0;
            }
            if (DMA) glds16(have > 0 ? p : zeros, __builtin_amdgcn_readfirstlane(to_p + n * 1024));
            else hold_p[n] = load_piece(p, have);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const T* q;
            int have;
            if (PRODUCT == kGradWeight) {
                const int r = row_of(c0 + c_q[n]);
                have = r >= 0 ? (DMA ? 8 : w_q[n]) : 0;
                q = src_q[n] + (int64_t)r * a.ld_q;
            } else if (PRODUCT == kGradInput) {
                have = c0 + c_q[n] < n_c ? (DMA ? 8 : w_q[n]) : 0;
                q = src_q[n] + (int64_t)c0 * a.ld_q;
            } else {
                have = n_c - c0 - c_q[n];
                q = src_q[n] + c0;
            }
            if (DMA) glds16(have > 0 ? q : zeros, __builtin_amdgcn_readfirstlane(to_q + n * 1024));
            else hold_q[n] = load_piece(q, have);
        }
    };
    auto store = [&](int stage) {
        char* s = smem + stage * kStage;
#pragma unroll
        for (int n = 0; n < NP; ++n) *reinterpret_cast<uint4*>(s + ((wave * NP + n) * 64 + lane) * 16) = hold_p[DMA ? 0 : n];
#pragma unroll
        for (int n = 0; n < NQ; ++n) *reinterpret_cast<uint4*>(s + kPBytes + ((wave * NQ + n) * 64 + lane) * 16) = hold_q[DMA ? 0 : n];
    };

    // ---- fragments
    const int pw = BP / WP * (wave % WP), qw = BQ / WQ * (wave / WP), fr = lane & 15, kg = lane >> 4;
    auto frag = [&](auto cols, auto width, const char* tile, int first, int i, int kk) -> typename F::V {
        constexpr bool C = decltype(cols)::value;
        constexpr int B = decltype(width)::value;
        if constexpr (C) {
            const int c = 32 * kk + 8 * kg + (fr >> 2);  // rows c and c + 4
            return columns_frag<typename F::V>(tile + c * (2 * B) + ((2 * (first + 16 * i)) ^ spread<B>(8 * kg + (fr >> 2))) + 8 * (fr & 3), 4 * 2 * B);
        } else {
            const int r = first + 16 * i + fr;
            return *reinterpret_cast<const typename F::V*>(tile + r * (2 * BC) + (((4 * kk + kg) ^ (fr & 7)) << 4));
        }
    };
    f32x4 acc[FP][FQ] = {}, accb[FP] = {};
    const bool sum_bias = PRODUCT == kGradWeight && a.dbias && q0 == 0 && qw == 0;
    typename F::V ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (T)1.0f;

    if (steps > 0) {
        fetch_segment(0);
        if (PRODUCT == kGradWeight && a.order) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        load(0, 0);
        if (!DMA) store(0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        barrier_lds_only();
    }
    for (int s = 0; s < steps; ++s) {
        if (s % (kSegment / BC) == 0) fetch_segment(s / (kSegment / BC) + 1);  // the segment before s's is no longer read
        if (s + 1 < steps) load(s + 1, (s + 1) & 1);
        const char* tp = smem + (s & 1) * kStage;
        const char* tq = tp + kPBytes;
#pragma unroll
        for (int kk = 0; kk < BC / 32; ++kk) {
            typename F::V fp[FP], fq[FQ];
#pragma unroll
            for (int j = 0; j < FQ; ++j) fq[j] = frag(std::integral_constant<bool, kQCols>(), std::integral_constant<int, BQ>(), tq, qw, j, kk);
#pragma unroll
            for (int i = 0; i < FP; ++i) fp[i] = frag(std::integral_constant<bool, kPCols>(), std::integral_constant<int, BP>(), tp, pw, i, kk);
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j) acc[i][j] = F::mfma(fq[j], fp[i], acc[i][j]);
            if (sum_bias)
#pragma unroll
                for (int i = 0; i < FP; ++i) accb[i] = F::mfma(ones, fp[i], accb[i]);
        }
        if (!DMA && s + 1 < steps) store((s + 1) & 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        barrier_lds_only();
    }

    // ---- lane: output row fr of fragment i, four consecutive q
    const T* bias = PRODUCT == kForward && a.bias && !none ? static_cast<const T*>(a.bias) + (int64_t)tl.g * a.n_out : nullptr;
    const bool whole = n_q % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;  // four results are one 8-byte store
#pragma unroll
    for (int i = 0; i < FP; ++i) {
        const int p = pw + 16 * i + fr;
        int64_t at;
        if (PRODUCT == kGradWeight) {
            if (p0 + p >= n_p) continue;
            at = ((int64_t)run * a.n_out + p0 + p) * a.n_in;
        } else {
            if (rows_lds[p] < 0) continue;
            at = (int64_t)rows_lds[p] * n_q;
        }
#pragma unroll
        for (int j = 0; j < FQ; ++j) {
            const int q = q0 + qw + 16 * j + 4 * kg;
            f32x4 v = acc[i][j];
            if (bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += q + e < n_q ? (float)bias[q + e] : 0.0f;
            if (PRODUCT == kGradWeight && a.chunk_rows) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (q + e < n_q) a.part[at + q + e] = v[e];
            } else if (whole) {
                typedef T T4 __attribute__((ext_vector_type(4)));
                if (q < n_q) *reinterpret_cast<T4*>(static_cast<T*>(a.out) + at + q) = T4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (q + e < n_q) static_cast<T*>(a.out)[at + q + e] = (T)v[e];
            }
        }
        if (sum_bias && lane < 16) {
            if (a.chunk_rows) a.part[(int64_t)a.chunks * a.n_out * a.n_in + (int64_t)run * a.n_out + p0 + p] = accb[i][0];
            else static_cast<T*>(a.dbias)[(int64_t)tl.g * a.n_out + p0 + p] = (T)accb[i][0];
        }
    }
}

// dW[g] = the sum of group g's chunks in their order; the same for db.  One workgroup: 256 elements of one group.
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_sum_kernel(Args a) {
    const int64_t n = (int64_t)a.n_out * a.n_in, all = n + (a.dbias ? a.n_out : 0);
    const int64_t blocks = (all + kThreads - 1) / kThreads;
    const int g = (int)(blockIdx.x / blocks);
    const int first = runs_before(a.offsets, a.G, g, (int)a.rows, a.chunk_rows), end = runs_before(a.offsets, a.G, g + 1, (int)a.rows, a.chunk_rows);
    const int last = end < a.chunks ? end : a.chunks;
    const int64_t i = (int64_t)(blockIdx.x % blocks) * kThreads + threadIdx.x;
    if (i >= all) return;
    const float* src = i < n ? a.part + i : a.part + (int64_t)a.chunks * n + (i - n);
    const int64_t step = i < n ? n : a.n_out;
    float s = 0.0f;
    for (int c = first; c < last; ++c) s += src[c * step];
    if (i < n) static_cast<T*>(a.out)[g * n + i] = (T)s;
    else static_cast<T*>(a.dbias)[(int64_t)g * a.n_out + (i - n)] = (T)s;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// The products of 16-bit types run on 128 x 128 or 256 x 256 tiles, fp32 on 64 x 64.
struct Shape {
    int bp, bq;
};
Shape shape_of(int dtype, int product, bool dma, int64_t rows, int G, int n_in, int n_out) {
    if (dtype == MCMC_DT_F32) return Shape{BP, BQ};
    const int64_t n_p = product == kGradWeight ? n_out : rows / G, n_q = product == kForward ? n_out : n_in;
    const int64_t tiles = (product == kGradWeight ? (int64_t)ceil_div(n_out, 256) * G : rows / 256) * ceil_div(n_q, 256);
    return dma && n_p >= 192 && n_q >= 192 && tiles >= 256 ? Shape{256, 256} : Shape{128, 128};
}

// rows per partial sum of dW: 0 (no split) when the output tiles alone fill the chip
int chunk_rows_of(int dtype, int64_t rows, int G, int n_in, int n_out) {
    const Shape sh = shape_of(dtype, kGradWeight, false, rows, G, n_in, n_out);
    const int64_t tiles = (int64_t)ceil_div(n_out, sh.bp) * ceil_div(n_in, sh.bq);
    if (tiles * G >= 512 || rows <= 512) return 0;
    int64_t per = ceil_div(rows * tiles, 1024);
    per = (per + 255) / 256 * 256;
    return per >= rows ? 0 : (int)per;
}
int chunks_of(int64_t rows, int G, int per) { return (int)(rows / per + (G < rows ? G : rows)); }

int check_grid(int64_t blocks) {
    MCMC_REQUIRE(blocks <= 0x7FFFFFFFLL, "rows, groups and widths are too large for one call (%lld workgroups)", (long long)blocks);
    return MCMC_OK;
}

template <typename T, int PRODUCT, int TP, int TQ, int WP, int WQ, bool DMA>
int launch_tile(unsigned blocks, const Args& a, hipStream_t s) {
    const size_t lds = 2 * (size_t)(TP + TQ) * 128 + (PRODUCT == kGradWeight ? 2 * kSegment : TP) * sizeof(int);
    const auto kern = grouped_tile_kernel<T, PRODUCT, TP, TQ, WP, WQ, DMA>;
    if (int rc = ensure_dyn_lds((const void*)kern, lds, "grouped_tile_kernel")) return rc;
    kern<<<blocks, 64 * WP * WQ, lds, s>>>(a);
    return check_launch("grouped_tile_kernel");
}

// every row of both operands starts on 16 bytes and is whole 16-byte chunks
bool whole_chunks(int product, const Args& a) {
    auto on16 = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; };
    return on16(a.p, a.ld_p) && on16(a.q, a.ld_q) && a.n_in % 8 == 0 && (product == kForward || a.n_out % 8 == 0);
}

template <typename T, int PRODUCT>
int launch_product(const Args& a, Shape sh, bool dma, unsigned blocks, hipStream_t s) {
    if constexpr (sizeof(T) == 4) {
        grouped_product_kernel<T, PRODUCT><<<blocks, kThreads, 0, s>>>(a);
        return check_launch("grouped_product_kernel");
    } else {
        if (sh.bp == 256) return launch_tile<T, PRODUCT, 256, 256, 2, 4, true>(blocks, a, s);
        return dma ? launch_tile<T, PRODUCT, 128, 128, 2, 2, true>(blocks, a, s) : launch_tile<T, PRODUCT, 128, 128, 2, 2, false>(blocks, a, s);
    }
}

template <typename T>
int launch(int dtype, int product, const Args& a, hipStream_t s) {
    const int n_q = product == kForward ? a.n_out : a.n_in;
    const bool dma = sizeof(T) == 2 && whole_chunks(product, a);
    const Shape sh = shape_of(dtype, product, dma, a.rows, a.G, a.n_in, a.n_out);
    const int64_t runs = product == kGradWeight ? (int64_t)ceil_div(a.n_out, sh.bp) * (a.chunk_rows ? a.chunks : a.G)
                                                : a.rows / sh.bp + (a.G + 1 < a.rows ? a.G + 1 : a.rows);
    const int64_t blocks = runs * ceil_div(n_q, sh.bq);
    if (int rc = check_grid(blocks)) return rc;
    if (product == kForward) return launch_product<T, kForward>(a, sh, dma, (unsigned)blocks, s);
    if (product == kGradInput) return launch_product<T, kGradInput>(a, sh, dma, (unsigned)blocks, s);
    if (int rc = launch_product<T, kGradWeight>(a, sh, dma, (unsigned)blocks, s)) return rc;
    if (!a.chunk_rows) return MCMC_OK;
    const int64_t sums = ((int64_t)a.n_out * a.n_in + (a.dbias ? a.n_out : 0) + kThreads - 1) / kThreads * a.G;
    if (int rc = check_grid(sums)) return rc;
    grouped_sum_kernel<T><<<(unsigned)sums, kThreads, 0, s>>>(a);
    return check_launch("grouped_sum_kernel");
}

int launch_typed(int dtype, int product, const Args& a, hipStream_t s) {
    if (dtype == MCMC_DT_F32) return launch<float>(dtype, product, a, s);
    if (dtype == MCMC_DT_BF16) return launch<__bf16>(dtype, product, a, s);
    return launch<_Float16>(dtype, product, a, s);
}

}  // namespace

int launch_grouped_linear_forward(int dtype, const void* x, int64_t ld_x, int64_t rows, const int* order, const int* offsets, int G, int n_in,
                                  int n_out, const void* weight, const void* bias, void* y, hipStream_t s) {
    return launch_typed(dtype, kForward, Args{x, weight, bias, y, nullptr, nullptr, order, offsets, ld_x, n_in, rows, G, n_in, n_out, 0, 0}, s);
}

int launch_grouped_linear_grad_input(int dtype, const void* dy, int64_t ld_dy, int64_t rows, const int* order, const int* offsets, int G, int n_in,
                                     int n_out, const void* weight, void* dx, hipStream_t s) {
    return launch_typed(dtype, kGradInput, Args{dy, weight, nullptr, dx, nullptr, nullptr, order, offsets, ld_dy, n_in, rows, G, n_in, n_out, 0, 0}, s);
}

int64_t grouped_linear_workspace_bytes(int dtype, int64_t rows, int G, int n_in, int n_out) {
    const int per = chunk_rows_of(dtype, rows, G, n_in, n_out);
    return per ? (int64_t)chunks_of(rows, G, per) * ((int64_t)n_in + 1) * n_out * 4 : 0;
}

int launch_grouped_linear_grad_weight(int dtype, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int64_t rows, const int* order,
                                      const int* offsets, int G, int n_in, int n_out, void* dweight, void* dbias, void* ws, hipStream_t s) {
    const int per = chunk_rows_of(dtype, rows, G, n_in, n_out);
    return launch_typed(dtype, kGradWeight,
                        Args{dy, x, nullptr, dweight, dbias, static_cast<float*>(ws), order, offsets, ld_dy, ld_x, rows, G, n_in, n_out, per,
                             per ? chunks_of(rows, G, per) : 0},
                        s);
}

}  // namespace mcmc
