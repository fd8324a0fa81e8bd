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
#include "common.hpp"

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

// The `tile`-th run of at most `per` rows, group after group (each group starts a run of its own), then the rows of no group.
// A wave looks at 64 groups at a time: their run counts, a prefix sum over the lanes, the lane whose group holds the tile.
// Offsets outside 0..rows are clamped: no offset leads out of the arrays.
__device__ __forceinline__ Tile find_tile(const int* __restrict__ offsets, int G, int rows, int tile, int per) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int g0 = 0; g0 <= G; g0 += 64) {
        const int g = g0 + lane;
        int b = 0, e = 0;
        if (g <= G) {
            b = clamp_pos(offsets[g], 0, rows);
            e = g < G ? clamp_pos(offsets[g + 1], b, rows) : rows;
        }
        const int n = (int)(((int64_t)e - b + per - 1) / per);
        int inc = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d);
            if (lane >= d) inc += o;
        }
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
// runs of the groups before g
__device__ __forceinline__ int runs_before(const int* __restrict__ offsets, int g, int rows, int per) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int i = lane; i < g; i += 64) {
        const int b = clamp_pos(offsets[i], 0, rows), e = clamp_pos(offsets[i + 1], b, rows);
        n += (int)(((int64_t)e - b + per - 1) / per);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
    return n;
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

// dW[g] = the sum of group g's chunks in their order; the same for db.  One workgroup: 256 elements of one group.
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_sum_kernel(Args a) {
    const int64_t n = (int64_t)a.n_out * a.n_in, all = n + (a.dbias ? a.n_out : 0);
    const int64_t blocks = (all + kThreads - 1) / kThreads;
    const int g = (int)(blockIdx.x / blocks);
    const int first = runs_before(a.offsets, g, (int)a.rows, a.chunk_rows), end = runs_before(a.offsets, g + 1, (int)a.rows, a.chunk_rows);
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

// rows per partial sum of dW: 0 (no split) when the output tiles alone fill the chip
int chunk_rows_of(int64_t rows, int G, int n_in, int n_out) {
    const int64_t tiles = (int64_t)ceil_div(n_out, BP) * ceil_div(n_in, BQ);
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

template <typename T>
int launch(int product, const Args& a, hipStream_t s) {
    const int n_q = product == kForward ? a.n_out : a.n_in;
    if (product == kGradWeight) {
        const int64_t blocks = (int64_t)ceil_div(n_q, BQ) * ceil_div(a.n_out, BP) * (a.chunk_rows ? a.chunks : a.G);
        if (int rc = check_grid(blocks)) return rc;
        grouped_product_kernel<T, kGradWeight><<<(unsigned)blocks, kThreads, 0, s>>>(a);
        if (int rc = check_launch("grouped_product_kernel (dW)")) return rc;
        if (!a.chunk_rows) return MCMC_OK;
        const int64_t sums = ((int64_t)a.n_out * a.n_in + (a.dbias ? a.n_out : 0) + kThreads - 1) / kThreads * a.G;
        if (int rc = check_grid(sums)) return rc;
        grouped_sum_kernel<T><<<(unsigned)sums, kThreads, 0, s>>>(a);
        return check_launch("grouped_sum_kernel");
    }
    const int64_t blocks = (a.rows / BP + (a.G + 1 < a.rows ? a.G + 1 : a.rows)) * ceil_div(n_q, BQ);
    if (int rc = check_grid(blocks)) return rc;
    if (product == kForward) grouped_product_kernel<T, kForward><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    else grouped_product_kernel<T, kGradInput><<<(unsigned)blocks, kThreads, 0, s>>>(a);
    return check_launch("grouped_product_kernel");
}

int launch_typed(int dtype, int product, const Args& a, hipStream_t s) {
    if (dtype == MCMC_DT_F32) return launch<float>(product, a, s);
    if (dtype == MCMC_DT_BF16) return launch<__bf16>(product, a, s);
    return launch<_Float16>(product, a, s);
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

int64_t grouped_linear_workspace_bytes(int64_t rows, int G, int n_in, int n_out) {
    const int per = chunk_rows_of(rows, G, n_in, n_out);
    return per ? (int64_t)chunks_of(rows, G, per) * ((int64_t)n_in + 1) * n_out * 4 : 0;
}

int launch_grouped_linear_grad_weight(int dtype, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int64_t rows, const int* order,
                                      const int* offsets, int G, int n_in, int n_out, void* dweight, void* dbias, void* ws, hipStream_t s) {
    const int per = chunk_rows_of(rows, G, n_in, n_out);
    return launch_typed(dtype, kGradWeight,
                        Args{dy, x, nullptr, dweight, dbias, static_cast<float*>(ws), order, offsets, ld_dy, ld_x, rows, G, n_in, n_out, per,
                             per ? chunks_of(rows, G, per) : 0},
                        s);
}

}  // namespace mcmc
