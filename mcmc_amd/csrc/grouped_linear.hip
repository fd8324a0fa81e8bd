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

enum Product { kForward = MCMC_GROUPED_FORWARD, kGradInput = MCMC_GROUPED_GRAD_INPUT, kGradWeight = MCMC_GROUPED_GRAD_WEIGHT };

struct Args {
    const void* p;  // x (forward), dy (dx, dW): rows of ld_p elements
    const void* q;  // W (forward, dx), x (dW): rows of ld_q elements; W: [G][n_out][n_in]
    const void* bias;
    void* out;      // y, dx, dW
    void* dbias;
    float* part;    // partial sums.  dW in chunks: [chunk][n_out][n_in] then [chunk][n_out]; a split contraction: [split][rows][n_q]
    const int* order;
    const int* offsets;
    int64_t ld_p, ld_q, rows;
    int G, n_in, n_out;
    int chunk_rows;  // dW: rows per partial sum (0: a group is one sum, written to `out`)
    int chunks;      // dW: partial sums there is room for
    int splits;      // forward, dx: parts of the contraction, each a workgroup's
    int split_c;     // contraction elements of a part
};

// ---- matrix instructions: 16 x 16 outputs, 32 contraction elements ---------------------------------------------------------
// a fragment: lane l holds row (l & 15) and eight consecutive elements from 8 (l >> 4); D: lane l holds column l & 15, rows
// 4 (l >> 4) + i
template <typename T>
struct Frag;
// s + the sum of a fragment's eight elements
__device__ __forceinline__ float add_elements(bf16x8 v, float s) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
    s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[0], v[1]}, one, s, false);
    s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[2], v[3]}, one, s, false);
    s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[4], v[5]}, one, s, false);
    return __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[6], v[7]}, one, s, false);
}
__device__ __forceinline__ float add_elements(f16x8 v, float s) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
    s = __builtin_amdgcn_fdot2(f16x2{v[0], v[1]}, one, s, false);
    s = __builtin_amdgcn_fdot2(f16x2{v[2], v[3]}, one, s, false);
    s = __builtin_amdgcn_fdot2(f16x2{v[4], v[5]}, one, s, false);
    return __builtin_amdgcn_fdot2(f16x2{v[6], v[7]}, one, s, false);
}

template <>
struct Frag<__bf16> {
    typedef __bf16 E;  // what the tiles in LDS hold
    typedef bf16x8 V;
    static constexpr int kPlanes = 1;
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0); }
};
template <>
struct Frag<_Float16> {
    typedef _Float16 E;
    typedef f16x8 V;
    static constexpr int kPlanes = 1;
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, d, 0, 0, 0); }
};
// fp32 on the bf16 pipe: the fp32 matrix instructions run at 1/16 of its rate.  x = h + m + l with h = x rounded to bf16's 8 bits, m =
// the rest rounded likewise, l = what is left (at most 8 bits); of the nine products the six down to h l + m m + l h are summed in
// fp32, the small ones first, so that a short sum is rounded once.  Left out: m l + l m + l l, at most 2^-24 |x y| (|m| <= 2^-8 |x|, |l| <=
// 2^-17 |x|), one fp32 rounding.  The split is exact down to |x| = 2^-110; below, l ends at bf16's smallest number, 2^-133 (the matrix
// instructions keep subnormals), so that x is off by up to 2^-134 however small it is.  Near the top of the range the six are not the product: an operand that rounds to an
// infinity has no such split (inf - inf), of a product that overflows, or nearly does, some terms are infinite and of either sign.  All of
// these end in a sum that is not finite, and infinities and NaN stay: such a sum is done over in fp32 (plain_sums).
template <>
struct Frag<float> {
    typedef __bf16 E;
    typedef bf16x8 V;
    static constexpr int kPlanes = 3;
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, d, 0, 0, 0); }
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
// The runs of at most `per` rows, group after group (each group starts runs of its own), then those of the rows of no group.  A wave looks
// at 64 groups at a time: their run counts, a prefix sum over the lanes.  Up to 63 groups are looked at once for both questions.
struct Runs {
    int total;                         // runs of groups 0 .. last_group
    int first, last, count, inclusive; // this lane's group, if one look is enough
};
__device__ __forceinline__ Runs count_runs(const int* __restrict__ offsets, int G, int rows, int per, int last_group) {
    Runs r;
    r.count = runs_of(offsets, G, rows, threadIdx.x & 63, per, r.first, r.last);
    if ((threadIdx.x & 63) > last_group) r.count = 0;
    r.inclusive = wave_inclusive(r.count);
    r.total = G < 64 ? __shfl(r.inclusive, 63) : runs_before(offsets, G, last_group + 1, rows, per);
    return r;
}
__device__ __forceinline__ Tile nth_run(const int* __restrict__ offsets, int G, int rows, int per, const Runs& r, int n) {
    int before = 0;
    for (int g0 = 0; g0 <= G; g0 += 64) {
        int b = r.first, e = r.last, count = r.count, inc = r.inclusive;
        if (g0 > 0 || G >= 64) {
            count = runs_of(offsets, G, rows, g0 + (threadIdx.x & 63), per, b, e);
            inc = wave_inclusive(count);
        }
        const uint64_t hit = __ballot(before + inc > n);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            const int start = __shfl(b, l), end = __shfl(e, l), mine = n - before - (__shfl(inc, l) - __shfl(count, l));
            const int64_t first = (int64_t)start + (int64_t)mine * per;
            return Tile{g0 + l, (int)first, (int)(first + per < end ? first + per : end)};
        }
        before += __shfl(inc, 63);
    }
    return Tile{-1, 0, 0};
}
__device__ __forceinline__ Tile find_tile(const int* __restrict__ offsets, int G, int rows, int n, int per) {
    return nth_run(offsets, G, rows, per, count_runs(offsets, G, rows, per, G), n);
}

__device__ __forceinline__ int row_at(const Args& a, int pos) {
    const int r = a.order ? a.order[pos] : pos;
    return (unsigned)r < (unsigned)a.rows ? r : -1;  // an index out of range reads as an empty row and is not written
}

constexpr int kThreads = 256;

// ---- the tile product ------------------------------------------------------------------------------------------------------
// BP x BQ outputs per workgroup of WP x WQ waves, BC contraction elements a step.  The tiles lie in LDS as they lie in memory, in
// 16-byte pieces of eight 16-bit elements (fp32: three planes of bf16):
//   "rows"    [BP or BQ][BC]     operands whose contraction index is contiguous (x, dy; W in the forward pass); fragments by
//             ds_read_b128.  The pieces of row r are permuted by turn(r): the rows a pass touches hit all banks.
//   "columns" [BC][BP or BQ]     operands whose output index is contiguous (W in dx; both in dW); fragments by ds_read_b64_tr_b16,
//             which hands each lane a column of four rows.  The 32-byte chunks of row c are permuted by spread(c): the eight rows a
//             pass touches ({0-3, 8-11} + 4n) hit all banks.
// A fragment's 16 rows or columns follow each other in the tile, but for Q's of 16-bit types ("paired"): fragments 2 h and 2 h + 1 hold
// 32 h + 8 (m >> 2) + 4 (j & 1) + (m & 3), so that a lane's results of two fragments are eight consecutive columns, one 16-byte
// store, and the four lanes of an output row store 64 consecutive bytes.
// 16-bit types, two LDS stages: the loads of step t+1 run while step t is multiplied, one barrier a step.
//   DMA: every row starts on 16 bytes and holds whole 8-element chunks: the pieces go global -> LDS directly (the permutation is
//   on the global side, a wave-instruction fills 1 KiB of LDS in order), 16 zero bytes stand in for what lies past the
//   contraction's end.  Otherwise they pass through registers, element by element where a chunk crosses the end of a row.
// fp32, one LDS stage (three planes are 48 KB at 128 x 128 x 32: two workgroups a CU, one multiplies while the other stages): the
// loads of step t+1 are in registers while step t is multiplied, and are split on their way into LDS.  (Two stages of 256 x 128, one
// workgroup a CU, the splitting between the products: the same at 2048 x 2048, 15 % slower at 256 x 128.)
// Measured, 16-bit, 32,768 rows, 4096 x 4096: one group 835 / 902 / 1,020 us (forward, dx, dW: 1,317 / 1,219 / 1,078 TFLOP/s), where the
// clock falls to what the power allows; eight groups of random sizes 1,001 / 1,030 / 1,065 (136 row tiles for 128: nine rounds of
// workgroups for eight).  8,192 rows, 8 groups, 2048 x 2048: 97 / 105 / 82 us, 707 / 656 / 834 TFLOP/s; rows that are not whole 16-byte
// pieces (2047 x 2045) 212 / 180 / 160.  fp32 there: 454 / 458 / 415 us, 151 / 150 / 166 TFLOP/s (the fp32 matrix instructions' dense
// product reaches 153 on this card).
__device__ const uint4 kZeros[2] = {};
constexpr int kSegment = 1024;  // dW: row numbers in LDS, two segments, the next one loaded while one is used

// permutation of the 16-byte pieces of row r: a pass of ds_read_b128 takes fragment rows {0-3, 12-15} of one lane group and {4-11} of the
// next; PAIRED: row m of the fragment is row 8 (m >> 2) + (m & 3) of the tile
template <int BC, bool PAIRED>
__device__ __forceinline__ int turn(int r) {
    if (BC == 64) return PAIRED ? (r & 3) | ((r >> 1) & 4) : r & 7;
    return -(r >> (PAIRED ? 3 : 2)) & 3;
}
template <int B>
__device__ __forceinline__ int spread(int c) {  // bytes to xor: bits 5.. of the offset in row c
    if (B >= 128) return ((c & 3) | ((c >> 1) & 4)) << 5;
    if (B == 64) return (((c >> 1) & 1) | ((c >> 2) & 2)) << 5;
    return 0;
}

// eight elements in registers; n of them exist
template <typename T>
struct Piece {
    T v[8];
};
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p, int n) {
    Piece<T> u;
    if (n >= 8) {
        __builtin_memcpy(u.v, p, sizeof(u.v));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // (a read that always happens, of the first element or of zeros: no branch per element)
            const T x = n > 0 ? p[i < n ? i : 0] : (T)0.0f;
            u.v[i] = i < n ? x : (T)0.0f;
        }
    }
    return u;
}
template <typename T>
__device__ __forceinline__ void store_piece(char* at, int plane_bytes, const Piece<T>& u) {
    if constexpr (sizeof(T) == 2) {
        __builtin_memcpy(__builtin_assume_aligned(at, 16), u.v, 16);
    } else {
        bf16x8 h, m, l;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = (__bf16)u.v[i];
            const float rest = u.v[i] - (float)h[i];
            m[i] = (__bf16)rest;
            l[i] = (__bf16)(rest - (float)m[i]);
        }
        *reinterpret_cast<bf16x8*>(at) = h;
        *reinterpret_cast<bf16x8*>(at + plane_bytes) = m;
        *reinterpret_cast<bf16x8*>(at + 2 * plane_bytes) = l;
    }
}

// Pieces without a branch between their loads.  whole: every piece has eight elements or none.  Otherwise a piece that ends past its
// row is read into the next row (`inside` says that there is one) and what is not its own is dropped; a wave with a piece of which
// that cannot be said reads element by element.
template <typename T>
__device__ __forceinline__ Piece<T> load_eight(const T* p, int n) {
    Piece<T> u;
    __builtin_memcpy(u.v, n > 0 ? p : reinterpret_cast<const T*>(kZeros), sizeof(u.v));
    return u;
}
template <typename T>
__device__ __forceinline__ void keep_first(Piece<T>& u, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u.v[i] = i < n ? u.v[i] : (T)0.0f;
}
template <typename T>
__device__ __forceinline__ Piece<T> load_through(const T* p, int n, bool inside) {
    if (__any(n > 0 && n < 8 && !inside)) return load_piece(p, n);
    Piece<T> u = load_eight(p, n);
    keep_first(u, n);
    return u;
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

// until at most N of this wave's loads (global -> LDS ones included) are in flight; they complete in the order of their issue
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// row[q .. q + N - 1] = value(0 .. N - 1) as far as the row goes: one store of 16 bytes, which may lie anywhere, or element by element
template <typename T, int N, typename Value>
__device__ __forceinline__ void store_some(T* row, int q, int width, Value value) {
    typedef T Some __attribute__((ext_vector_type(N)));
    typedef Some Anywhere __attribute__((aligned(sizeof(T))));
    Some o;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = (T)value(e);  // the one rounding of a 16-bit result
    if (q + N <= width) {
        *reinterpret_cast<Anywhere*>(row + q) = o;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (q + e < width) row[q + e] = o[e];
    }
}

// fp32: of the 16 x 16 N results of N fragments, those that are not finite (see Frag<float>) once more, from memory, with the fp32 matrix
// instructions, which follow fp32's rules.  p(c): element c of the contraction for row l & 15 of P, q(c, j): for column l & 15 of Q's fragment
// j; lane l asks for c = l >> 4, + 4, + 8 ...; start(j, e): what result e of fragment j starts from.  All lanes of a wave take part or none.
// Rare, so it is short rather than fast; what is NaN stays so, and once all of them are, it ends.  32,768 rows, 8 groups, 2048 x 2048, one row of
// infinities: the gradient pass 6 ms more (all of dW has that row), forward and NaN no more than without; all infinities: 27 ms more.
template <int N, typename Start, typename P, typename Q>
__device__ __forceinline__ void plain_sums(f32x4 (&acc)[N], bool valid, Start start, int n, P p, Q q) {
    static_assert(N <= 8, "");
    float all = 0.0f;  // not finite if one of them is not
#pragma unroll
    for (int k = 0; k < 4 * N; ++k) all += acc[k >> 2][k & 3];
    if (!__any(valid && !__builtin_isfinite(all))) return;
    unsigned which = 0;
    f32x4 s[N];
#pragma unroll
    for (int k = 0; k < 4 * N; ++k) {
        which |= (unsigned)(valid && !__builtin_isfinite(acc[k >> 2][k & 3])) << k;
        s[k >> 2][k & 3] = start(k >> 2, k & 3);
    }
    const int kg = (threadIdx.x & 63) >> 4;
    for (int c0 = 0; c0 < n; c0 += 16) {
        bool open = false;
#pragma unroll
        for (int k = 0; k < 4 * N; ++k) open |= (which >> k & 1) && !__builtin_isnan(s[k >> 2][k & 3]);
        if (!__any(open)) break;
#pragma unroll
        for (int d = 0; d < 16; d += 4) {
            const int c = c0 + d + kg;
            const float x = c < n ? p(c) : 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(c < n ? q(c, j) : 0.0f, x, s[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int k = 0; k < 4 * N; ++k) acc[k >> 2][k & 3] = which >> k & 1 ? s[k >> 2][k & 3] : acc[k >> 2][k & 3];
}

// workgroup id -> tile id: ids go round the eight XCDs, each XCD gets a contiguous run of tiles (its L2 sees neighbours)
__device__ __forceinline__ int64_t xcd_order(int64_t id, int64_t n) {
    const int64_t x = id & 7, i = id >> 3, q = n >> 3, r = n & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

template <typename T, int PRODUCT, int BP, int BQ, int WP, int WQ, bool DMA, int BC, int STAGES>
__global__ __launch_bounds__(64 * WP * WQ, 2) void grouped_tile_kernel(Args a) {
    typedef Frag<T> F;
    typedef typename F::V V;
    constexpr bool kWide = sizeof(T) == 4;
    constexpr int NW = WP * WQ, NT = 64 * NW;
    constexpr bool kPair = !kWide;
    constexpr bool kAhead = STAGES == 1;  // one stage: the next step waits in registers
    static_assert(DMA ? STAGES >= 2 : STAGES <= 2, "");
    constexpr bool kPCols = PRODUCT == kGradWeight, kQCols = PRODUCT != kForward;
    constexpr int kPBytes = BP * BC * 2, kQBytes = BQ * BC * 2, kStage = (kPBytes + kQBytes) * F::kPlanes;
    constexpr int NP = kPBytes / 1024 / NW, NQ = kQBytes / 1024 / NW;  // 1-KiB pieces of a stage each wave loads
    constexpr int FP = BP / WP / 16, FQ = BQ / WQ / 16;
    static_assert(NP >= 1 && NQ >= 1 && FP >= 1 && FQ >= 1 && !(DMA && kWide), "every wave loads and multiplies; fp32 is split in registers");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* const rows_lds = reinterpret_cast<int*>(smem + STAGES * kStage);  // dW: [2][kSegment] row numbers; else [BP]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rows = (int)a.rows;
    const int n_q = PRODUCT == kForward ? a.n_out : a.n_in, n_p = PRODUCT == kGradWeight ? a.n_out : BP;
    const int q_tiles = (n_q + BQ - 1) / BQ;
    // ---- which tile: bands of eight row tiles (dW: eight tiles of one group), q outside, so that the workgroups that run
    // together share both operands
    constexpr int kBand = 8;
    int64_t id;
    int run = 0, split = 0, p0 = 0, q0;
    Tile tl;
    if (PRODUCT == kGradWeight) {
        const int p_tiles = (a.n_out + BP - 1) / BP, per_run = p_tiles * q_tiles;
        int64_t runs = a.G;
        Runs all;
        if (a.chunk_rows) {
            all = count_runs(a.offsets, a.G, rows, a.chunk_rows, a.G - 1);
            runs = all.total < a.chunks ? all.total : a.chunks;  // (offsets that decrease could ask for more)
        }
        if ((int64_t)blockIdx.x >= runs * per_run) return;
        // A group whose tiles alone fill the chip is shared by all XCDs, as another may have far fewer rows (8 groups of 2,000 to 6,000
        // rows, 4096 x 4096 bf16: 1,325 us with a group to an XCD, 1,070 like this); smaller ones stay on one, which then reads their
        // rows once (64 groups of 48 tiles: 170 us, shared 187)
        if (!a.chunk_rows && per_run >= 256) {
            run = (int)(blockIdx.x / per_run);
            id = xcd_order(blockIdx.x % per_run, per_run);
        } else {
            id = xcd_order(blockIdx.x, runs * per_run);
            run = (int)(id / per_run);
            id %= per_run;
        }
        const int in = (int)id, band = in / (kBand * q_tiles), high = p_tiles - band * kBand < kBand ? p_tiles - band * kBand : kBand;
        const int at = in - band * kBand * q_tiles;
        p0 = (band * kBand + at % high) * BP;
        q0 = at / high * BQ;
        if (a.chunk_rows) {
            tl = nth_run(a.offsets, a.G, rows, a.chunk_rows, all, run);
        } else {
            tl.g = run;
            runs_of(a.offsets, a.G, rows, run, 1, tl.first, tl.last);
        }
    } else {
        const Runs all = count_runs(a.offsets, a.G, rows, BP, a.G);
        const int64_t tiles = all.total, block = blockIdx.x / a.splits;
        if (block >= tiles * q_tiles) return;
        split = (int)(blockIdx.x % a.splits);
        id = xcd_order(block, tiles * q_tiles);
        const int64_t band = id / (kBand * q_tiles), left = tiles - band * kBand, high = left < kBand ? left : kBand;
        const int64_t at = id - band * kBand * q_tiles;
        tl = nth_run(a.offsets, a.G, rows, BP, all, (int)(band * kBand + at % high));
        q0 = (int)(at / high) * BQ;
        for (int i = t; i < BP; i += NT) rows_lds[i] = tl.first + i < tl.last ? row_at(a, tl.first + i) : -1;
        __syncthreads();
    }
    const bool none = PRODUCT != kGradWeight && tl.g == a.G;
    int n_c = none ? 0 : PRODUCT == kForward ? a.n_in : PRODUCT == kGradInput ? a.n_out : tl.last - tl.first;
    const T* P = static_cast<const T*>(a.p);
    const T* Q = static_cast<const T*>(a.q) + (PRODUCT != kGradWeight && !none ? (int64_t)tl.g * a.n_in * a.n_out : 0);
    if (PRODUCT != kGradWeight && a.splits > 1) {  // this workgroup's part of the contraction
        const int c = split * a.split_c;
        n_c = n_c - c < a.split_c ? (n_c > c ? n_c - c : 0) : a.split_c;
        P += c;
        Q += PRODUCT == kForward ? c : (int64_t)c * a.ld_q;
    }
    const int steps = (n_c + BC - 1) / BC;
    const T* const zeros = reinterpret_cast<const T*>(kZeros);

    // ---- where this lane's pieces come from.  "rows": the chunk's address at step 0, kept.  "columns": row of the tile and first column,
    // made from the lane number where they are used: kept in registers for all pieces they would crowd out the accumulators
    // (`now_lane` is the lane number behind an empty asm statement, so that the compiler does not move the arithmetic out of the loop).
    // A piece's row in the tile is a lane's part plus a wave's (col_row0), which share no bits that spread() looks at: the permutation is
    // the exclusive or of theirs, and the wave's is scalar arithmetic.
    const T *src_p[kPCols ? 1 : NP], *src_q[kQCols ? 1 : NQ];
    int c_p = 0, c_q[kQCols ? 1 : NQ];  // "rows": first element of the chunk at step 0 (all of P's pieces of a lane have the same one)
    unsigned has_next_p = 0, has_next_q = 0;  // "rows", !DMA: bit n: eight elements from anywhere in piece n's row are memory of the operand
    int now_lane = lane;
    auto col_row0 = [&](int n, int np, int b) { return (wave * np + n) * (64 / (b / 8)); };
    auto col_row = [&](int n, int np, int b) { return col_row0(n, np, b) + now_lane / (b / 8); };
    auto column_of = [&](auto width, int n, int np) {
        constexpr int B = decltype(width)::value;
        return (8 * (now_lane % (B / 8)) ^ (spread<B>(now_lane / (B / 8)) >> 1)) ^ (spread<B>(col_row0(n, np, B)) >> 1);
    };
    if constexpr (!kPCols) {
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const int piece = (wave * NP + n) * 64 + lane, r = piece / (BC / 8), row = rows_lds[r] < 0 ? 0 : rows_lds[r];
            c_p = 8 * ((piece % (BC / 8)) ^ turn<BC, false>(r));
            src_p[n] = P + (int64_t)row * a.ld_p + c_p;  // rows past the end: any, not stored
            if (row + 1 < rows && a.ld_p > 7) has_next_p |= 1u << n;
        }
    }
    if constexpr (!kQCols) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int piece = (wave * NQ + n) * 64 + lane, r = piece / (BC / 8), row = q0 + r < n_q ? q0 + r : n_q - 1;
            c_q[n] = 8 * ((piece % (BC / 8)) ^ turn<BC, kPair>(r));
            src_q[n] = Q + (int64_t)row * a.ld_q + c_q[n];
            if (row + 1 < n_q && a.ld_q > 7) has_next_q |= 1u << n;
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
    Piece<T> hold_p[DMA ? 1 : NP], hold_q[DMA ? 1 : NQ];
    int rest_p = 8, rest_q[kQCols ? 1 : NQ];  // "rows" in hold_*: elements before the contraction's end
    // dW: the rows of this lane's pieces, looked up before the pieces are asked for (both operands' pieces lie alike if BP == BQ)
    int row_p[kPCols ? NP : 1], row_q[kPCols && BP != BQ ? NQ : 1];
    auto look_up = [&](int step) {
        asm volatile("" : "+v"(now_lane));
        if constexpr (kPCols) {
#pragma unroll
            for (int n = 0; n < NP; ++n) row_p[n] = row_of(step * BC + col_row(n, NP, BP));
            if constexpr (BP != BQ)
#pragma unroll
                for (int n = 0; n < NQ; ++n) row_q[n] = row_of(step * BC + col_row(n, NQ, BQ));
        }
    };
    // Piece n (P's, then Q's) of a step: where it starts, how many of its elements exist, and whether eight may be read all the same (they
    // end in a row that exists)
    auto piece = [&](int n, int step, const T*& p, int& have, bool& inside) {
        const int c0 = step * BC;
        inside = true;
        if (n < NP) {
            if constexpr (kPCols) {
                int col = p0 + column_of(std::integral_constant<int, BP>(), n, NP);
                have = row_p[n] >= 0 ? n_p - col : 0;
                if (DMA) col = col < n_p - 8 ? col : n_p - 8;  // columns past the end: any, not stored
                else inside = row_p[n] + 1 < rows && col + 8 <= a.ld_p + n_p;
                if (DMA) have = row_p[n] >= 0 ? 8 : 0;
                p = P + (int64_t)row_p[n] * a.ld_p + col;
            } else {
                have = n_c - c0 - c_p;
                p = src_p[n] + c0;
                if (!DMA) inside = has_next_p >> n & 1;
            }
        } else {
            const int m = n - NP;
            if constexpr (kQCols) {
                const int c = col_row(m, NQ, BQ);
                int r, col = q0 + column_of(std::integral_constant<int, BQ>(), m, NQ);
                if constexpr (PRODUCT == kGradWeight) r = BP != BQ ? row_q[BP != BQ ? m : 0] : row_p[m];
                else r = c0 + c < n_c ? c0 + c : -1;
                have = r >= 0 ? n_q - col : 0;
                if (DMA) col = col < n_q - 8 ? col : n_q - 8;
                else inside = r + 1 < (PRODUCT == kGradWeight ? rows : n_c) && col + 8 <= a.ld_q + n_q;
                if (DMA) have = r >= 0 ? 8 : 0;
                p = Q + (int64_t)r * a.ld_q + col;
            } else {
                have = n_c - c0 - c_q[m];
                p = src_q[m] + c0;
                if (!DMA) inside = has_next_q >> m & 1;
            }
        }
    };
    auto load = [&](int n, int step, int stage) {  // DMA: into LDS
        const T* p;
        int have;
        bool inside;
        piece(n, step, p, have, inside);
        const unsigned to = lds_address(smem + stage * kStage) + (n < NP ? (wave * NP + n) * 1024 : kPBytes + (wave * NQ + n - NP) * 1024);
        glds16(have > 0 ? p : zeros, __builtin_amdgcn_readfirstlane(to));
    };
    auto load_all = [&](int step, int stage) {  // !DMA: into hold_*, no branch between the loads
        look_up(step);
        if constexpr (DMA) {
#pragma unroll
            for (int n = 0; n < NP + NQ; ++n) load(n, step, stage);
        } else {
            const T* p[NP + NQ];
            int have[NP + NQ];
            bool beyond = false;  // a piece that is not whole and has no row after its own
#pragma unroll
            for (int n = 0; n < NP + NQ; ++n) {
                bool inside;
                piece(n, step, p[n], have[n], inside);
                beyond |= have[n] > 0 && have[n] < 8 && !inside;
            }
            const bool slow = __any(beyond);
            if (!slow) {
#pragma unroll
                for (int n = 0; n < NP; ++n) hold_p[n] = load_eight(p[n], have[n]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) hold_q[n] = load_eight(p[NP + n], have[NP + n]);
            } else {
#pragma unroll
                for (int n = 0; n < NP; ++n) hold_p[n] = load_piece(p[n], have[n]);
#pragma unroll
                for (int n = 0; n < NQ; ++n) hold_q[n] = load_piece(p[NP + n], have[NP + n]);
            }
            // what was read past an operand's contraction is dropped when it is stored (past its output columns, it does not matter)
            if constexpr (!kPCols) rest_p = have[0];
            if constexpr (!kQCols)
#pragma unroll
                for (int n = 0; n < NQ; ++n) rest_q[n] = have[NP + n];
        }
    };
    const bool ragged = n_c % 8 != 0;
    auto store = [&](int stage) {
        char* s = smem + stage * kStage;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            if (!DMA && !kPCols && ragged) keep_first(hold_p[DMA ? 0 : n], rest_p);
            store_piece(s + ((wave * NP + n) * 64 + lane) * 16, kPBytes, hold_p[DMA ? 0 : n]);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            if (!DMA && !kQCols && ragged) keep_first(hold_q[DMA ? 0 : n], rest_q[kQCols ? 0 : n]);
            store_piece(s + F::kPlanes * kPBytes + ((wave * NQ + n) * 64 + lane) * 16, kQBytes, hold_q[DMA ? 0 : n]);
        }
    };

    // ---- fragments
    const int pw = BP / WP * (wave % WP), qw = BQ / WQ * (wave / WP), fr = lane & 15, kg = lane >> 4;
    // byte offset of fragment 0 in its tile; fragment i: "rows" + 16 i rows, "columns" ^ 32 i; paired "rows" + 32 (i >> 1) + 4 (i & 1)
    // rows, "columns" ^ 64 (i >> 1) + 8 (i & 1) (no carry: a wave's first column is a multiple of all its fragments' columns).  The
    // second 32 contraction elements: "rows" ^ 64, "columns" + 32 rows.
    auto frag_at = [&](auto cols, auto paired, auto width, int first) {
        constexpr int B = decltype(width)::value;
        constexpr bool kTwo = decltype(paired)::value;
        if constexpr (decltype(cols)::value) {
            const int c = 8 * kg + (fr >> 2);  // rows c and c + 4
            return c * (2 * B) + ((2 * first + (kTwo ? 16 * (fr & 3) : 0)) ^ spread<B>(c)) + (kTwo ? 0 : 8 * (fr & 3));
        } else {
            const int r = kTwo ? 8 * (fr >> 2) + (fr & 3) : fr;
            return (first + r) * (2 * BC) + ((kg ^ turn<BC, kTwo>(r)) << 4);
        }
    };
    auto frag = [&](auto cols, auto paired, auto width, const char* tile, int at, int i, int kk) -> V {
        constexpr int B = decltype(width)::value;
        constexpr bool kTwo = decltype(paired)::value;
        if constexpr (decltype(cols)::value)
            return columns_frag<V>(tile + (at ^ (kTwo ? 64 * (i >> 1) : 32 * i)) + (kTwo ? 8 * (i & 1) : 0) + kk * 32 * (2 * B), 4 * 2 * B);
        else
            return *reinterpret_cast<const V*>(tile + (at ^ (64 * kk)) + (kTwo ? 32 * (i >> 1) + 4 * (i & 1) : 16 * i) * (2 * BC));
    };
    typedef std::integral_constant<bool, kPCols> PCols;
    typedef std::integral_constant<bool, kQCols> QCols;
    typedef std::integral_constant<bool, kPair> Pair;
    int at_p = frag_at(PCols(), std::false_type(), std::integral_constant<int, BP>(), pw);
    int at_q = frag_at(QCols(), Pair(), std::integral_constant<int, BQ>(), qw);
    f32x4 acc[FP][FQ] = {};
    // db: this lane's share of the sums of dy's columns.  fp32 results: a plain sum loses more than torch's pairwise one, so every
    // kSegment rows the running sum goes into a second one
    float accb[FP] = {}, sumb[FP] = {};
    const bool sum_bias = PRODUCT == kGradWeight && a.dbias && q0 == 0 && qw == 0;
    auto p_frag = [&](const char* stage, int l, int i, int kk) {
        return frag(PCols(), std::false_type(), std::integral_constant<int, BP>(), stage + l * kPBytes, at_p, i, kk);
    };
    auto q_frag = [&](const char* stage, int l, int j, int kk) {
        return frag(QCols(), Pair(), std::integral_constant<int, BQ>(), stage + F::kPlanes * kPBytes + l * kQBytes, at_q, j, kk);
    };
    if (steps > 0) {
        fetch_segment(0);
        if (PRODUCT == kGradWeight && a.order) {
            wait_loads<0>();
            __syncthreads();
        }
    }
    if constexpr (DMA) {
        // Two halves of 32 contraction elements a step.  While the matrix instructions of one half run, the fragments of the next are
        // read: the second half's during the first; the barrier between them says that everybody has read this stage and that the
        // next one has arrived; during the second half the next step's first fragments are read and the step after it is asked for,
        // into the stage just read.  A P fragment's register takes its successor as soon as its products are issued; the last two
        // and Q's have two sets, so that all reads of a half are issued two groups before they are waited for.
        static_assert(BC == 64 && STAGES == 2 && FP >= 4 && FQ <= FP, "two halves, two stages");
        constexpr int NL = NP + NQ, NT2 = FP - 2;
        V fp[NT2], tail[2][2], fq[2][FQ];
        auto read_group = [&](int g, int half, int stage) {  // of group g: the reads for `half` of `stage`
            const char* at = smem + stage * kStage;
            if (g < 2) tail[half][g] = p_frag(at, 0, NT2 + g, half);
            if (g < FQ) fq[half][g] = q_frag(at, 0, g, half);
            if (g >= 1 && g - 1 < NT2) fp[g - 1] = p_frag(at, 0, g - 1, half);
        };
        auto multiply = [&](int i, int half) {
            const V p = i < NT2 ? fp[i < NT2 ? i : 0] : tail[half][i < NT2 ? 0 : i - NT2];
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = F::mfma(fq[half][j], p, acc[i][j]);
        };
        if (steps > 0) {
            load_all(0, 0);
            load_all(1, 1);
            wait_loads<NL>();
            barrier_lds_only();
        }
        if (PRODUCT == kGradWeight && sum_bias) {
            // The waves that also sum dy's columns (those of the first output columns, one wave in 16 of a 4096 x 4096 dW) read each
            // fragment where it is multiplied: the sums' registers beside two sets of fragments would be kept in memory, and every
            // reload of one waits for all loads in flight.  They meet the others at the same barriers.
            for (int s = 0; s < steps; ++s) {
                const int now = s & 1;
                if (s % (kSegment / BC) == 0) fetch_segment(s / (kSegment / BC) + 1);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int j = 0; j < FQ; ++j) fq[0][j] = q_frag(smem + now * kStage, 0, j, half);
#pragma unroll
                    for (int i = 0; i < FP; ++i) {
                        const V p = p_frag(smem + now * kStage, 0, i, half);
#pragma unroll
                        for (int j = 0; j < FQ; ++j) acc[i][j] = F::mfma(fq[0][j], p, acc[i][j]);
                        accb[i] = add_elements(p, accb[i]);
                    }
                }
                wait_loads<0>();
                barrier_lds_only();
                load_all(s + 2, now);
            }
        } else {
            if (steps > 0)
#pragma unroll
                for (int g = 0; g < FP; ++g) read_group(g, 0, 0);
            for (int s = 0; s < steps; ++s) {
                const int now = s & 1;
                if (s % (kSegment / BC) == 0) fetch_segment(s / (kSegment / BC) + 1);  // the segment before s's is no longer read
                asm volatile("" : "+v"(at_p), "+v"(at_q));  // as now_lane: the fragments' offsets are made where they are used
#pragma unroll
                for (int g = 0; g < FP; ++g) {
                    multiply(g, 0);
                    read_group(g, 1, now);
                    __builtin_amdgcn_sched_barrier(0);
                }
                wait_loads<0>();
                barrier_lds_only();
                look_up(s + 2);
#pragma unroll
                for (int g = 0; g < FP; ++g) {
                    multiply(g, 1);
                    read_group(g, 0, now ^ 1);
#pragma unroll
                    for (int n = g * NL / FP; n < (g + 1) * NL / FP; ++n) load(n, s + 2, now);  // past the last step: zeros, nobody reads them
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        wait_loads<0>();  // no load may outlive its workgroup's LDS
    } else {
        // through registers: all of Q's fragments against one of P's after the other, which are read two ahead
        auto multiply = [&](const char* at) {
            constexpr int KK = BC / 32, NI = KK * F::kPlanes * FP;  // P fragments of the stage: [kk][plane][i]
            V fq[F::kPlanes][FQ], fp[3];
            auto read_p = [&](int x) { return p_frag(at, F::kPlanes - 1 - x / FP % F::kPlanes, x % FP, x / (F::kPlanes * FP)); };
            fp[0] = read_p(0);
            fp[1] = read_p(1);
#pragma unroll
            for (int x = 0; x < NI; ++x) {
                const int i = x % FP, l = F::kPlanes - 1 - x / FP % F::kPlanes;
                if (x % (F::kPlanes * FP) == 0)
#pragma unroll
                    for (int m = 0; m < F::kPlanes; ++m)
#pragma unroll
                        for (int j = 0; j < FQ; ++j) fq[m][j] = q_frag(at, m, j, x / (F::kPlanes * FP));
                if (x + 2 < NI) fp[(x + 2) % 3] = read_p(x + 2);
#pragma unroll
                for (int m = F::kPlanes - 1 - l; m >= 0; --m)
#pragma unroll
                    for (int j = 0; j < FQ; ++j) acc[i][j] = F::mfma(fq[m][j], fp[x % 3], acc[i][j]);
                if (sum_bias) accb[i] = add_elements(fp[x % 3], accb[i]);
            }
        };
        if (steps > 0) {
            load_all(0, 0);
            if (!kAhead) {
                store(0);
                barrier_lds_only();
            }
        }
        for (int s = 0; s < steps; ++s) {
            const int now = kAhead ? 0 : s & 1;
            if (s % (kSegment / BC) == 0) {
                fetch_segment(s / (kSegment / BC) + 1);  // the segment before s's is no longer read
                if (kWide && sum_bias)
#pragma unroll
                    for (int i = 0; i < FP; ++i) sumb[i] += accb[i], accb[i] = 0.0f;
            }
            if (kAhead) {
                store(0);
                barrier_lds_only();
            }
            if (s + 1 < steps) load_all(s + 1, 0);
            multiply(smem + now * kStage);
            if (!kAhead && s + 1 < steps) store(now ^ 1);
            wait_loads<0>();
            barrier_lds_only();
        }
    }
    auto plain_element = [&](const T* base, int64_t ld, int c, int col) {  // dW: column col of the run's row c; 0 where an index is out of range
        const int r = a.order ? a.order[tl.first + c] : tl.first + c;
        return (unsigned)r < (unsigned)rows ? (float)base[(int64_t)r * ld + col] : 0.0f;
    };
    if constexpr (kWide) {
#pragma unroll
        for (int i = 0; i < FP; ++i) {
            const int p = pw + 16 * i + fr, row = kPCols ? p0 + p : rows_lds[p];
            const bool valid = kPCols ? row < n_p : row >= 0;
            plain_sums(
                acc[i], valid, [](int, int) { return 0.0f; }, n_c,
                [&](int c) { return !valid ? 0.0f : kPCols ? plain_element(P, a.ld_p, c, row) : (float)P[(int64_t)row * a.ld_p + c]; },
                [&](int c, int j) {
                    const int q = q0 + qw + 16 * j + fr;
                    if (q >= n_q) return 0.0f;
                    return PRODUCT == kGradWeight ? plain_element(Q, a.ld_q, c, q)
                                                  : (float)Q[PRODUCT == kForward ? (int64_t)q * a.ld_q + c : (int64_t)c * a.ld_q + q];
                });
        }
    }

    // ---- lane: output row fr of P's fragment i, and of Q's fragments the columns column(j) .. + 3 (paired: of two, eight)
    const T* bias = PRODUCT == kForward && a.bias && !none && split == 0 ? static_cast<const T*>(a.bias) + (int64_t)tl.g * a.n_out : nullptr;
    auto column = [&](int j) { return q0 + qw + (kPair ? 32 * (j >> 1) + 8 * kg + 4 * (j & 1) : 16 * j + 4 * kg); };
    if (bias)
#pragma unroll
        for (int j = 0; j < FQ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int q = column(j) + e;
                const float b = (float)bias[q < n_q ? q : 0];
#pragma unroll
                for (int i = 0; i < FP; ++i) acc[i][j][e] += b;
            }
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
        if (PRODUCT == kGradWeight && a.chunk_rows) {
#pragma unroll
            for (int j = 0; j < FQ; ++j) store_some<float, 4>(a.part + at, column(j), n_q, [&](int e) { return acc[i][j][e]; });
        } else if (PRODUCT != kGradWeight && a.splits > 1) {
#pragma unroll
            for (int j = 0; j < FQ; ++j)
                store_some<float, 4>(a.part + ((int64_t)split * rows + rows_lds[p]) * n_q, column(j), n_q, [&](int e) { return acc[i][j][e]; });
        } else {
            constexpr int kOnce = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < FQ; j += kOnce / 4)
                store_some<T, kOnce>(static_cast<T*>(a.out) + at, column(j), n_q, [&](int e) { return acc[i][j + (e >> 2)][e & 3]; });
        }
        if (sum_bias) {
            float v = sumb[i] + accb[i];  // of the rows 8 kg .. 8 kg + 7 of every 32
            v += __shfl_xor(v, 16);
            v += __shfl_xor(v, 32);
            if (kWide && !__builtin_isfinite(v)) {  // (the four lanes of a column agree)
                v = 0.0f;
#pragma unroll 8
                for (int c = kg; c < n_c; c += 4) v += plain_element(P, a.ld_p, c, p0 + p);
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
            }
            if (kg != 0) continue;
            if (a.chunk_rows) a.part[(int64_t)a.chunks * a.n_out * a.n_in + (int64_t)run * a.n_out + p0 + p] = v;
            else static_cast<T*>(a.dbias)[(int64_t)tl.g * a.n_out + p0 + p] = (T)v;
        }
    }
}

// ---- short contractions: the weights stay in LDS, the rows stream through registers ------------------------------------------------
// Forward and dx where the contraction has at most 32 NC elements (a layer of the ensemble's networks, not of wide experts): such a
// product is bound by reading P and writing the output.  A workgroup takes a run of one group's rows and up to `q_tile` outputs; the
// weights of those are in LDS as fragments, lane after lane (a fragment is one conflict-free ds_read_b128), and each wave
// takes 16 rows at a time: their P fragments straight from memory (lane: row l & 15, eight elements from 8 (l >> 4)), no barrier
// between rows.  The next 16 rows are loaded while these are multiplied, their numbers one step before that.
// A lane's results are four columns (m = 4 kg .. 4 kg + 3) of each of a 64-column block's four fragments.  fp32: fragment j holds columns
// 16 j + m.  16-bit: fragments 2 h and 2 h + 1 hold columns 32 h + 8 (m >> 2) + 4 (j & 1) + (m & 3), so that two of them are eight
// consecutive columns.  Either way a lane stores 16 bytes at a time and the four lanes of a row 64 consecutive bytes.
// Measured, bf16, 8 groups, rows gathered by `order`, one product repeated, forward / dx (the tile kernel): 3,650,000 rows 256 -> 128 657 /
// 658 us (735 / 804), 4.3 TB/s; 1,048,576 rows 128 -> 64 93 / 102 (134 / 120), 64 -> 1 39 / 34 (95 / 77), 11 -> 256 158 / 150 (200 / 197).  Rows in
// order: 64 -> 1 32 / 30, the others 0 to 10 % less.  The 134 MB of 64 columns stay in the last-level cache between such calls; within a training
// step 64 -> 1 takes 43 / 37.
constexpr int kStripWaves = 8;
// LDS for a workgroup's weights: two workgroups a CU; fp32, whose registers allow one, most of it
template <typename T>
constexpr int strip_lds() { return sizeof(T) == 4 ? 96 * 1024 : 64 * 1024; }

template <typename T, int PRODUCT, int NC>
__global__ __launch_bounds__(64 * kStripWaves, sizeof(T) == 4 ? 2 : 4) void grouped_strip_kernel(Args a, int q_tile, int run_rows) {
    typedef Frag<T> F;
    typedef typename F::V V;
    constexpr int PL = F::kPlanes, NT = 64 * kStripWaves;
    extern __shared__ __attribute__((aligned(16))) char smem[];  // [plane][64-column block][4 j][NC][64 lanes] 16 bytes, then float bias[q_tile]
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, fr = lane & 15, kg = lane >> 4, rows = (int)a.rows;
    const int n_q = PRODUCT == kForward ? a.n_out : a.n_in, n_c = PRODUCT == kForward ? a.n_in : a.n_out;
    const int q_tiles = (n_q + q_tile - 1) / q_tile;
    const int64_t id = xcd_order(blockIdx.x, gridDim.x);  // the q tiles of a run of rows are neighbours
    const Tile tl = find_tile(a.offsets, a.G, rows, (int)(id / q_tiles), run_rows);
    if (tl.g < 0) return;
    const int q0 = (int)(id % q_tiles) * q_tile, width = n_q - q0 < q_tile ? n_q - q0 : q_tile, blocks = (width + 63) / 64;
    const int plane_bytes = blocks * 4 * NC * 1024;
    const bool none = tl.g == a.G;
    const T* const P = static_cast<const T*>(a.p);
    const T* const W = static_cast<const T*>(a.q) + (none ? 0 : (int64_t)tl.g * a.n_in * a.n_out);
    float* const bias = reinterpret_cast<float*>(smem + PL * plane_bytes);

    // ---- weights and bias -> LDS.  Piece (column, eight contraction elements): consecutive lanes take consecutive columns in dx (W's
    // rows are read along), consecutive chunks of a column in the forward pass
    for (int i = t; i < blocks * 64 * NC * 4; i += NT) {
        const int col = PRODUCT == kForward ? i / (NC * 4) : i % (blocks * 64), ch = PRODUCT == kForward ? i % (NC * 4) : i / (blocks * 64);
        const int c = 8 * ch, q = q0 + col;
        const bool have = !none && q < n_q;
        Piece<T> u;
        if (PRODUCT == kForward) {
            u = load_piece(W + (have ? (int64_t)q * a.ld_q + c : 0), have ? n_c - c : 0);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) u.v[e] = have && c + e < n_c ? W[(int64_t)(c + e) * a.ld_q + q] : (T)0.0f;
        }
        const int in = col & 63, j = sizeof(T) == 4 ? in >> 4 : 2 * (in >> 5) + ((in >> 2) & 1);
        const int m = sizeof(T) == 4 ? in & 15 : 4 * ((in >> 3) & 3) + (in & 3);
        store_piece(smem + ((((col >> 6) * 4 + j) * NC + (ch >> 2)) * 64 + (ch & 3) * 16 + m) * 16, plane_bytes, u);
    }
    for (int i = t; i < blocks * 64; i += NT)
        bias[i] = PRODUCT == kForward && a.bias && !none && q0 + i < n_q ? (float)static_cast<const T*>(a.bias)[(int64_t)tl.g * a.n_out + q0 + i] : 0.0f;
    __syncthreads();

    auto row_of = [&](int first) { return first + fr < tl.last ? row_at(a, first + fr) : -1; };
    auto load_one = [&](int row, int k) {
        const T* const at = P + (int64_t)(row < 0 ? 0 : row) * a.ld_p + 8 * kg + 32 * k;
        const int n = row < 0 || none ? 0 : n_c - 8 * kg - 32 * k;
        return n_c % 8 == 0 ? load_eight(at, n) : load_through(at, n, row + 1 < rows && 32 * k + 8 * kg + 8 <= a.ld_p + n_c);
    };
    auto load_rows = [&](int row, Piece<T> (&u)[NC]) {
        if (n_c % 8 == 0) {
#pragma unroll
            for (int k = 0; k < NC; ++k) u[k] = load_one(row, k);
        } else {
#pragma unroll
            for (int k = 0; k < NC; ++k) u[k] = load_one(row, k);
        }
    };
    auto column = [&](int b, int j) { return 64 * b + (sizeof(T) == 4 ? 16 * j + 4 * kg : 32 * (j >> 1) + 8 * kg + 4 * (j & 1)); };
    constexpr int kStep = 16 * kStripWaves;
    int first = tl.first + 16 * wave;
    int row = row_of(first), row_next = row_of(first + kStep);
    Piece<T> u[NC];
    load_rows(row, u);
    for (; first < tl.last; first += kStep) {
        const int out_row = row;
        const bool more = first + kStep < tl.last;
        row = row_next;
        T* const out = static_cast<T*>(a.out) + (int64_t)(out_row < 0 ? 0 : out_row) * n_q + q0;
        V p[sizeof(T) == 4 ? 1 : NC];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < NC; ++k) __builtin_memcpy(&p[k], u[k].v, 16);
            if (more) load_rows(row, u);
        }
        if (more) row_next = row_of(first + 2 * kStep);
        for (int b = 0; b < blocks; ++b) {
            f32x4 acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = *reinterpret_cast<const f32x4*>(bias + column(b, j));
            const char* w = smem + (b * 4 * NC * 64 + lane) * 16;
#pragma unroll
            for (int k = 0; k < NC; ++k) {
                V q[PL];
                if constexpr (sizeof(T) == 2) {
                    q[0] = p[k];
                } else {  // split where it is used (behind an empty asm statement): the planes of all k would not fit the registers
#pragma unroll
                    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(u[k].v[e]));
                    char planes[PL * 16];
                    store_piece(planes, 16, u[k]);
                    if (b + 1 == blocks && more) {
                        int next = row;
                        asm volatile("" : "+v"(next));
                        u[k] = load_one(next, k);
                    }
#pragma unroll
                    for (int l = 0; l < PL; ++l) __builtin_memcpy(&q[l], planes + 16 * l, 16);
                }
#pragma unroll
                for (int l = PL - 1; l >= 0; --l)  // small products first, as in the tile kernel
#pragma unroll
                    for (int m = PL - 1 - l; m >= 0; --m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] = F::mfma(*reinterpret_cast<const V*>(w + m * plane_bytes + (j * NC + k) * 1024), q[l], acc[j]);
                if (sizeof(T) == 4) __builtin_amdgcn_sched_barrier(0);  // (all k's splits and reads at once would not fit the registers)
            }
            if constexpr (sizeof(T) == 4)
                plain_sums(
                    acc, out_row >= 0 && !none, [&](int j, int e) { return bias[column(b, j) + e]; }, n_c,
                    [&](int c) { return out_row < 0 ? 0.0f : (float)P[(int64_t)out_row * a.ld_p + c]; },
                    [&](int c, int j) {
                        const int q = q0 + 64 * b + 16 * j + fr;
                        if (q >= n_q) return 0.0f;
                        return (float)W[PRODUCT == kForward ? (int64_t)q * a.ld_q + c : (int64_t)c * a.ld_q + q];
                    });
            if (out_row < 0) continue;
            constexpr int kOnce = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 4; j += kOnce / 4) store_some<T, kOnce>(out, column(b, j), width, [&](int e) { return acc[j + (e >> 2)][e & 3]; });
        }
    }
}

// ---- dW where one side is a handful of columns (the output layer, the first layer) ------------------------------------------------
// dW[t][c] = sum_r thin[r][t] wide[r][c], at most 16 columns t: bound by reading the wide rows once.  On matrix instructions of
// 16 x 16 outputs whose lane (fr, kg) holds kRows rows of one column: it loads its 8 columns 8 fr .. of rows kRows kg + r of both in
// whole accesses (16 lanes read a row's 128 columns side by side), and instruction j takes column 8 fr + j of them, so nothing is
// turned through LDS.  16-bit: 16 rows an instruction, four rows' halves brought together; fp32: the fp32 instruction, 4 rows.
// Four waves take turns at 64 rows of a run and meet in LDS in their order.  1,048,576 rows, 8 groups, bf16, with the chunks' sum
// (the tile kernel), rows gathered by `order`: 64 -> 1 48 us (188), 2.8 TB/s, within a training step 50 and 5 for the sum; 64 -> 16 50 (67);
// 11 -> 256 126 (203), 4.4 TB/s.  Rows in order: 45, 46, 115.
// THIN_OUT: thin = dy (n_out columns), db is its column sum; otherwise thin = x (n_in <= 15), and db comes from a column of ones.
template <typename T>
struct ThinFrag;
template <>
struct ThinFrag<float> {
    typedef float V;
    static constexpr int kRows = 1;
    static __device__ __forceinline__ void put(V& v, int, float x) { v = x; }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, d, 0, 0, 0); }
};
template <>
struct ThinFrag<__bf16> {
    typedef s16x4 V;
    static constexpr int kRows = 4;
    static __device__ __forceinline__ void put(V& v, int r, __bf16 x) { v[r] = __builtin_bit_cast(short, x); }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, d, 0, 0, 0); }
};
template <>
struct ThinFrag<_Float16> {
    typedef _Float16 V __attribute__((ext_vector_type(4)));
    static constexpr int kRows = 4;
    static __device__ __forceinline__ void put(V& v, int r, _Float16 x) { v[r] = x; }
    static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 d) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, d, 0, 0, 0); }
};
constexpr int kThinMost = 16;
constexpr int kThinCols = 128;

template <typename T, bool THIN_OUT>
__global__ __launch_bounds__(256) void grouped_thin_kernel(Args a) {
    __shared__ float sums[4][kThinMost][kThinCols];
    __shared__ float sums_b[4][kThinMost];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, fr = lane & 15, kg = lane >> 4, rows = (int)a.rows;
    const T* const thin = static_cast<const T*>(THIN_OUT ? a.p : a.q);
    const T* const wide = static_cast<const T*>(THIN_OUT ? a.q : a.p);
    const int64_t ld_t = THIN_OUT ? a.ld_p : a.ld_q, ld_w = THIN_OUT ? a.ld_q : a.ld_p;
    const int n_t = THIN_OUT ? a.n_out : a.n_in, n_w = THIN_OUT ? a.n_in : a.n_out;
    const int col_blocks = (n_w + kThinCols - 1) / kThinCols, run = blockIdx.x / col_blocks, w0 = blockIdx.x % col_blocks * kThinCols;
    Tile tl;
    if (a.chunk_rows) {
        tl = find_tile(a.offsets, a.G, rows, run, a.chunk_rows);
        if (tl.g < 0 || tl.g >= a.G || run >= a.chunks) return;
    } else {
        tl.g = run;
        runs_of(a.offsets, a.G, rows, run, 1, tl.first, tl.last);
    }
    const int c = w0 + 8 * fr;
    f32x4 acc[8] = {};
    float sum_b = 0.0f;
    typedef ThinFrag<T> F;
    constexpr int KR = F::kRows, kSteps = 64 / (4 * KR), kAtOnce = KR == 1 ? 4 : 2;  // loads in flight: 4 (fp32: of 32 bytes), 8 rows a lane
    int mine = tl.first + 64 * wave + lane < tl.last ? row_at(a, tl.first + 64 * wave + lane) : -1;
    for (int first = tl.first + 64 * wave; first < tl.last; first += 256) {
        const int next = first + 256 + lane < tl.last ? row_at(a, first + 256 + lane) : -1;
#pragma unroll 1
        for (int s0 = 0; s0 < kSteps; s0 += kAtOnce) {
            Piece<T> w[kAtOnce][KR];
            T th[kAtOnce][KR];
            int row[kAtOnce][KR];
#pragma unroll
            for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
                for (int r = 0; r < KR; ++r) {
                    row[s][r] = __shfl(mine, 4 * KR * (s0 + s) + KR * kg + r);
                    th[s][r] = *(row[s][r] >= 0 && fr < n_t ? thin + (int64_t)row[s][r] * ld_t + fr : reinterpret_cast<const T*>(kZeros));
                }
            if (n_w % 8 == 0) {
#pragma unroll
                for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
                    for (int r = 0; r < KR; ++r) w[s][r] = load_eight(wide + (int64_t)row[s][r] * ld_w + c, row[s][r] < 0 ? 0 : n_w - c);
            } else {
#pragma unroll
                for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
                    for (int r = 0; r < KR; ++r)
                        w[s][r] = load_through(wide + (int64_t)row[s][r] * ld_w + c, row[s][r] < 0 ? 0 : n_w - c, row[s][r] + 1 < rows && c + 8 <= ld_w + n_w);
            }
#pragma unroll
            for (int s = 0; s < kAtOnce; ++s) {
                typename F::V tv;
#pragma unroll
                for (int r = 0; r < KR; ++r) {
                    if (!THIN_OUT && fr == n_t) th[s][r] = row[s][r] >= 0 ? (T)1.0f : (T)0.0f;
                    if (THIN_OUT) sum_b += (float)th[s][r];
                    F::put(tv, r, th[s][r]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    typename F::V wv;
#pragma unroll
                    for (int r = 0; r < KR; ++r) F::put(wv, r, w[s][r].v[j]);
                    acc[j] = F::mfma(tv, wv, acc[j]);
                }
            }
        }
        mine = next;
    }
    // lane: thin columns 4 kg + i, wide columns 8 fr + j
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[wave][4 * kg + i][8 * fr + j] = acc[j][i];
    sum_b += __shfl_xor(sum_b, 16);
    sum_b += __shfl_xor(sum_b, 32);
    if (kg == 0) sums_b[wave][fr] = sum_b;
    __syncthreads();
    const int64_t n = (int64_t)a.n_out * a.n_in, at = (int64_t)run * n, at_b = (a.chunk_rows ? (int64_t)a.chunks * n : 0) + (int64_t)run * a.n_out;
    auto put = [&](bool b, int64_t i, float v) {
        if (a.chunk_rows) a.part[i] = v;
        else static_cast<T*>(b ? a.dbias : a.out)[i] = (T)v;
    };
    for (int i = t; i < kThinMost * kThinCols; i += 256) {
        const int th = THIN_OUT ? i / kThinCols : i % kThinMost, w = THIN_OUT ? i % kThinCols : i / kThinMost;
        if (w0 + w >= n_w) continue;
        const float v = sums[0][th][w] + sums[1][th][w] + sums[2][th][w] + sums[3][th][w];
        if (th < n_t) put(false, at + (THIN_OUT ? (int64_t)th * a.n_in + w0 + w : (int64_t)(w0 + w) * a.n_in + th), v);
        else if (!THIN_OUT && a.dbias && th == n_t) put(true, at_b + w0 + w, v);
    }
    if (THIN_OUT && a.dbias && w0 == 0 && t < n_t) put(true, at_b + t, sums_b[0][t] + sums_b[1][t] + sums_b[2][t] + sums_b[3][t]);
}

// dW[g] = the sum of group g's chunks, in 64 bits (free: the kernel waits for memory); the same for db.  A workgroup sums 256 / SLICES
// elements of one group: each slice of the chunks in its order, then the slices in theirs.
template <typename T, int SLICES>
__global__ __launch_bounds__(kThreads) void grouped_sum_kernel(Args a) {
    constexpr int kElems = kThreads / SLICES;
    __shared__ double part[SLICES][kElems];
    const int64_t n = (int64_t)a.n_out * a.n_in, all = n + (a.dbias ? a.n_out : 0);
    const int64_t blocks = (all + kElems - 1) / kElems;
    const int g = (int)(blockIdx.x / blocks), e = threadIdx.x % kElems, slice = threadIdx.x / kElems;
    const int first = runs_before(a.offsets, a.G, g, (int)a.rows, a.chunk_rows);
    int b, end;
    end = first + runs_of(a.offsets, a.G, (int)a.rows, g, a.chunk_rows, b, end);
    const int last = end < a.chunks ? end : a.chunks;
    const int64_t i = (int64_t)(blockIdx.x % blocks) * kElems + e;
    double s = 0.0;
    if (i < all) {
        const float* src = i < n ? a.part + i : a.part + (int64_t)a.chunks * n + (i - n);
        const int64_t step = i < n ? n : a.n_out;
#pragma unroll 8
        for (int c = first + slice; c < last; c += SLICES) s += (double)src[c * step];
    }
    if (SLICES > 1) {
        part[slice][e] = s;
        __syncthreads();
        if (slice != 0) return;
        for (int k = 1; k < SLICES; ++k) s += part[k][e];
    }
    if (i >= all) return;
    if (i < n) static_cast<T*>(a.out)[g * n + i] = (T)s;
    else static_cast<T*>(a.dbias)[(int64_t)g * a.n_out + (i - n)] = (T)s;
}

// y or dx = the sum of a split contraction's parts, in their order
template <typename T>
__global__ __launch_bounds__(kThreads) void grouped_join_kernel(const float* __restrict__ part, int splits, int64_t n, T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    float s = part[i];
    for (int k = 1; k < splits; ++k) s += part[k * n + i];
    out[i] = (T)s;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// 256 x 256 outputs a workgroup read each operand half as often as 128 x 128 (32,768 rows, 8 groups, 4096 x 4096: 1,043 / 1,076 / 1,114 us
// against 1,289 / 1,380 / 1,577), but there is one workgroup a CU, and it is not worth its start where few tiles or few rows fill it:
// less than a tile a CU (dW of 1024 x 1024, 8 groups: 74 us against 54; of 512 x 512 in chunks: 160 against 117), groups below a tile
// (125 rows each, 1024 x 1024: 27 against 18 us).  Between (1024 x 1024, 2,000 rows a group) the two are within 10 %.
struct Shape {
    int bp, bq;
};
Shape shape_of(int product, bool dma, int64_t rows, int G, int n_in, int n_out) {
    const int64_t n_p = product == kGradWeight ? n_out : rows / G, n_q = product == kForward ? n_out : n_in;
    const int64_t tiles = (product == kGradWeight ? (int64_t)ceil_div(n_out, 256) * G : rows / 256) * ceil_div(n_q, 256);
    return dma && n_p >= 192 && n_q >= 192 && tiles >= 256 ? Shape{256, 256} : Shape{128, 128};
}

// rows per partial sum of dW: 0 (no split) when the output tiles alone fill the chip (65,536 rows, 8 groups, 512 x 512: 161 us whole, 88
// in chunks; 1,048,576 rows 128 -> 64: 2,687 and 88)
int chunk_rows_of(int64_t rows, int G, int n_in, int n_out) {
    const int64_t tiles = (int64_t)ceil_div(n_out, 128) * ceil_div(n_in, 128);
    if (tiles * G >= 512 || rows <= 512) return 0;
    // as many as run at once, two workgroups a CU, counting the short chunk that ends each group: no tail, and no more partial sums
    // than that takes (524,288 rows, 8 groups, 256 x 128 fp32: 289 us, twice as many chunks 333)
    int64_t per = ceil_div(rows * tiles, tiles * G < 256 ? 512 - tiles * G : 256);
    per = (per + 255) / 256 * 256;
    return per >= rows ? 0 : (int)per;
}
int chunks_of(int64_t rows, int G, int per) { return (int)(rows / per + (G < rows ? G : rows)); }

int check_grid(int64_t blocks, int threads) {  // a launch counts its threads in 32 bits
    MCMC_REQUIRE(blocks * threads <= 0xFFFFFFFFLL, "rows, groups and widths are too large for one call (%lld workgroups)", (long long)blocks);
    return MCMC_OK;
}

template <typename T, int PRODUCT, int BP, int BQ, int WP, int WQ, bool DMA, int BC, int STAGES>
int launch_tile(unsigned blocks, const Args& a, hipStream_t s) {
    const size_t lds = (size_t)STAGES * (BP + BQ) * BC * 2 * Frag<T>::kPlanes + (PRODUCT == kGradWeight ? 2 * kSegment : BP) * sizeof(int);
    const auto kern = grouped_tile_kernel<T, PRODUCT, BP, BQ, WP, WQ, DMA, BC, STAGES>;
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
    if constexpr (sizeof(T) == 2) {
        if (sh.bp == 256) return launch_tile<T, PRODUCT, 256, 256, 2, 4, true, 64, 2>(blocks, a, s);
        if (dma) return launch_tile<T, PRODUCT, 128, 128, 2, 2, true, 64, 2>(blocks, a, s);
        return launch_tile<T, PRODUCT, 128, 128, 2, 2, false, 32, 2>(blocks, a, s);
    } else {
        return launch_tile<T, PRODUCT, 128, 128, 2, 2, false, 32, 1>(blocks, a, s);
    }
}

// The strip kernel for contractions of up to 256 elements whose weights fit the workgroups' LDS: all of them, or, where the contraction
// is so short (64) that reading P again for every q_tile columns costs little beside the output, any number (524,288 rows 256 -> 128 fp32,
// two tiles: 353 us, the tile kernel 308).
// Returns 0 where the tile kernel is to run.
template <typename T>
int strip_q_tile(int n_c, int n_q) {
    const int steps = ceil_div(n_c, 32), nc = steps <= 1 ? 1 : steps <= 2 ? 2 : steps <= 4 ? 4 : 8;
    const int tile = strip_lds<T>() / (nc * 64 * Frag<T>::kPlanes) / 64 * 64;
    if (steps > 8 || (n_q > tile && nc > 2)) return 0;
    return ceil_div(n_q, 64) * 64 < tile ? ceil_div(n_q, 64) * 64 : tile;
}

template <typename T, int PRODUCT, int NC>
int launch_strip_n(const Args& a, int q_tile, int run, unsigned blocks, hipStream_t s) {
    const size_t lds = (size_t)NC * 64 * Frag<T>::kPlanes * q_tile + q_tile * sizeof(float);
    const auto kern = grouped_strip_kernel<T, PRODUCT, NC>;
    if (int rc = ensure_dyn_lds((const void*)kern, lds, "grouped_strip_kernel")) return rc;
    kern<<<blocks, 64 * kStripWaves, lds, s>>>(a, q_tile, run);
    return check_launch("grouped_strip_kernel");
}

struct Strip {
    int run;         // rows per workgroup
    int64_t blocks;
};
// Rows per workgroup, whole turns of its waves: eight times the bytes of its weights in LDS and 4 KB, for what it costs to start (a workgroup
// with fewer rows spends its time there, one with more leaves a long tail: 1,048,576 rows 11 -> 256 bf16, rule 256: 1,024 rows 203 us, 256 rows 166;
// 256 -> 11 fp32, rule 640: 128 rows 481, 256 rows 402, 640 rows 335, 1,024 rows 351), but no fewer workgroups than 1,024 as long as each has a turn.
template <typename T>
Strip strip_of(int64_t rows, int G, int n_c, int n_q, int q_tile) {
    const int nc = n_c <= 32 ? 1 : n_c <= 64 ? 2 : n_c <= 128 ? 4 : 8;
    const int64_t weights = (int64_t)nc * 64 * Frag<T>::kPlanes * q_tile, row = (int64_t)sizeof(T) * (n_c + (n_q < q_tile ? n_q : q_tile));
    constexpr int kTurn = 16 * kStripWaves;
    int64_t run = 8 * (weights + 4096) / row;
    run = rows / 1024 < run ? rows / 1024 : run;
    run = run / kTurn * kTurn;
    run = run < kTurn ? kTurn : run;
    return Strip{(int)run, (rows / run + (G + 1 < rows ? G + 1 : rows)) * ceil_div(n_q, q_tile)};
}

template <typename T, int PRODUCT>
int launch_strip(const Args& a, int q_tile, hipStream_t s) {
    const int n_q = PRODUCT == kForward ? a.n_out : a.n_in, n_c = PRODUCT == kForward ? a.n_in : a.n_out;
    const Strip p = strip_of<T>(a.rows, a.G, n_c, n_q, q_tile);
    if (int rc = check_grid(p.blocks, 64 * kStripWaves)) return rc;
    if (n_c <= 32) return launch_strip_n<T, PRODUCT, 1>(a, q_tile, p.run, (unsigned)p.blocks, s);
    if (n_c <= 64) return launch_strip_n<T, PRODUCT, 2>(a, q_tile, p.run, (unsigned)p.blocks, s);
    if (n_c <= 128) return launch_strip_n<T, PRODUCT, 4>(a, q_tile, p.run, (unsigned)p.blocks, s);
    return launch_strip_n<T, PRODUCT, 8>(a, q_tile, p.run, (unsigned)p.blocks, s);
}

// Parts of a long contraction (forward, dx) where the output has too few tiles to fill the chip: a step of one workgroup waits for
// memory, so 64 of them take 30 us on however few tiles.  4096 -> 512, 8 rows in 2 groups: 30 us whole, 15 in parts with the launch
// that joins them; up to 1,024 elements the joining costs more than the steps (512 -> 512, 1,000 rows: 10 us whole, 16 in parts).
struct Split {
    int parts, c;
};
template <typename T>
Split split_of(int product, int64_t rows, int G, int n_in, int n_out) {
    const int n_c = product == kForward ? n_in : n_out, n_q = product == kForward ? n_out : n_in;
    const int64_t tiles = (rows / 128 + (G + 1 < rows ? G + 1 : rows)) * ceil_div(n_q, 128);
    if (product == kGradWeight || rows == 0 || strip_q_tile<T>(n_c, n_q) || tiles >= 256 || n_c < (sizeof(T) == 4 ? 1024 : 1536)) return Split{1, n_c};
    int64_t parts = 512 / tiles;
    parts = parts > 16 ? 16 : parts;
    parts = parts > n_c / 256 ? n_c / 256 : parts;
    const int c = ceil_div(ceil_div(n_c, parts), 64) * 64;
    return Split{ceil_div(n_c, c), c};
}

// From 64 groups on every workgroup of a forward or dx product walks the offsets, 64 groups a step of 0.3 us, twice: with as many groups as
// rows the time grows with their square (64 -> 64 bf16: 4,096 groups, 8,192 rows 0.25 ms; 65,536 and 65,536 rows 56 ms; 2^20 and 2^20 would
// take 14 s).  What would take more than a few seconds is refused; 4,096 workgroups count as the least, which one walk takes as well.
template <typename T>
int check_walks(int product, int64_t rows, int G, int n_in, int n_out) {
    if (product == kGradWeight || G < 64 || rows == 0) return MCMC_OK;
    const int n_c = product == kForward ? n_in : n_out, n_q = product == kForward ? n_out : n_in, q_tile = strip_q_tile<T>(n_c, n_q);
    int64_t blocks = q_tile ? strip_of<T>(rows, G, n_c, n_q, q_tile).blocks
                            : (rows / 128 + (G + 1 < rows ? G + 1 : rows)) * ceil_div(n_q, 128) * split_of<T>(product, rows, G, n_in, n_out).parts;
    blocks = blocks < 4096 ? 4096 : blocks;
    MCMC_REQUIRE(blocks <= ((int64_t)1 << 38) / G, "%d groups are too many for %lld rows: their offsets would be searched for seconds", G, (long long)rows);
    return MCMC_OK;
}

template <typename T>
int launch(int product, Args a, hipStream_t s) {
    const int n_q = product == kForward ? a.n_out : a.n_in;
    if (product != kGradWeight) {
        if (const int q_tile = strip_q_tile<T>(product == kForward ? a.n_in : a.n_out, n_q))
            return product == kForward ? launch_strip<T, kForward>(a, q_tile, s) : launch_strip<T, kGradInput>(a, q_tile, s);
    }
    const Split split = split_of<T>(product, a.rows, a.G, a.n_in, a.n_out);
    a.splits = split.parts;
    a.split_c = split.c;
    const bool dma = sizeof(T) == 2 && whole_chunks(product, a);
    const Shape sh = shape_of(product, dma, a.rows, a.G, a.n_in, a.n_out);
    const int64_t runs = product == kGradWeight ? (int64_t)ceil_div(a.n_out, sh.bp) * (a.chunk_rows ? a.chunks : a.G)
                                                : (a.rows / sh.bp + (a.G + 1 < a.rows ? a.G + 1 : a.rows)) * a.splits;
    const int64_t blocks = runs * ceil_div(n_q, sh.bq);
    if (int rc = check_grid(blocks, sh.bp == 256 ? 512 : 256)) return rc;
    if (product != kGradWeight) {
        if (int rc = product == kForward ? launch_product<T, kForward>(a, sh, dma, (unsigned)blocks, s)
                                         : launch_product<T, kGradInput>(a, sh, dma, (unsigned)blocks, s))
            return rc;
        if (a.splits == 1) return MCMC_OK;
        const int64_t n = a.rows * n_q, joins = (n + kThreads - 1) / kThreads;
        if (int rc = check_grid(joins, kThreads)) return rc;
        grouped_join_kernel<T><<<(unsigned)joins, kThreads, 0, s>>>(a.part, a.splits, n, static_cast<T*>(a.out));
        return check_launch("grouped_join_kernel");
    }
    const bool thin_out = a.n_out <= kThinMost;
    if (thin_out || a.n_in < kThinMost) {
        const int64_t thin = (int64_t)ceil_div(thin_out ? a.n_in : a.n_out, kThinCols) * (a.chunk_rows ? a.chunks : a.G);
        if (int rc = check_grid(thin, 256)) return rc;
        if (thin_out) grouped_thin_kernel<T, true><<<(unsigned)thin, 256, 0, s>>>(a);
        else grouped_thin_kernel<T, false><<<(unsigned)thin, 256, 0, s>>>(a);
        if (int rc = check_launch("grouped_thin_kernel")) return rc;
    } else if (int rc = launch_product<T, kGradWeight>(a, sh, dma, (unsigned)blocks, s)) {
        return rc;
    }
    if (!a.chunk_rows) return MCMC_OK;
    // few chunks a group: a thread sums them all; many: eight threads share them (1,048,576 rows in one group, 504 chunks, 64 -> 1: 49 us
    // in all, 65 with one thread; up to 64 chunks the same)
    const int slices = a.chunks / a.G > 16 ? 8 : 1;
    const int64_t sums = ((int64_t)a.n_out * a.n_in + (a.dbias ? a.n_out : 0) + kThreads / slices - 1) / (kThreads / slices) * a.G;
    if (int rc = check_grid(sums, kThreads)) return rc;
    if (slices == 8) grouped_sum_kernel<T, 8><<<(unsigned)sums, kThreads, 0, s>>>(a);
    else grouped_sum_kernel<T, 1><<<(unsigned)sums, kThreads, 0, s>>>(a);
    return check_launch("grouped_sum_kernel");
}

int launch_typed(int dtype, int product, const Args& a, hipStream_t s) {
    if (dtype == MCMC_DT_F32) return launch<float>(product, a, s);
    if (dtype == MCMC_DT_BF16) return launch<__bf16>(product, a, s);
    return launch<_Float16>(product, a, s);
}

}  // namespace

int launch_grouped_linear_forward(int dtype, const void* x, int64_t ld_x, int64_t rows, const int* order, const int* offsets, int G, int n_in,
                                  int n_out, const void* weight, const void* bias, void* y, void* ws, hipStream_t s) {
    return launch_typed(dtype, kForward,
                        Args{x, weight, bias, y, nullptr, static_cast<float*>(ws), order, offsets, ld_x, n_in, rows, G, n_in, n_out, 0, 0, 1, 0}, s);
}

int launch_grouped_linear_grad_input(int dtype, const void* dy, int64_t ld_dy, int64_t rows, const int* order, const int* offsets, int G, int n_in,
                                     int n_out, const void* weight, void* dx, void* ws, hipStream_t s) {
    return launch_typed(dtype, kGradInput,
                        Args{dy, weight, nullptr, dx, nullptr, static_cast<float*>(ws), order, offsets, ld_dy, n_in, rows, G, n_in, n_out, 0, 0, 1, 0}, s);
}

// < 0: an error, for calls that are refused
int64_t grouped_linear_workspace_bytes(int product, int dtype, int64_t rows, int G, int n_in, int n_out) {
    if (product == kGradWeight) {
        const int per = chunk_rows_of(rows, G, n_in, n_out);
        return per ? (int64_t)chunks_of(rows, G, per) * ((int64_t)n_in + 1) * n_out * 4 : 0;
    }
    const bool wide = dtype == MCMC_DT_F32;
    if (int rc = wide ? check_walks<float>(product, rows, G, n_in, n_out) : check_walks<__bf16>(product, rows, G, n_in, n_out)) return rc;
    const Split split = wide ? split_of<float>(product, rows, G, n_in, n_out) : split_of<__bf16>(product, rows, G, n_in, n_out);
    return split.parts > 1 ? (int64_t)split.parts * rows * (product == kForward ? n_out : n_in) * 4 : 0;
}

int launch_grouped_linear_grad_weight(int dtype, const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, int64_t rows, const int* order,
                                      const int* offsets, int G, int n_in, int n_out, void* dweight, void* dbias, void* ws, hipStream_t s) {
    const int per = chunk_rows_of(rows, G, n_in, n_out);
    return launch_typed(dtype, kGradWeight,
                        Args{dy, x, nullptr, dweight, dbias, static_cast<float*>(ws), order, offsets, ld_dy, ld_x, rows, G, n_in, n_out, per,
                             per ? chunks_of(rows, G, per) : 0, 1, 0},
                        s);
}

}  // namespace mcmc
