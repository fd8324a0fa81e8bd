// Activation and dropout of one layer as an operator of its own, the mask drawn from the 'MASK' Philox stream where it is used and
// never stored: what the fused kernels do between two linear layers (bayesian_ensemble.py:85-86), for any row width.
//
//   forward   y  = keep ? act(x) * s : 0            s = fp32(1 / (1-p)), act = ELU (alpha 1) or the identity
//   backward  dx = keep ? dy * (act'(x) * s) : 0    act'(x) = x > 0 ? 1 : exp(x); the same mask drawn again
//
// keep of column c of row r: elem = elem_begin + c, block counter (((elem>>4)<<1) | ((elem>>2)&1), pair, 'MASK', row_begin + r),
// slot = 4*((elem>>3)&1) + (elem&3) -> 16-bit half slot&1 of word slot>>1, kept iff it is < floor((1-p) * 65536)
// (dropmask.hpp: the same definition, so a hidden layer of mcmc_train_forward gets the same masks from here).
//
// A block's eight halves belong to columns 0-3 and 8-11 (block 0) or 4-7 and 12-15 (block 1) of a 16-column tile.  A lane owns eight
// CONSECUTIVE columns, so that its accesses are whole 16-byte pieces: it computes one block and swaps two words with its
// neighbour lane, which owns the other eight columns of the tile (unit u = row * units_per_row + column / 8; units_per_row is
// even, so the two lanes always meet).
// A dropped element is +0 whatever x holds, NaN and infinities included (a select, not a product).
//
// Bound: memory, 2 accesses an element forward, 3 backward with an activation.  1,048,576 x 256 bf16 with ELU: forward 200 us, backward
// 295 us, 5.4 TB/s both; 36,501 x 1,001 fp16 (rows that start anywhere): 35 us, 4.2 TB/s.
#include "common.hpp"
#include "elu.hpp"
#include "philox.hpp"

namespace mcmc {

namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 2;  // units per thread, both in flight together

struct DropArgs {
    const void* x;   // forward: input; backward with an activation: the forward's input
    const void* dy;  // backward
    void* out;
    int64_t ld_x, ld_dy, ld_out;  // elements between rows
    int64_t units;                // rows of this launch * units_per_row
    uint32_t units_per_row, width;
    uint64_t seed;
    const uint64_t* seed_dev;     // not NULL: the key is read when the kernel runs
    uint32_t threshold, pair, row_begin, block_begin;
    float scale;
};

// eight elements starting at column c of a row of `width`: one 16-byte access (32 for fp32) where all eight are inside, element
// by element at the row's end.  Rows need only the element's own alignment: gfx950 global accesses may be unaligned.
template <typename T>
__device__ __forceinline__ void load8(const T* row, uint32_t c, uint32_t width, float (&v)[8]) {
    if (c + 8 <= width) {
        T t[8];
        __builtin_memcpy(t, row + c, sizeof(t));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < width ? (float)row[c + i] : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, uint32_t c, uint32_t width, const float (&v)[8]) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];  // the one rounding of a 16-bit result
    if (c + 8 <= width) {
        __builtin_memcpy(row + c, t, sizeof(t));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < width) row[c + i] = t[i];
    }
}

// the value of the neighbouring lane (lane ^ 1): a quad permutation [1,0,3,2]
__device__ __forceinline__ uint32_t neighbour(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true); }

template <typename T, bool ELU, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropArgs a) {
    const uint64_t seed = a.seed_dev ? *a.seed_dev : a.seed;
    const int64_t u0 = (int64_t)blockIdx.x * (kThreads * kUnits);
    const int64_t row0 = u0 / a.units_per_row;
    const uint32_t c0 = (uint32_t)(u0 - row0 * a.units_per_row);
    float x[kUnits][8], g[kUnits][8];
    int64_t row[kUnits];
    uint32_t unit[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const uint32_t d = c0 + threadIdx.x + kThreads * i, q = d / a.units_per_row;
        unit[i] = d - q * a.units_per_row;
        row[i] = row0 + q;
        if (u0 + threadIdx.x + kThreads * i < a.units) {
            if (!BACKWARD || ELU) load8(static_cast<const T*>(a.x) + row[i] * a.ld_x, 8 * unit[i], a.width, x[i]);
            if (BACKWARD) load8(static_cast<const T*>(a.dy) + row[i] * a.ld_dy, 8 * unit[i], a.width, g[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        // unit 2t + b of a row computes block b of tile t (all lanes: the neighbour may need the words)
        const u32x4 w = philox4x32_10(u32x4{a.block_begin + unit[i], a.pair, kTagMask, a.row_begin + (uint32_t)row[i]}, (uint32_t)seed, (uint32_t)(seed >> 32));
        const bool odd = unit[i] & 1;
        const uint32_t r0 = neighbour(odd ? w.x : w.z), r1 = neighbour(odd ? w.y : w.w);
        // columns 0-3 of the unit: block 0's words, columns 4-7: block 1's; the even unit uses words 0,1, the odd one 2,3
        const uint32_t h[4] = {odd ? r0 : w.x, odd ? r1 : w.y, odd ? w.z : r0, odd ? w.w : r1};
        if (u0 + threadIdx.x + kThreads * i >= a.units) continue;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t half = (j & 1) ? h[j >> 1] >> 16 : h[j >> 1] & 0xFFFFu;
            float v;
            if (BACKWARD) {
                // (the factors first: dy * s alone may overflow where the result does not)
                v = g[i][j] * (ELU ? a.scale * (x[i][j] > 0.0f ? 1.0f : __expf(x[i][j])) : a.scale);
            } else {
                v = x[i][j];
                if (ELU) v = v > 0.0f ? v : elu_neg(v);
                v *= a.scale;
            }
            o[j] = half < a.threshold ? v : 0.0f;
        }
        store8(static_cast<T*>(a.out) + row[i] * a.ld_out, 8 * unit[i], a.width, o);
    }
}

// A launch counts its threads in 32 bits: larger calls go row by row in pieces of at most 2^31 threads (2^32 units, at least 16 rows)
constexpr int64_t kMostUnits = (int64_t)1 << 32;

template <typename T>
int launch(DropArgs a, int64_t rows, bool elu, bool backward, hipStream_t s) {
    const int64_t most = kMostUnits / a.units_per_row;
    for (; rows > 0; rows -= most) {
        a.units = (rows < most ? rows : most) * (int64_t)a.units_per_row;
        const dim3 grid((unsigned)((a.units + kThreads * kUnits - 1) / (kThreads * kUnits)));
        if (elu && backward) dropout_kernel<T, true, true><<<grid, kThreads, 0, s>>>(a);
        else if (elu) dropout_kernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
        else if (backward) dropout_kernel<T, false, true><<<grid, kThreads, 0, s>>>(a);
        else dropout_kernel<T, false, false><<<grid, kThreads, 0, s>>>(a);
        if (int rc = check_launch("dropout_kernel")) return rc;
        if (rows <= most) break;
        if (a.x) a.x = static_cast<const T*>(a.x) + most * a.ld_x;
        if (a.dy) a.dy = static_cast<const T*>(a.dy) + most * a.ld_dy;
        a.out = static_cast<T*>(a.out) + most * a.ld_out;
        a.row_begin += (uint32_t)most;
    }
    return MCMC_OK;
}

}  // namespace

int launch_dropout(int dtype, bool elu, bool backward, const void* x, int64_t ld_x, const void* dy, int64_t ld_dy, int64_t rows, int64_t width,
                   uint64_t seed, const uint64_t* seed_dev, float p_drop, uint32_t pair, uint32_t row_begin, uint32_t elem_begin, void* out,
                   int64_t ld_out, hipStream_t s) {
    DropArgs a;
    a.x = x;
    a.dy = dy;
    a.out = out;
    a.ld_x = ld_x;
    a.ld_dy = ld_dy;
    a.ld_out = ld_out;
    a.units_per_row = 2 * (uint32_t)((width + 15) / 16);
    a.width = (uint32_t)width;
    a.seed = seed;
    a.seed_dev = seed_dev;
    a.threshold = (uint32_t)((1.0f - p_drop) * 65536.0f);
    a.pair = pair;
    a.row_begin = row_begin;
    a.block_begin = (elem_begin >> 4) << 1;
    a.scale = (float)(1.0 / (1.0 - (double)p_drop));
    if (dtype == MCMC_DT_F32) return launch<float>(a, rows, elu, backward, s);
    if (dtype == MCMC_DT_BF16) return launch<__bf16>(a, rows, elu, backward, s);
    return launch<_Float16>(a, rows, elu, backward, s);
}

}  // namespace mcmc
