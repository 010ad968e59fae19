// Orthogonalised updates, gfx950: the nearest matrix with singular values near one to a gradient, by Newton-Schulz products,
// and the weight update that takes it as its direction (the Muon rule).  The reference stops at RMSprop per element
// (source/basicOps.cu:1192-1197); this is its counterpart for whole matrices.
//
//   X0 = G / (|G|_F + 1e-7), transposed if G has more rows than columns, so that X is m x n with m <= n
//   steps times:  A = X X^T;  P = b A + c A A;  X <- a X + P X         (a, b, c) = (3.4445, -4.7750, 2.0315)
//
// Every polynomial step maps singular values of at most 1.21 to at most 1.21 and multiplies small ones by 3.4445.
//
// The products are what this costs: 3 m^2 n + m^3 multiply-adds per step after the symmetry of A and A A (only tiles on and
// above the diagonal are computed).  In fp32 the matrix cores give 157 TFLOP/s; here each operand is kept as two fp16
// numbers, x 2^14 = hi + lo (2^10 for P), and a product is the three fp16 products hi hi + hi lo + lo hi in fp32
// accumulators.  What is left out, lo lo, and the rounding of lo are 2^-22 of the product, so the result is about as far from
// the exact one as plain fp32 products leave it.  Root mean square over gradients, five steps, 16 x 3000, 64 x 64, 64 x 16384,
// 140 x 5000, 256 x 6000, 300 x 300, 700 x 2900, 784 x 1024, 1000 x 4001, 2048 x 2048 and 4096 x 4096: 0.2 to 1.4 times as far for
// Gaussian numbers, half of the rows zero, few strong directions; up to 2.4 times (and 1.2 10^-6 of |out|) for gradients
// of one or two rows or of one column, where roundings do not average out.  The factors keep entries below 65504 (|X| <=
// 1.21, |A| <= 1.46, |P| <= 2.81) and lo above the smallest fp16 number for entries down to 2^-13 of
// the largest.  a X stays outside the product, with X read back as hi + lo: folding a into P's diagonal costs a factor of
// three in accuracy for nearly low-rank gradients.
//
// Several steps on m x m matrices alone, with X updated once at their end (A and its polynomials commute; 6.6 ms in place of
// 10.8 for 4096 x 16384), are not sound in these numbers: the polynomial Q of two or three steps has entries of up to 12 or 41 where a
// row has a large singular value to itself, and (a^g + Q) X, of about 1, keeps their rounding: 4 10^-6 to 9 10^-6 of |out| for
// gradients of one or two rows or of one column, up to 11 times plain fp32.
//
// A gradient of 16 bits is its own hi if only the power of two of the scale is applied to it, so X0 X0^T is one product and P X0
// two, with nothing lost but the rounding of the rest of the scale, in [1, 2), which goes to their results (split_kernel).
// (One product in place of three in later steps too is not sound: hi alone is off by up to 2^-11 the same way in all equal entries, such as the
// diagonal of A for orthogonal rows, and the next steps multiply that by ten: 5 10^-3 of |out| for 17 x 498.)
//
// Layout: a matrix is blocks of 256 rows, in them groups of 32 columns: a 128-byte line per row, 32 hi, then 32 lo.  A stage of
// the product is then one line (or two) per row, all of them in a row in memory, and the tile in LDS is the fp32 kernel's
// [row][32 words] with its swizzle (cn_gemm.hip).  All sizes are padded to whole tiles with zeros, so nothing in the
// product needs a bounds check.  X is kept in both orientations (the Gram product sums over n, the update over m), P
// and A are symmetric.
//
// Work split: see `Group` for how tiles go to workgroups, cost_of for which cut of a product is taken.  A workgroup that
// computes a whole tile applies the formula to its accumulators and writes the next operand in both orientations; parts of a
// tile go to memory and a second kernel adds them in order.  Either way the result does not depend on scheduling.
//
// Measured (one MI355X): X^T P of 4096 x 16384 in 1.38 ms, 1.20 PFLOP/s of fp16 products with the write-out of X and X^T in it
// (0.8 GB, of which little overlaps); the library's own 8192^3 fp16 product reaches 1.31 on the same card.  The chip runs
// at its power limit (1.75 GHz on random numbers, 2.1 on zeros), so what would be won by fewer stalls is lost in clock.
#include "cn_dtypes.h"

namespace cn {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kUnit = 16384.0f, kPolyUnit = 1024.0f;  // the stored number for 1: of X and A, and of P
constexpr int kPad = 256;                           // rows and columns are padded to whole tiles

int64_t padded(int64_t n) { return (n + kPad - 1) / kPad * kPad; }

// ---- split numbers -----------------------------------------------------------------------------------------------------
// Element (row, col) of a split matrix of `cols` columns: blocks of 256 rows, in them groups of 32 columns, in them the rows,
// 64 numbers each: 32 hi, then 32 lo.  Returns the place of hi, lo is 32 further.
__device__ __forceinline__ size_t split_at(int64_t row, int64_t col, int64_t cols) {
    return ((size_t)(row >> 8) * (size_t)(cols >> 5) + (size_t)(col >> 5)) * (256 * 64) + (size_t)(row & 255) * 64 + (col & 31);
}
// Four consecutive columns (col a multiple of 4), in stored units.  What a number was computed with is hidden from its
// conversion: a product that becomes fp16 by one fused instruction in the one place and is rounded to fp32 before in the other gave
// two different hi where it was near a tie (one of 10^4 elements of A for 16-bit gradients, each off by 2^-11 of itself).
__device__ __forceinline__ void split_store(f16_t *m, size_t at, const float (&v)[4]) {
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = v[e];
        asm("" : "+v"(x));
        hi[e] = (f16_t)x;
        lo[e] = (f16_t)(x - (float)hi[e]);
    }
    *reinterpret_cast<f16x4 *>(m + at) = hi;
    *reinterpret_cast<f16x4 *>(m + at + 32) = lo;
}

// ---- the update whose direction is wanted ---------------------------------------------------------------------------------
// G itself, or momentum and gradient of a training step.
struct Source {
    const void *grad;          // rows x cols of grad_kind
    int64_t ldg;
    float *momentum;           // rows x cols fp32, or NULL: the update is the gradient
    int64_t ldm;
    float mu;
    int nesterov;
    int64_t rows, cols;
};

// VEC neighbouring elements of what the update is made of, and the update; `advance` moves the momentum on (once per step).
template <int VEC> struct Pieces {
    float g[VEC], m[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_pieces(const Source &s, int64_t r, int64_t c, Pieces<VEC> &p) {
    load_f32<VEC>((const T *)s.grad + r * s.ldg + c, p.g);
    if (s.momentum) load_f32<VEC>(s.momentum + r * s.ldm + c, p.m);
}
template <int VEC>
__device__ __forceinline__ void update_of(const Source &s, Pieces<VEC> &p, bool advance, float (&u)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        if (advance && s.momentum) p.m[e] = s.mu * p.m[e] + p.g[e];
        u[e] = !s.momentum ? p.g[e] : s.nesterov ? p.g[e] + s.mu * p.m[e] : p.m[e];
    }
}

constexpr int kNormBlocks = 2048, kNormRows = 8;

__device__ __forceinline__ double block_sum(double v, double *scratch) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = 0.0;
    for (unsigned w = 0; w < blockDim.x / 64; ++w) sum += scratch[w];
    return sum;
}

// Moves the momentum on and sums the squares of the update, in 64 bits (no overflow for any finite fp32), a part per workgroup.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void norm_kernel(Source s, double *parts) {
    __shared__ double scratch[4];
    double sum = 0.0;
    const int64_t tiles_c = (s.cols + 256 * VEC - 1) / (256 * VEC);
    for (int64_t t = blockIdx.x; t < tiles_c * ((s.rows + kNormRows - 1) / kNormRows); t += gridDim.x) {
        const int64_t r0 = t / tiles_c * kNormRows, c = ((t % tiles_c) * 256 + threadIdx.x) * VEC;
        if (c >= s.cols) continue;
        Pieces<VEC> p[kNormRows];
#pragma unroll
        for (int i = 0; i < kNormRows; ++i)
            if (r0 + i < s.rows) load_pieces<T, VEC>(s, r0 + i, c, p[i]);
#pragma unroll
        for (int i = 0; i < kNormRows; ++i) {
            if (r0 + i >= s.rows) break;
            float u[VEC];
            update_of<VEC>(s, p[i], true, u);
            if (s.momentum) store_f32<VEC>(s.momentum + (r0 + i) * s.ldm + c, p[i].m);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += (double)u[e] * (double)u[e];
        }
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// X0 in both orientations, zeros in the padding.  A workgroup takes 64 x 64 elements of X (m x n).  `exact` (a gradient of 16
// bits): only the power of two of the scale is applied, so that the stored numbers are the gradient's own, hi alone; the rest,
// r in [1, 2), goes to the products of X0: factors = 1, r, r r.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void split_kernel(Source s, const double *parts, int part_count, int flip, int exact, int64_t mp,
                                                    int64_t np, f16_t *x, f16_t *xt, float *factors) {
    __shared__ double scratch[4];
    __shared__ float tile[64][65];
    const int64_t blocks_n = np / 64;
    const int64_t i0 = blockIdx.x / blocks_n * 64, j0 = blockIdx.x % blocks_n * 64;  // of X
    // read along the rows of G, whichever way it lies
    const int64_t r0 = flip ? j0 : i0, c0 = flip ? i0 : j0;
    constexpr int kLanes = 64 / VEC, kReads = 64 * kLanes / 256;
    const int read_row = threadIdx.x / kLanes, read_col = threadIdx.x % kLanes * VEC;
    float u[kReads][VEC];
#pragma unroll
    for (int q = 0; q < kReads; ++q) {
        const int64_t r = r0 + read_row + q * (256 / kLanes), c = c0 + read_col;
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[q][e] = 0.0f;
        if (r < s.rows && c < s.cols) {
            Pieces<VEC> p;
            load_pieces<T, VEC>(s, r, c, p);
            update_of<VEC>(s, p, false, u[q]);
        }
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < part_count; i += 256) sum += parts[i];
    sum = block_sum(sum, scratch);
    double to_unit = (double)kUnit / (sqrt(sum) + 1e-7);
    float rest = 1.0f;
    if (exact && to_unit > 0.0) {  // neither 0 nor NaN: the gradient is finite
        int exponent;
        rest = 2.0f * (float)frexp(to_unit, &exponent);
        to_unit = ldexp(1.0, exponent - 1);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        factors[0] = 1.0f;
        factors[1] = rest;
        factors[2] = rest * rest;
    }
#pragma unroll
    for (int q = 0; q < kReads; ++q)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int a = read_row + q * (256 / kLanes), b = read_col + e;
            const float v = (float)((double)u[q][e] * to_unit);
            if (flip) tile[b][a] = v; else tile[a][b] = v;
        }
    __syncthreads();
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int i = row + 16 * q;
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = tile[i][col + e];
            w[e] = tile[col + e][i];
        }
        split_store(x, split_at(i0 + i, j0 + col, np), v);
        split_store(xt, split_at(j0 + i, i0 + col, mp), w);
    }
}

// ---- products ------------------------------------------------------------------------------------------------------------
// D[i][j] = sum over k of U[i][k] V[j][k], both operands split, and what becomes of it.
enum Finish {
    GRAM = 0,  // y D, symmetric
    POLY = 1,  // x old + y D, symmetric
    STEP = 2,  // X <- x X + y D^T, both orientations; D = X^T P, n x m
    LAST = 3   // the same, into the result
};
//
// Units of work: a group of `count` consecutive tiles, each cut along k into `parts`; workgroup w of a group takes part
// w / count of tile first + (w % count) * rounds, and the rounds - 1 tiles behind it.  So the workgroups of an XCD, which take
// neighbouring w, stream the same k of neighbouring tiles at the same time and share it in their L2.
struct Group {
    int first, count, parts, rounds, slot;  // slot: where its parts begin
};
constexpr int kMaxGroups = 4;
struct Product {
    const f16_t *u, *v;
    int64_t u_cols, v_cols;  // columns of the split matrices (padded)
    int tiles_j;             // tiles along j
    int stages;              // of k
    int triangle;            // the result is symmetric: only tiles with j >= i
    Group group[kMaxGroups];  // unused ones: all 0
    float *parts;            // TILE x TILE numbers per unit of a group with more than one part per tile
    const f16_t *old;        // POLY: A; STEP, LAST: X
    float x, y;              // in stored units
    const float *factor;     // x and y are multiplied by this
    f16_t *to;                // symmetric results; STEP: X (its own elements only, so in place)
    f16_t *to_t;             // STEP: X^T of the next step (this one's is an operand)
    int64_t to_cols, to_t_cols;
    void *out;               // LAST: the result, as the caller has it, or the weights
    int out_dtype;
    int64_t ldo, m, n;
    int flip;                // the caller's matrix is n x m
    int wide;                // its rows allow accesses of four numbers
    int update;              // out = keep * out - rate * X
    float keep, rate;
};

// TILE x TILE results of a workgroup: KS x WM x WN wavefronts of FM x FN blocks of 32 x 32, KS of them on the same blocks, each
// with its share of a stage's k.  A stage is LINES 128-byte lines of every row (one where the products are of one part), DEPTH of
// them are in LDS: 128 KiB in all, one workgroup per compute unit, so that what is in flight covers the way from the L2 even
// where a stage has little to compute.  (64 x 64 with one line a stage: 0.31 us each, mostly the barrier's round trip.)
template <int TILE> struct Shape;
template <> struct Shape<256> { static constexpr int KS = 1, WM = 2, WN = 4, FM = 4, FN = 2, LINES = 1, DEPTH = 2; };
template <> struct Shape<128> { static constexpr int KS = 2, WM = 2, WN = 2, FM = 2, FN = 2, LINES = 2, DEPTH = 2; };
template <> struct Shape<64> { static constexpr int KS = 2, WM = 2, WN = 2, FM = 1, FN = 1, LINES = 2, DEPTH = 4; };
template <int TILE> constexpr int threads_of() { return Shape<TILE>::KS * Shape<TILE>::WM * Shape<TILE>::WN * 64; }
template <int TILE> constexpr int lds_of() { return Shape<TILE>::DEPTH * Shape<TILE>::LINES * 2 * TILE * 128 + threads_of<TILE>() * 64; }
constexpr int lines_of(int tile, int terms) {
    return terms == 1 ? 1 : tile == 256 ? Shape<256>::LINES : tile == 128 ? Shape<128>::LINES : Shape<64>::LINES;
}
// k of a stage.
constexpr int depth_of(int tile, int terms) { return lines_of(tile, terms) * (terms == 1 ? 64 : 32); }

__device__ __forceinline__ int swizzle(int row) { return (row & 7) ^ ((row >> 3) & 3); }

// Tile number to its row and column of tiles; symmetric: row by row, each from the diagonal on.
__device__ __forceinline__ void tile_place(int tile, int tiles_j, bool triangle, int &ti, int &tj) {
    if (!triangle) {
        ti = tile / tiles_j;
        tj = tile - ti * tiles_j;
        return;
    }
    ti = 0;
    int left = tile;
    while (left >= tiles_j - ti) {
        left -= tiles_j - ti;
        ++ti;
    }
    tj = ti + left;
}

// The units of this workgroup, one per group: lane g of every wavefront finds and keeps that of group g.
struct Units {
    int tile;    // ti * 65536 + tj
    int stages;  // begin * 65536 + end
    int slot;    // < 0: whole tiles
    int rounds;  // 0: the group has no unit for this workgroup
    __device__ __forceinline__ Units(const Product &g, int w) {
        tile = stages = slot = rounds = 0;
        const int lane = threadIdx.x & 63;
        if (lane < kMaxGroups) {
            const Group a = g.group[lane];
            if (w < a.count * a.parts) {
                const int part = w / a.count, place = w - part * a.count;
                int ti, tj;
                tile_place(a.first + place * a.rounds, g.tiles_j, g.triangle, ti, tj);
                tile = ti << 16 | tj;
                stages = g.stages * part / a.parts << 16 | g.stages * (part + 1) / a.parts;
                slot = a.parts > 1 ? a.slot + w : -1;
                rounds = a.rounds;
            }
        }
    }
};
// What a workgroup is at: a stage of a unit.  All of it the same for every lane.
struct Cursor {
    int group = -1, ti = 0, tj = 0, stage = 0, end = 0, slot = 0, rounds = 0;
    __device__ __forceinline__ bool next_unit(const Product &g, const Units &u) {
        if (rounds > 1) {  // the next tile, all of it
            --rounds;
            stage = 0;
            if (++tj == g.tiles_j) {
                ++ti;
                tj = g.triangle ? ti : 0;
            }
            return true;
        }
#pragma unroll 1
        while (++group < kMaxGroups) {
            rounds = __builtin_amdgcn_readlane(u.rounds, group);
            if (rounds == 0) continue;
            const int tile = __builtin_amdgcn_readlane(u.tile, group), stages = __builtin_amdgcn_readlane(u.stages, group);
            ti = tile >> 16;
            tj = tile & 0xffff;
            stage = stages >> 16;
            end = stages & 0xffff;
            slot = __builtin_amdgcn_readlane(u.slot, group);
            return true;
        }
        return false;
    }
};

// What a lane needs of an old matrix for a 32 x 32 block: rows j, along i.
struct Old {
    f16x4 hi[4], lo[4];
};
template <int FINISH>
__device__ __forceinline__ void load_old(const Product &g, const f16_t *from, int64_t i0, int64_t j0, Old &o) {
    if (FINISH == GRAM) return;
    const int sub = (threadIdx.x & 63) >> 3, quad = threadIdx.x & 7;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const f16_t *at = from + split_at(j0 + 8 * p + sub, i0 + 4 * quad, g.to_cols);
        o.hi[p] = *reinterpret_cast<const f16x4 *>(at);
        o.lo[p] = *reinterpret_cast<const f16x4 *>(at + 32);
    }
}

// Four numbers of the result, along a row of the caller's matrix.
__device__ __forceinline__ void write_result(const Product &g, int64_t row, int64_t col, const float (&x)[4]) {
    const int64_t rows = g.flip ? g.n : g.m, cols = g.flip ? g.m : g.n, at = row * g.ldo + col;
    if (row >= rows) return;
    if (g.wide && col + 4 <= cols) {
        float w[4] = {x[0], x[1], x[2], x[3]};
        if (g.out_dtype == CN_F32) {
            float *out = (float *)g.out + at;
            if (g.update) {
                float old[4];
                load_f32<4>(out, old);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = g.keep * old[e] - g.rate * w[e];
            }
            store_f32<4>(out, w);
        } else if (g.out_dtype == CN_F16) {
            store_f32<4>((f16_t *)g.out + at, w);
        } else {
            store_f32<4>((bf16_t *)g.out + at, w);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= cols) break;
        if (g.out_dtype == CN_F32) {
            float *out = (float *)g.out + at + e;
            *out = g.update ? g.keep * *out - g.rate * x[e] : x[e];
        } else if (g.out_dtype == CN_F16) {
            ((f16_t *)g.out)[at + e] = (f16_t)x[e];
        } else {
            ((bf16_t *)g.out)[at + e] = (bf16_t)x[e];
        }
    }
}

// One 32 x 32 block of D, corner (i0, j0), from a wavefront's sums as the matrix instructions leave them: number r of lane
// (half, l) is row 8 (r / 4) + 4 half + r % 4, column l.  Matrices are read and written as rows j, along i (symmetric ones may be,
// D = X^T P belongs to row j of X), then, with `mirror`, as rows i, along j.  `stage`: 4 KiB of LDS of the
// wavefront's own, [j][i] in 16-byte columns xor-swizzled by j / 2, so that eight lanes write 64 bytes of a row at a time.
template <int FINISH>
__device__ __forceinline__ void finish_block(const Product &g, float factor, const f32x16 &sum, const Old &old, int64_t i0, int64_t j0,
                                             bool mirror, float *stage) {
    const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4 *>(stage + l32 * 32 + (((2 * q + half) ^ (l32 >> 1)) & 7) * 4) =
            f32x4{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
    const int sub = lane >> 3, quad = lane & 7;
    constexpr bool last = FINISH == LAST;
    const float x = g.x * factor, y = g.y * factor;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int j = 8 * p + sub;
        f32x4 *at = reinterpret_cast<f32x4 *>(stage + j * 32 + ((quad ^ (j >> 1)) & 7) * 4);
        f32x4 v = *at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] *= y;
            if (FINISH != GRAM) v[e] = x * ((float)old.hi[p][e] + (float)old.lo[p][e]) + v[e];
        }
        const float w[4] = {v[0], v[1], v[2], v[3]};
        if (!last) {
            split_store(g.to, split_at(j0 + j, i0 + 4 * quad, g.to_cols), w);
        } else if (!g.flip) {
            const float r[4] = {w[0] * (1.0f / kUnit), w[1] * (1.0f / kUnit), w[2] * (1.0f / kUnit), w[3] * (1.0f / kUnit)};
            write_result(g, j0 + j, i0 + 4 * quad, r);
        }
        *at = v;
    }
    if (last ? !g.flip : !mirror) return;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int i = 8 * p + sub;
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = 4 * quad + e;
            w[e] = stage[j * 32 + (((i >> 2) ^ (j >> 1)) & 7) * 4 + (i & 3)];
            if (last) w[e] *= 1.0f / kUnit;
        }
        if (last) write_result(g, i0 + i, j0 + 4 * quad, w);
        else split_store(FINISH == STEP ? g.to_t : g.to, split_at(i0 + i, j0 + 4 * quad, g.to_t_cols), w);
    }
}

template <int N> struct Constant { static constexpr int value = N; };
// f(Constant<0>) ... f(Constant<N - 1>): registers can only be named by constants.
template <int N, typename F>
__device__ __forceinline__ void for_each(F &&f) {
    if constexpr (N > 0) {
        for_each<N - 1>(f);
        f(Constant<N - 1>{});
    }
}

template <int COUNT>
__device__ __forceinline__ void wait_for_all_but() {  // vmcnt(COUNT)
    __builtin_amdgcn_s_waitcnt(0x0f70 | (COUNT & 15) | ((COUNT >> 4) << 14));
}

// TERMS = 3: hi hi + hi lo + lo hi, a stage is 32 of k.  TERMS = 1: hi hi alone, a stage is 64 of k, the hi halves of two
// groups, in the same place in LDS.
template <int TILE, int TERMS, int FINISH>
__global__ __launch_bounds__(threads_of<TILE>(), 1) void product_kernel(Product g) {
    using S = Shape<TILE>;
    constexpr int kWaves = S::KS * S::WM * S::WN, kLines = lines_of(TILE, TERMS);
    constexpr int kLoads = kLines * TILE / 8 / kWaves;  // 1 KiB loads per operand, stage and wavefront
    extern __shared__ __attribute__((aligned(16))) char smem[];         // [DEPTH][U, V][line][TILE rows][128 bytes], then 4 KiB per wavefront
    constexpr int kOperand = S::LINES * TILE * 128, kMask = S::DEPTH - 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int half = lane >> 5, l32 = lane & 31;
    const int share = wave / (S::WM * S::WN), wave_i = wave % (S::WM * S::WN) / S::WN, wave_j = wave % S::WN;

    // Workgroups of one XCD (ids congruent mod 8) take neighbouring runs and share operands in its L2.
    const unsigned W = gridDim.x, xcd = blockIdx.x % 8u, idx = blockIdx.x / 8u, per = W / 8u, rem = W % 8u;
    const int w = (int)(xcd * per + (xcd < rem ? xcd : rem) + idx);
    const Units units(g, w);
    const float factor = __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(*g.factor)));
    Cursor at, ahead;  // the stage that is computed, the one that is requested next
    bool more = ahead.next_unit(g, units);  // something is left to request
    int requested = 0;                      // stages requested and not yet computed

    uint32_t off[kLoads];  // this lane's 16 bytes of each 1 KiB (8 rows), from the corner of the tile's stage
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int at = (j * kWaves + wave) * 8 + (lane >> 3), row = at % TILE;
        const uint32_t column = (uint32_t)((lane & 7) ^ swizzle(row));
        off[j] = (uint32_t)(at / TILE) * (256 * 128) + (uint32_t)row * 128 + (TERMS > 1 ? column * 16 : (column >> 2) * (256 * 128) + (column & 3) * 16);
    }
    // Inline assembly because the compiler would make every later LDS read wait for a load it knows to write LDS; the wait
    // is at the head of each stage.  No output registers.
    constexpr uint32_t kStep = depth_of(TILE, TERMS) / 32 * 256 * 128;  // bytes from a stage's corner to the next one's
    const uint32_t lds_first = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem) + (uint32_t)(wave * 1024);
    uint64_t next_u = 0, next_v = 0;  // corners of the stage that is requested next
    auto aim = [&]() {
        const int64_t column = (int64_t)ahead.stage * depth_of(TILE, TERMS);
        next_u = reinterpret_cast<uint64_t>(g.u + split_at((int64_t)ahead.ti * TILE, column, g.u_cols));
        next_v = reinterpret_cast<uint64_t>(g.v + split_at((int64_t)ahead.tj * TILE, column, g.v_cols));
    };
    auto issue_one = [&](uint64_t addr, uint32_t lds) {
        const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)addr),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(addr >> 32)) & 0xffffu, 0xffffffffu, 0x00020000u};
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(lds + (uint32_t)(j * kWaves) * 1024u), "v"(off[j]), "s"(rsrc)
                         : "memory", "m0");
    };
    int ahead_slot = 0;
    auto issue = [&]() {
        const uint32_t lds = lds_first + (uint32_t)ahead_slot * (2 * kOperand);
        issue_one(next_u, lds);
        issue_one(next_v, lds + kOperand);
        ahead_slot = (ahead_slot + 1) & kMask;
        ++requested;
        next_u += kStep;
        next_v += kStep;
        if (++ahead.stage == ahead.end) {
            more = ahead.next_unit(g, units);
            if (more) aim();
        }
    };
    aim();

    f32x16 acc[S::FM][S::FN];

    // Lane (half, i) reads k = 16 s + 8 half .. + 7 of row i: 16-byte column 2 s + half of its row, lo four columns further.
    constexpr int kSteps = TERMS > 1 ? 2 : 4;
    auto frag = [&](int base, int row, int quad) {
        return *reinterpret_cast<const f16x8 *>(smem + base + row * 128 + ((quad ^ swizzle(row)) << 4));
    };
    // KS == 1: a stage is kSteps x FM groups of matrix instructions, one block row of the wavefront at one s each; a group's
    // operands are read from LDS while the group before it computes, the first group's of a stage behind the barrier that
    // publishes it, which sits before the last group of the stage before.  (With all of a step's reads in front of its
    // instructions the wavefronts, in step after the barrier, took turns between LDS and matrix cores: 4400 cycles a stage
    // of 256 x 256 x 32 instead of the 3100 that they compute.)
    constexpr int kGroups = kSteps * S::FM;
    static_assert(S::KS > 1 || kGroups % 2 == 0, "the buffers alternate across stages");
    f16x8 uh[2], ul[2], vh[2][S::FN], vl[2][S::FN];
    auto read_group = [&](int slot, int group) {  // into buffer group % 2 (U) and s % 2 (V)
        const int bu = slot * 2 * kOperand, bv = bu + kOperand, s = group / S::FM, mi = group % S::FM;
        if (mi == 0) {
#pragma unroll
            for (int ni = 0; ni < S::FN; ++ni) {
                const int row = (wave_j * S::FN + ni) * 32 + l32;
                vh[s & 1][ni] = frag(bv, row, 2 * s + half);
                if (TERMS > 1) vl[s & 1][ni] = frag(bv, row, 4 + 2 * s + half);
            }
        }
        const int row = (wave_i * S::FM + mi) * 32 + l32;
        uh[group & 1] = frag(bu, row, 2 * s + half);
        if (TERMS == 3) ul[group & 1] = frag(bu, row, 4 + 2 * s + half);
    };
    auto multiply_group = [&](int group) {
        const int s = group / S::FM, mi = group % S::FM;
#pragma unroll
        for (int term = 3 - TERMS; term < 3; ++term)
#pragma unroll
            for (int ni = 0; ni < S::FN; ++ni)
                acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_f16(term == 0 ? ul[group & 1] : uh[group & 1],
                                                                     term == 1 ? vl[s & 1][ni] : vh[s & 1][ni], acc[mi][ni], 0, 0, 0);
    };
    // KS == 2: a wavefront's half of the stage's steps at once; the other wavefronts of its SIMD cover the reads.
    auto compute = [&](int slot, auto request) {
        // two lines: one for each half of the wavefronts; one line: half of its steps
        constexpr int kMySteps = kSteps * kLines / S::KS;
        const int bu = slot * 2 * kOperand + (kLines == 2 ? share * TILE * 128 : 0), bv = bu + kOperand;
#pragma unroll
        for (int q = 0; q < kMySteps; ++q) {
            const int column = 2 * ((kLines == 2 ? 0 : share * kMySteps) + q) + half;
            f16x8 ah[S::FM], al[S::FM], bh[S::FN], bl[S::FN];
#pragma unroll
            for (int ni = 0; ni < S::FN; ++ni) {
                const int row = (wave_j * S::FN + ni) * 32 + l32;
                bh[ni] = frag(bv, row, column);
                if (TERMS > 1) bl[ni] = frag(bv, row, 4 + column);
            }
#pragma unroll
            for (int mi = 0; mi < S::FM; ++mi) {
                const int row = (wave_i * S::FM + mi) * 32 + l32;
                ah[mi] = frag(bu, row, column);
                if (TERMS == 3) al[mi] = frag(bu, row, 4 + column);
            }
            if (q == 0) request();  // its address arithmetic runs while the operands are on their way
#pragma unroll
            for (int term = 3 - TERMS; term < 3; ++term)
#pragma unroll
                for (int mi = 0; mi < S::FM; ++mi)
#pragma unroll
                    for (int ni = 0; ni < S::FN; ++ni)
                        acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_f16(term == 0 ? al[mi] : ah[mi], term == 1 ? bl[ni] : bh[ni],
                                                                             acc[mi][ni], 0, 0, 0);
        }
    };

    // Stages are requested into every slot up front and then, stage by stage, into the slot that was read last.
#pragma unroll 1
    for (int d = 0; d < S::DEPTH - (S::KS > 1 ? 1 : 0) && more; ++d) issue();
    int slot = 0;
    bool counted = true;  // only stage loads are outstanding
    if (S::KS == 1) {
        if (requested == S::DEPTH) wait_for_all_but<(S::DEPTH - 1) * 2 * kLoads>();
        else wait_for_all_but<0>();
        __syncthreads();
        read_group(0, 0);
    }
    while (at.next_unit(g, units)) {
#pragma unroll
        for (int mi = 0; mi < S::FM; ++mi)
#pragma unroll
            for (int n = 0; n < S::FN; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[mi][n][r] = 0.0f;
        constexpr int kBlocks = S::FM * S::FN, kMine = (kBlocks + S::KS - 1) / S::KS;  // that a wavefront finishes
        const int from = share * kMine, until = from + kMine < kBlocks ? from + kMine : kBlocks;
        auto place_i = [&](int b) { return (int64_t)at.ti * TILE + (wave_i * S::FM + b / S::FN) * 32; };
        auto place_j = [&](int b) { return (int64_t)at.tj * TILE + (wave_j * S::FN + b % S::FN) * 32; };
        const bool finishes = at.slot < 0 && from < until;
        Old old, next;
        if (S::KS == 2 && finishes) load_old<FINISH>(g, g.old, place_i(from), place_j(from), old);  // on its way during the stages
        for (; at.stage < at.end; ++at.stage) {
            if constexpr (S::KS == 1) {
#pragma unroll
                for (int group = 0; group + 1 < kGroups; ++group) {
                    read_group(slot, group + 1);
                    multiply_group(group);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (requested > 1) {
                    wait_for_all_but<0>();  // the next stage has landed
                    __syncthreads();        // for every wavefront's loads; and everyone has read the last of this stage
                    slot = (slot + 1) & kMask;
                    read_group(slot, 0);
                    if (more) issue();  // into the slot of the stage before
                }
                --requested;
                multiply_group(kGroups - 1);
                __builtin_amdgcn_sched_barrier(0);
            } else {
                // this stage has landed when at most the DEPTH - 2 younger ones are outstanding
                if (S::DEPTH > 2 && counted && requested == S::DEPTH - 1) wait_for_all_but<(S::DEPTH - 2) * 2 * kLoads>();
                else wait_for_all_but<0>();
                counted = true;
                __syncthreads();  // for every wavefront's loads, and everyone is done with the slot that is filled next
                compute(slot, [&]() {
                    if (more) issue();
                });
                slot = (slot + 1) & kMask;
                --requested;
            }
        }
        counted = false;
        float *own = reinterpret_cast<float *>(smem + S::DEPTH * 2 * kOperand) + wave * 1024;
        if constexpr (S::KS == 2) {
            // the two halves meet: each wavefront of a pair takes half of their blocks (the first one a single block)
            const float *theirs = own + (share ? -1 : 1) * (S::WM * S::WN * 1024);
            auto exchange = [&](auto first, auto second) {  // block this wavefront gives, block it takes
                constexpr int give = decltype(first)::value, take = decltype(second)::value;
                if constexpr (give < kBlocks) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x16 &a = acc[give / S::FN][give % S::FN];
                        *reinterpret_cast<f32x4 *>(own + q * 256 + lane * 4) = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                    }
                }
                __syncthreads();
                if constexpr (take < kBlocks) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(theirs + q * 256 + lane * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[take / S::FN][take % S::FN][4 * q + e] += x[e];
                    }
                }
                __syncthreads();
            };
            if (share == 0) {
                exchange(Constant<kMine>{}, Constant<0>{});
                if constexpr (kMine > 1) exchange(Constant<kMine + 1>{}, Constant<1>{});
            } else {
                exchange(Constant<0>{}, Constant<kMine>{});
                if constexpr (kMine > 1) exchange(Constant<1>{}, Constant<kMine + 1>{});
            }
        }
        // a finished block, or its part of the sum as the registers lie: [32 x 32 block][number / 4][lane][4]
        const bool mirror = !(g.triangle && at.ti == at.tj);
        // One copy of the code for all blocks (unrolled it would be most of the kernel, fetched anew by every launch): the block's
        // registers are picked by a branch.  Old values are requested a block ahead, in front of the stores of the block before:
        // the counter that a load is waited for with would otherwise drain them first.
        if (S::KS == 1 && finishes) load_old<FINISH>(g, g.old, place_i(from), place_j(from), old);
#pragma unroll 1
        for (int b = from; b < until; ++b) {
            f32x16 sum;
            for_each<kBlocks>([&](auto step) {
                constexpr int k = decltype(step)::value;
                if (b == k) {
                    sum = acc[k / S::FN][k % S::FN];
                    asm volatile("" : "+v"(sum));  // a branch, not sixteen selects for every block
                }
            });
            if (at.slot < 0) {
                if (b + 1 < until) load_old<FINISH>(g, g.old, place_i(b + 1), place_j(b + 1), next);
                finish_block<FINISH>(g, factor, sum, old, place_i(b), place_j(b), mirror, own);
                old = next;
            } else {
                float *out = g.parts + (size_t)at.slot * TILE * TILE;
                const int block = (wave_i * S::FM + b / S::FN) * (TILE / 32) + wave_j * S::FN + b % S::FN;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4 *>(out + block * 1024 + q * 256 + lane * 4) =
                        f32x4{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]};
            }
        }
    }
}

// The tiles of groups with several parts: the parts are added in order.  A wavefront takes a 32 x 32 block.
template <int TILE, int FINISH>
__global__ __launch_bounds__(256) void join_kernel(Product g, int from) {
    __shared__ __attribute__((aligned(16))) float stage[4][1024];
    constexpr int kSide = TILE / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int tile = from + blockIdx.x / (kSide * kSide / 4), block = blockIdx.x % (kSide * kSide / 4) * 4 + wave;
    Group a = g.group[0];
#pragma unroll
    for (int i = 1; i < kMaxGroups; ++i)
        if (g.group[i].count > 0 && tile >= g.group[i].first) a = g.group[i];
    if (a.parts < 2) return;
    int ti, tj;
    tile_place(tile, g.tiles_j, g.triangle, ti, tj);
    const int64_t i0 = (int64_t)ti * TILE + block / kSide * 32, j0 = (int64_t)tj * TILE + block % kSide * 32;
    Old old;
    load_old<FINISH>(g, g.old, i0, j0, old);
    f32x16 sum;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.0f;
    constexpr int kBatch = 4;  // parts in flight: few tiles of a long k have dozens each
    for (int first = 0; first < a.parts; first += kBatch) {
        f32x4 x[kBatch][4];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (first + j >= a.parts) break;
            const float *p = g.parts + (size_t)(a.slot + (first + j) * a.count + tile - a.first) * TILE * TILE + block * 1024 + lane * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q) x[j][q] = *reinterpret_cast<const f32x4 *>(p + q * 256);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (first + j >= a.parts) break;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[4 * q + e] += x[j][q][e];
        }
    }
    finish_block<FINISH>(g, *g.factor, sum, old, i0, j0, !(g.triangle && ti == tj), stage[wave]);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// How a product is cut.
struct Cut {
    int tile, workgroups, tiles, tiles_j, stages;
    int groups, slots;
    Group group[kMaxGroups];
    int whole;  // tiles before the first group with parts
};
constexpr int kSlots = 256;  // workgroups at a time, one per compute unit
// At most `most_parts` parts to a tile; 1: whole tiles.
Cut cut_with(int64_t rows_i, int64_t rows_j, int64_t depth, bool triangle, int terms, int tile, int most_parts) {
    Cut c{};
    const int64_t ti = (rows_i + tile - 1) / tile, tj = (rows_j + tile - 1) / tile;
    c.tile = tile;
    c.tiles_j = (int)tj;
    c.tiles = (int)(triangle ? tj * (tj + 1) / 2 : ti * tj);
    c.stages = (int)((depth + depth_of(tile, terms) - 1) / depth_of(tile, terms));
    auto add = [&](int count, int parts, int rounds) {
        const int first = c.groups ? c.group[c.groups - 1].first + c.group[c.groups - 1].count * c.group[c.groups - 1].rounds : 0;
        c.group[c.groups++] = Group{first, count, parts, rounds, c.slots};
        if (parts > 1) c.slots += count * parts;
        if (count * parts > c.workgroups) c.workgroups = count * parts;
        if (c.slots == 0) c.whole += count * rounds;
    };
    int left = c.tiles;
    if (left >= kSlots) {
        add(kSlots, 1, left / kSlots);
        left %= kSlots;
    }
    if (most_parts == 1) {
        if (left) add(left, 1, 1);
        return c;
    }
    const int least = tile == 256 ? 8 : 4;  // a part has so many stages or more
    int most = c.stages / least < 1 ? 1 : c.stages / least;
    if (most > most_parts) most = most_parts;
    while (left > 0) {
        const bool final = c.groups + 1 == kMaxGroups;
        int parts = final ? kSlots / left : (kSlots + left - 1) / left;
        if (parts > most) parts = most;
        if (parts < 1) parts = 1;
        const int count = kSlots / parts < left ? kSlots / parts : left;
        add(count, parts, 1);
        left -= count;
    }
    return c;
}
// The time a cut is expected to take, in microseconds: what its workgroups do one after the other, and the join.  Measured on
// 784 x 1024, 1000 x 4001, 4096 x 4096 and 4096 x 16384: a stage's time by tile size and number of products, a tile's
// epilogue, storing a part; a launch takes 4 us more than what runs in it, the parts are written and read at about 8 TB/s together,
// and the parts of a tile take 0.25 us each one after the other (64 x 16384 in 64 parts: 185 us, in 16 127).
double cost_of(const Cut &c, int terms) {
    const int size = c.tile == 256 ? 0 : c.tile == 128 ? 1 : 2;
    static const double stage[3][3] = {{2.1, 2.07, 2.42}, {1.2, 1.28, 1.55}, {0.55, 0.52, 0.53}};  // [size][products - 1]
    static const double finish[3] = {13.0, 3.0, 1.5}, store[3] = {3.0, 2.0, 1.0};
    double t = 4.0;
    int busy = 0, parts = 0;
    for (const Group &g : c.group) {
        if (g.count == 0) continue;
        // a chip that is not full runs at a higher clock
        const double one = stage[size][terms - 1] * (size < 2 && g.count * g.parts < 200 ? 0.72 : 1.0);
        t += g.rounds * (c.stages / (double)g.parts * one + (g.parts > 1 ? store[size] : finish[size]));
        busy += g.parts > 1 ? g.count * g.parts : 0;
        if (g.parts > parts) parts = g.parts;
    }
    if (busy) t += 4.5 + 0.25 * parts + (double)busy * c.tile * c.tile * 8 / 8e6;
    return t;
}
Cut cut_product(int64_t rows_i, int64_t rows_j, int64_t depth, bool triangle, int terms) {
    Cut best{};
    double least = 0.0;
    for (int tile : {256, 128, 64})
        for (int most_parts : {1, 16, kSlots}) {
            const Cut c = cut_with(rows_i, rows_j, depth, triangle, terms, tile, most_parts);
            const double t = cost_of(c, terms);
            if (best.tile == 0 || t < least) {
                best = c;
                least = t;
            }
        }
    return best;
}

struct Space {
    f16_t *x, *xt[2], *a, *p;
    float *parts, *factors;
    double *norms;
    size_t bytes;
};
struct Sizes {
    int64_t m, n, mp, np;
    int flip;
    Cut gram[2], square, apply[2];  // [all parts of X, or of an exact X0 hi alone]
};
Sizes sizes_of(int64_t rows, int64_t cols) {
    Sizes z;
    z.flip = rows > cols;
    z.m = z.flip ? cols : rows;
    z.n = z.flip ? rows : cols;
    z.mp = padded(z.m);
    z.np = padded(z.n);
    z.square = cut_product(z.m, z.m, z.m, true, 3);
    for (int exact = 0; exact < 2; ++exact) {
        z.gram[exact] = cut_product(z.m, z.m, z.n, true, exact ? 1 : 3);
        z.apply[exact] = cut_product(z.n, z.m, z.m, false, exact ? 2 : 3);
    }
    return z;
}

Space lay_out(void *workspace, const Sizes &z) {
    Carver c(workspace);
    Space s{};
    s.x = c.take<f16_t>((size_t)z.mp * z.np * 2);
    s.xt[0] = c.take<f16_t>((size_t)z.mp * z.np * 2);
    s.xt[1] = c.take<f16_t>((size_t)z.mp * z.np * 2);
    s.a = c.take<f16_t>((size_t)z.mp * z.mp * 2);
    s.p = c.take<f16_t>((size_t)z.mp * z.mp * 2);
    size_t parts = 0;
    for (const Cut *cut : {&z.gram[0], &z.gram[1], &z.square, &z.apply[0], &z.apply[1]}) {
        const size_t need = (size_t)cut->slots * cut->tile * cut->tile;
        if (need > parts) parts = need;
    }
    s.parts = c.take<float>(parts);
    s.norms = c.take<double>(kNormBlocks);
    s.factors = c.take<float>(3);
    s.bytes = c.used;
    return s;
}

template <int TILE, int TERMS, int FINISH>
cn_status run_product(const Product &g, const Cut &c, int device, hipStream_t st) {
    static OncePerDevice configured;
    const cn_status status = configured.lds(device, lds_of<TILE>(), &product_kernel<TILE, TERMS, FINISH>);
    if (status != CN_OK) return status;
    hipLaunchKernelGGL((product_kernel<TILE, TERMS, FINISH>), dim3(c.workgroups), dim3(threads_of<TILE>()), lds_of<TILE>(), st, g);
    if (c.slots > 0)
        hipLaunchKernelGGL((join_kernel<TILE, FINISH>), dim3((c.tiles - c.whole) * (TILE / 32) * (TILE / 32) / 4), dim3(256), 0, st, g, c.whole);
    CN_HIP(hipGetLastError());
    return CN_OK;
}
template <int TERMS, int FINISH>
cn_status run_product(const Product &g, const Cut &c, int device, hipStream_t st) {
    return c.tile == 256 ? run_product<256, TERMS, FINISH>(g, c, device, st) : c.tile == 128 ? run_product<128, TERMS, FINISH>(g, c, device, st)
                                                                                             : run_product<64, TERMS, FINISH>(g, c, device, st);
}

struct Result {
    void *out;
    int dtype;
    int64_t ldo;
    int update;
    float keep, rate;
};

template <typename T>
cn_status newton_schulz(const Source &src, int steps, const Result &res, const Sizes &z, const Space &s, int device, hipStream_t st) {
    const int exact = sizeof(T) == 2 && !src.momentum;
    int norm_blocks = 0;
    auto begin = [&](auto vector) {
        constexpr int VEC = decltype(vector)::value;
        const int64_t tiles = ((src.cols + 256 * VEC - 1) / (256 * VEC)) * ((src.rows + kNormRows - 1) / kNormRows);
        norm_blocks = (int)(tiles < kNormBlocks ? tiles : kNormBlocks);
        hipLaunchKernelGGL((norm_kernel<T, VEC>), dim3(norm_blocks), dim3(256), 0, st, src, s.norms);
        hipLaunchKernelGGL((split_kernel<T, VEC>), dim3((unsigned)((z.mp / 64) * (z.np / 64))), dim3(256), 0, st, src, s.norms, norm_blocks,
                           z.flip, exact, z.mp, z.np, s.x, s.xt[0], s.factors);
    };
    const bool wide = src.cols % 4 == 0 && src.ldg % 4 == 0 && aligned_to(src.grad, 4 * sizeof(T)) &&
                      (!src.momentum || (src.ldm % 4 == 0 && aligned_to(src.momentum, 16)));
    if (wide) begin(Constant<4>{}); else begin(Constant<1>{});
    CN_HIP(hipGetLastError());
    Product base{};
    base.parts = s.parts;
    base.to_t_cols = z.mp;
    base.factor = s.factors;
    base.out = res.out; base.out_dtype = res.dtype; base.ldo = res.ldo; base.m = z.m; base.n = z.n; base.flip = z.flip;
    base.wide = res.ldo % 4 == 0 && aligned_to(res.out, 4 * dtype_bytes(res.dtype));
    base.update = res.update; base.keep = res.keep; base.rate = res.rate;
    auto with = [&](const Cut &c, const f16_t *u, const f16_t *v, int64_t depth) {
        Product g = base;
        g.u = u; g.v = v;
        g.u_cols = g.v_cols = depth;
        g.tiles_j = c.tiles_j;
        g.stages = c.stages;
        for (int i = 0; i < kMaxGroups; ++i) g.group[i] = c.group[i];
        return g;
    };
    int at = 0;  // which X^T is current
    for (int done = 0; done < steps; ++done) {
        const bool first = done == 0, last = done + 1 == steps, hi_alone = exact && first, two = hi_alone && !last;
        Product g = with(z.gram[hi_alone], s.x, s.x, z.np);
        g.triangle = 1;
        g.y = 1.0f / kUnit;
        g.factor = s.factors + (first ? 2 : 0);
        g.to = s.a;
        g.to_cols = z.mp;
        cn_status status = hi_alone ? run_product<1, GRAM>(g, z.gram[1], device, st) : run_product<3, GRAM>(g, z.gram[0], device, st);
        if (status != CN_OK) return status;
        g = with(z.square, s.a, s.a, z.mp);
        g.triangle = 1;
        g.old = s.a;
        g.x = kB * kPolyUnit / kUnit;
        g.y = kC * kPolyUnit / (kUnit * kUnit);
        g.to = s.p;
        g.to_cols = z.mp;
        status = run_product<3, POLY>(g, z.square, device, st);
        if (status != CN_OK) return status;
        const Cut &c = z.apply[two];
        g = with(c, s.xt[at], s.p, z.mp);
        g.old = s.x;
        g.x = kA;
        g.y = 1.0f / kPolyUnit;
        g.factor = s.factors + (first ? 1 : 0);
        g.to = s.x;
        g.to_cols = z.np;
        g.to_t = s.xt[at ^ 1];
        status = last ? run_product<3, LAST>(g, c, device, st) : two ? run_product<2, STEP>(g, c, device, st) : run_product<3, STEP>(g, c, device, st);
        if (status != CN_OK) return status;
        at ^= 1;
    }
    return CN_OK;
}

constexpr int64_t kMostSide = (int64_t)1 << 17;  // rows or columns: 32-bit tile offsets and grids

cn_status check_sizes(const char *what, int64_t rows, int64_t cols, int steps) {
    if (rows < 0 || cols < 0) { set_error("%s: negative dimension", what); return CN_ERR_SHAPE; }
    if (steps < 1 || steps > 100) { set_error("%s: %d steps (1 to 100)", what, steps); return CN_ERR_ARG; }
    if (rows > kMostSide || cols > kMostSide) { set_error("%s: more than %lld rows or columns", what, (long long)kMostSide); return CN_ERR_SHAPE; }
    return CN_OK;
}

cn_status start(const char *what, const Source &src, int grad_dtype, int steps, const Result &res, void *workspace,
                size_t workspace_bytes, void *stream) {
    const Sizes z = sizes_of(src.rows, src.cols);
    const Space s = lay_out(workspace, z);
    if (workspace_bytes < s.bytes) {
        set_error("%s: workspace of %zu bytes, %zu needed", what, workspace_bytes, s.bytes);
        return CN_ERR_WORKSPACE;
    }
    if (!aligned_to(workspace, 256)) { set_error("%s: the workspace is not aligned to 256 bytes", what); return CN_ERR_ARG; }
    if (src.momentum && (src.momentum == src.grad || src.momentum == res.out || src.grad == res.out)) {
        set_error("%s: momentum, gradient and weights are not three matrices", what);
        return CN_ERR_ARG;
    }
    Context *ctx;
    const cn_status status = current_context(&ctx);
    if (status != CN_OK) return status;
    hipStream_t st = (hipStream_t)stream;
    if (grad_dtype == CN_F32) return newton_schulz<float>(src, steps, res, z, s, ctx->device, st);
    if (grad_dtype == CN_F16) return newton_schulz<f16_t>(src, steps, res, z, s, ctx->device, st);
    return newton_schulz<bf16_t>(src, steps, res, z, s, ctx->device, st);
}

}  // namespace

}  // namespace cn

using namespace cn;

extern "C" {

size_t cn_orthogonalize_workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || rows > kMostSide || cols > kMostSide) return 0;
    return lay_out(nullptr, sizes_of(rows, cols)).bytes;
}

cn_status cn_orthogonalize(const void *G, int dtype, int64_t rows, int64_t cols, int64_t ldg, int steps, void *out, int out_dtype,
                           int64_t ldo, void *workspace, size_t workspace_bytes, void *stream) {
    if (!known_dtype(dtype) || !known_dtype(out_dtype)) { set_error("orthogonalize: unknown element type"); return CN_ERR_ARG; }
    const cn_status status = check_sizes("orthogonalize", rows, cols, steps);
    if (status != CN_OK) return status;
    if (ldg < cols || ldo < cols) { set_error("orthogonalize: leading dimension too small"); return CN_ERR_SHAPE; }
    if (rows == 0 || cols == 0) return CN_OK;
    if (!G || !out || !workspace) { set_error("orthogonalize: NULL pointer"); return CN_ERR_NULL; }
    Source src{};
    src.grad = G; src.ldg = ldg; src.rows = rows; src.cols = cols;
    const Result res{out, out_dtype, ldo, 0, 0.0f, 0.0f};
    return start("orthogonalize", src, dtype, steps, res, workspace, workspace_bytes, stream);
}

cn_status cn_muon_update(float *momentum, int64_t ldm, const void *grad, int grad_dtype, int64_t ldg, float *w, int64_t ldw,
                         int64_t rows, int64_t cols, float momentum_factor, int nesterov, float learning_rate, float weight_decay,
                         int steps, void *workspace, size_t workspace_bytes, void *stream) {
    if (!known_dtype(grad_dtype)) { set_error("muon_update: unknown element type %d", grad_dtype); return CN_ERR_ARG; }
    const cn_status status = check_sizes("muon_update", rows, cols, steps);
    if (status != CN_OK) return status;
    if (ldm < cols || ldg < cols || ldw < cols) { set_error("muon_update: leading dimension too small"); return CN_ERR_SHAPE; }
    if (rows == 0 || cols == 0) return CN_OK;
    if (!momentum || !grad || !w || !workspace) { set_error("muon_update: NULL pointer"); return CN_ERR_NULL; }
    Source src{};
    src.grad = grad; src.ldg = ldg; src.momentum = momentum; src.ldm = ldm;
    src.mu = momentum_factor; src.nesterov = nesterov != 0;
    src.rows = rows; src.cols = cols;
    const Result res{w, CN_F32, ldw, 1, 1.0f - learning_rate * weight_decay, learning_rate};
    return start("muon_update", src, grad_dtype, steps, res, workspace, workspace_bytes, stream);
}

}  // extern "C"
