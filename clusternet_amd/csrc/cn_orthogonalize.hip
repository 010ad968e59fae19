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
// numbers, x 2^14 = hi + lo, and a product is the three fp16 products hi hi + hi lo + lo hi in fp32 accumulators, which
// runs at up to a third of the fp16 rate (2.5 PFLOP/s).  What is left out, lo lo, and the rounding of lo are 2^-22 of the
// product, so the result is as far from the exact one as plain fp32 products leave it (measured on the CPU for
// Gaussian, power-law and nearly rank-8 spectra: within 5 % of fp32's error in every case).  The factor 2^14 keeps
// entries of all four matrices below 65504 (|X| <= 1.21, |A| <= 1.46, |P| <= 2.81) and lo above the smallest
// fp16 number for entries down to 2^-13 of the largest.  a X stays outside the product, with X read back as hi + lo:
// folding a into P's diagonal costs a factor of three in accuracy for nearly low-rank gradients.
//
// Layout: a matrix is rows of 128-byte groups, 32 columns each: 32 hi, then 32 lo.  A stage of the product (32 of k) is then
// one 128-byte line per row, and the tile in LDS is the fp32 kernel's [row][32 words] with its swizzle (cn_gemm.hip).  All
// sizes are padded to whole tiles with zeros, so nothing in the product needs a bounds check.  X is kept in both
// orientations (the Gram product sums over n, the update over m), P and A are symmetric.
//
// Work split: the tiles' stages, laid end to end, are dealt to W workgroups in equal contiguous runs, so the 136 tiles above the
// diagonal of a 4096 x 4096 result load all compute units evenly.  A run that begins or ends inside a tile leaves a part of
// that tile's sum; a second kernel adds a tile's parts in order, applies the formula and writes the next operand (both
// orientations), so the result does not depend on scheduling.
#include "cn_dtypes.h"

namespace cn {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kUnit = 16384.0f;                   // the stored number for 1
constexpr float kProduct = 1.0f / (kUnit * kUnit);  // of an accumulator
constexpr int kPad = 256;                           // rows and columns are padded to whole tiles
constexpr int kStage = 32;                          // of k

int64_t padded(int64_t n) { return (n + kPad - 1) / kPad * kPad; }

// ---- split numbers -----------------------------------------------------------------------------------------------------
// Element (row, col) of a split matrix of `cols` columns: hi at row * 2 cols + (col / 32) * 64 + col % 32, lo 32 further.
__device__ __forceinline__ size_t split_at(int64_t row, int64_t col, int64_t cols) {
    return (size_t)row * 2 * cols + (size_t)(col >> 5) * 64 + (col & 31);
}
// Four consecutive columns (col a multiple of 4), in stored units.
__device__ __forceinline__ void split_store(f16_t *m, size_t at, const float (&v)[4]) {
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = (f16_t)v[e];
        lo[e] = (f16_t)(v[e] - (float)hi[e]);
    }
    *reinterpret_cast<f16x4 *>(m + at) = hi;
    *reinterpret_cast<f16x4 *>(m + at + 32) = lo;
}
__device__ __forceinline__ void split_load(const f16_t *m, size_t at, float (&v)[4]) {
    const f16x4 hi = *reinterpret_cast<const f16x4 *>(m + at), lo = *reinterpret_cast<const f16x4 *>(m + at + 32);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)hi[e] + (float)lo[e];
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

// One element of the update.  `advance`: the momentum is moved on (once per step), else read as it is.
template <typename T>
__device__ __forceinline__ float update_of(const Source &s, int64_t r, int64_t c, bool advance) {
    const float g = (float)((const T *)s.grad)[r * s.ldg + c];
    if (!s.momentum) return g;
    float *at = s.momentum + r * s.ldm + c;
    float m = *at;
    if (advance) {
        m = s.mu * m + g;
        *at = m;
    }
    return s.nesterov ? g + s.mu * m : m;
}

constexpr int kNormBlocks = 1024;

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
template <typename T>
__global__ __launch_bounds__(256) void norm_kernel(Source s, double *parts) {
    __shared__ double scratch[4];
    double sum = 0.0;
    const int64_t tiles_c = (s.cols + 255) / 256;
    for (int64_t t = blockIdx.x; t < tiles_c * ((s.rows + 15) / 16); t += gridDim.x) {
        const int64_t r0 = t / tiles_c * 16, c = (t % tiles_c) * 256 + threadIdx.x;
        if (c >= s.cols) continue;
#pragma unroll 8
        for (int i = 0; i < 16; ++i)
            if (r0 + i < s.rows) {
                const double u = (double)update_of<T>(s, r0 + i, c, true);
                sum += u * u;
            }
    }
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// X0 in both orientations, zeros in the padding.  A workgroup takes 64 x 64 elements of X (m x n).
template <typename T>
__global__ __launch_bounds__(256) void split_kernel(Source s, const double *parts, int part_count, int flip, int64_t mp, int64_t np,
                                                    f16_t *x, f16_t *xt) {
    __shared__ double scratch[4];
    __shared__ float tile[64][65];
    double sum = 0.0;
    for (int i = threadIdx.x; i < part_count; i += 256) sum += parts[i];
    sum = block_sum(sum, scratch);
    const double to_unit = (double)kUnit / (sqrt(sum) + 1e-7);
    const int64_t blocks_n = np / 64;
    const int64_t i0 = blockIdx.x / blocks_n * 64, j0 = blockIdx.x % blocks_n * 64;  // of X
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 8
    for (int q = 0; q < 16; ++q) {
        const int a = wave + 4 * q;
        // read along the rows of G, whichever way it lies
        const int64_t r = (flip ? j0 : i0) + a, c = (flip ? i0 : j0) + lane;
        const float v = r < s.rows && c < s.cols ? (float)((double)update_of<T>(s, r, c, false) * to_unit) : 0.0f;
        if (flip) tile[lane][a] = v; else tile[a][lane] = v;
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
// D[i][j] = sum over k of U[i][k] V[j][k], both operands split.  `parts` receives TILE x TILE fp32 numbers per (tile, workgroup)
// pair, at slot tile + workgroup: along a run either the tile or the workgroup moves on, so every part has a slot of its own.
struct Product {
    const f16_t *u, *v;
    int64_t u_cols, v_cols;  // columns of the split matrices (padded)
    int tiles_j;             // tiles along j
    int tiles;               // all tiles; symmetric: those with j >= i
    int symmetric;
    int stages;              // of k
    float *parts;
};

template <int TILE> struct Shape;
template <> struct Shape<256> { static constexpr int WM = 2, WN = 4, FM = 4, FN = 2; };  // wavefronts, 32 x 32 blocks of each
template <> struct Shape<128> { static constexpr int WM = 2, WN = 2, FM = 2, FN = 2; };
template <int TILE> constexpr int threads_of() { return Shape<TILE>::WM * Shape<TILE>::WN * 64; }

__device__ __forceinline__ int swizzle(int row) { return (row & 7) ^ ((row >> 3) & 3); }

// Tile number to its row and column of tiles; symmetric: row by row, each from the diagonal on.
__device__ __forceinline__ void tile_place(int tile, int tiles_j, int symmetric, int &ti, int &tj) {
    if (!symmetric) {
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

template <int TILE>
__global__ __launch_bounds__(threads_of<TILE>(), 2) void product_kernel(Product g) {
    using S = Shape<TILE>;
    constexpr int kWaves = S::WM * S::WN, kLoads = TILE / 8 / kWaves;  // 1 KiB loads per operand, stage and wavefront
    extern __shared__ __attribute__((aligned(16))) char smem[];         // [2 stages][U, V][TILE rows][128 bytes]
    constexpr int kOperand = TILE * 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int half = lane >> 5, l32 = lane & 31;
    const int wave_i = wave / S::WN, wave_j = wave % S::WN;

    // Workgroups of one XCD (ids congruent mod 8) take neighbouring runs and share operands in its L2.
    const unsigned W = gridDim.x, xcd = blockIdx.x % 8u, idx = blockIdx.x / 8u, per = W / 8u, rem = W % 8u;
    const int w = (int)(xcd * per + (xcd < rem ? xcd : rem) + idx);
    const int64_t total = (int64_t)g.tiles * g.stages;
    const int64_t u0 = total * w / (int)W, u1 = total * (w + 1) / (int)W;
    if (u0 >= u1) return;
    int tile = __builtin_amdgcn_readfirstlane((int)(u0 / g.stages));
    int stage = __builtin_amdgcn_readfirstlane((int)(u0 % g.stages));
    int left = __builtin_amdgcn_readfirstlane((int)(u1 - u0));
    int ti, tj;
    tile_place(tile, g.tiles_j, g.symmetric, ti, tj);

    uint32_t off_u[kLoads], off_v[kLoads];  // this lane's 16 bytes of each 1 KiB (8 rows), from the tile's corner
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int row = (j * kWaves + wave) * 8 + (lane >> 3);
        const uint32_t quad = (uint32_t)(((lane & 7) ^ swizzle(row)) * 16);
        off_u[j] = (uint32_t)row * (uint32_t)(g.u_cols * 4) + quad;
        off_v[j] = (uint32_t)row * (uint32_t)(g.v_cols * 4) + quad;
    }
    // Inline assembly because the compiler would make every later LDS read wait for a load it knows to write LDS; the wait
    // is at the end of each stage.  No output registers.
    auto issue_one = [&](const f16_t *corner, const uint32_t (&off)[kLoads], int lds) {
        const uint64_t addr = reinterpret_cast<uint64_t>(corner);
        const u32x4 rsrc = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)addr),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(addr >> 32)) & 0xffffu, 0xffffffffu, 0x00020000u};
        const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem) +
                              (uint32_t)(lds + wave * 1024);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"(lds0 + (uint32_t)(j * kWaves) * 1024u), "v"(off[j]), "s"(rsrc)
                         : "memory", "m0");
    };
    auto issue = [&](int ti_, int tj_, int stage_, int slot) {
        issue_one(g.u + (int64_t)ti_ * TILE * 2 * g.u_cols + (int64_t)stage_ * 64, off_u, slot * 2 * kOperand);
        issue_one(g.v + (int64_t)tj_ * TILE * 2 * g.v_cols + (int64_t)stage_ * 64, off_v, slot * 2 * kOperand + kOperand);
    };

    f32x16 acc[S::FM][S::FN];

    // Lane (half, i) reads k = 16 s + 8 half .. + 7 of row i: 16-byte column 2 s + half of its row, lo four columns further.
    auto frag = [&](int base, int row, int quad) {
        return *reinterpret_cast<const f16x8 *>(smem + base + row * 128 + ((quad ^ swizzle(row)) << 4));
    };
    auto compute = [&](int slot) {
        const int bu = slot * 2 * kOperand, bv = bu + kOperand;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f16x8 uh[S::FM], ul[S::FM], vh[S::FN], vl[S::FN];
#pragma unroll
            for (int ni = 0; ni < S::FN; ++ni) {
                const int row = (wave_j * S::FN + ni) * 32 + l32;
                vh[ni] = frag(bv, row, 2 * s + half);
                vl[ni] = frag(bv, row, 4 + 2 * s + half);
            }
#pragma unroll
            for (int mi = 0; mi < S::FM; ++mi) {
                const int row = (wave_i * S::FM + mi) * 32 + l32;
                uh[mi] = frag(bu, row, 2 * s + half);
                ul[mi] = frag(bu, row, 4 + 2 * s + half);
            }
#pragma unroll
            for (int term = 0; term < 3; ++term)
#pragma unroll
                for (int mi = 0; mi < S::FM; ++mi)
#pragma unroll
                    for (int ni = 0; ni < S::FN; ++ni)
                        acc[mi][ni] = __builtin_amdgcn_mfma_f32_32x32x16_f16(term == 0 ? ul[mi] : uh[mi], term == 1 ? vl[ni] : vh[ni],
                                                                             acc[mi][ni], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    issue(ti, tj, stage, 0);
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the stage is in LDS
    __syncthreads();
    int slot = 0;
    while (left > 0) {  // a tile, or as much of it as the run holds
        const int here = left < g.stages - stage ? left : g.stages - stage;
        left -= here;
        int ni = ti, nj = tj + 1;
        if (nj == g.tiles_j) {
            ++ni;
            nj = g.symmetric ? ni : 0;
        }
#pragma unroll
        for (int mi = 0; mi < S::FM; ++mi)
#pragma unroll
            for (int n = 0; n < S::FN; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[mi][n][r] = 0.0f;
        for (int i = 1; i <= here; ++i) {  // the loads of the next stage, of this tile or the next, run under this one's products
            if (i < here) issue(ti, tj, stage + i, slot ^ 1);
            else if (left > 0) issue(ni, nj, 0, slot ^ 1);
            compute(slot);
            __builtin_amdgcn_s_waitcnt(0x0f70);
            __syncthreads();
            slot ^= 1;
        }
        float *out = g.parts + (size_t)(tile + w) * TILE * TILE + (wave_i * S::FM * 32 + 4 * half) * TILE + wave_j * S::FN * 32 + l32;
#pragma unroll
        for (int mi = 0; mi < S::FM; ++mi)
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int n = 0; n < S::FN; ++n) out[(mi * 32 + 8 * (r >> 2) + (r & 3)) * TILE + n * 32] = acc[mi][n][r];
        stage = 0;
        ++tile;
        ti = ni;
        tj = nj;
    }
}

// ---- what becomes of a product --------------------------------------------------------------------------------------------
enum Finish {
    GRAM = 0,  // A
    POLY = 1,  // P = b A + c A A
    STEP = 2,  // X <- a X + P X, both orientations
    LAST = 3   // the same, into the result
};
struct FinishArgs {
    const float *parts;
    int tile, tiles_j, symmetric, stages, workgroups;
    int64_t total;           // tiles * stages
    const f16_t *old;        // POLY: A;  STEP, LAST: X^T
    int64_t cols;            // columns of D's split form: mp
    f16_t *to, *to_t;        // D's split form and its transpose's (GRAM, POLY: the same matrix, mirrored)
    int64_t cols_t;
    // LAST
    void *out;               // the result, rows x cols as the caller has it (fp32 or 16 bits), or the weights (fp32)
    int64_t ldo, m, n;       // D is n x m
    int flip;                // the caller's matrix is n x m
    int update;              // out = keep * out - rate * X
    float keep, rate;
};

template <int MODE, typename E>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs g) {
    __shared__ float mirror[64][65];
    const int per_side = g.tile / 64;
    const int tile = blockIdx.x / (per_side * per_side), block = blockIdx.x % (per_side * per_side);
    int ti, tj;
    tile_place(tile, g.tiles_j, g.symmetric, ti, tj);
    const int bi = block / per_side * 64, bj = block % per_side * 64;
    const int64_t i0 = (int64_t)ti * g.tile + bi, j0 = (int64_t)tj * g.tile + bj;
    // the workgroups whose runs touch this tile: w holds units total * w / W .. total * (w + 1) / W - 1
    const int64_t first = (int64_t)tile * g.stages, last = first + g.stages - 1;
    const int w0 = (int)(((first + 1) * g.workgroups - 1) / g.total), w1 = (int)(((last + 1) * g.workgroups - 1) / g.total);
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * 4;
    float v[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q][e] = 0.0f;
    for (int w = w0; w <= w1; ++w) {
        const float *p = g.parts + (size_t)(tile + w) * g.tile * g.tile + (size_t)(bi + row) * g.tile + bj + col;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p + (size_t)(16 * q) * g.tile);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] += x[e];
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int i = row + 16 * q;
        const size_t at = split_at(i0 + i, j0 + col, g.cols);
        if (MODE == GRAM) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] *= kProduct * kUnit;
        } else {
            float old[4];
            split_load(g.old, at, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (MODE == POLY) v[q][e] = kB * old[e] + (kC * kProduct * kUnit) * v[q][e];
                else v[q][e] = kA * old[e] + (kProduct * kUnit) * v[q][e];
            }
        }
        if (MODE != LAST) split_store(g.to, at, v[q]);
#pragma unroll
        for (int e = 0; e < 4; ++e) mirror[i][col + e] = v[q][e];
    }
    if (MODE == LAST) {
        __syncthreads();
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 4
        for (int q = 0; q < 16; ++q) {
            const int a = wave + 4 * q;
            // D[i][j] = X[j][i]; written along the rows of the caller's matrix
            const int64_t r = (g.flip ? i0 : j0) + a, c = (g.flip ? j0 : i0) + lane;
            if (r >= (g.flip ? g.n : g.m) || c >= (g.flip ? g.m : g.n)) continue;
            const float x = (g.flip ? mirror[a][lane] : mirror[lane][a]) * (1.0f / kUnit);
            E *out = (E *)g.out + r * g.ldo + c;
            *out = (E)(g.update ? g.keep * (float)*out - g.rate * x : x);
        }
        return;
    }
    if (g.symmetric && ti == tj) return;  // a tile on the diagonal holds both halves
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int j = row + 16 * q;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mirror[col + e][j];
        split_store(g.to_t, split_at(j0 + j, i0 + col, g.cols_t), x);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// Tiles of 256 x 256 feed every matrix instruction from fewer LDS and L2 bytes; tiles of 128 x 128 spread small products
// over more compute units.
int tile_for(int64_t mp, int64_t np) { return mp * np >= (int64_t)2048 * 2048 ? 256 : 128; }
int workgroups_for(int tile, int64_t total) {
    const int most = tile == 256 ? 256 : 512;
    const int64_t w = total / 4;  // at least four stages each
    return (int)(w < 1 ? 1 : w > most ? most : w);
}

struct Space {
    f16_t *x, *xt, *a, *p;
    float *parts;
    double *norms;
    size_t bytes;
};
struct Sizes {
    int64_t m, n, mp, np;
    int flip, tile;
};
Sizes sizes_of(int64_t rows, int64_t cols) {
    Sizes z;
    z.flip = rows > cols;
    z.m = z.flip ? cols : rows;
    z.n = z.flip ? rows : cols;
    z.mp = padded(z.m);
    z.np = padded(z.n);
    z.tile = tile_for(z.mp, z.np);
    return z;
}
int64_t tiles_along(int64_t n, int tile) { return (n + tile - 1) / tile; }

Space lay_out(void *workspace, const Sizes &z) {
    Carver c(workspace);
    Space s;
    s.x = c.take<f16_t>((size_t)z.mp * z.np * 2);
    s.xt = c.take<f16_t>((size_t)z.mp * z.np * 2);
    s.a = c.take<f16_t>((size_t)z.mp * z.mp * 2);
    s.p = c.take<f16_t>((size_t)z.mp * z.mp * 2);
    const int64_t tm = tiles_along(z.m, z.tile), tn = tiles_along(z.n, z.tile);
    const int64_t sm = (z.m + kStage - 1) / kStage, sn = (z.n + kStage - 1) / kStage;
    const int64_t gram = tm * (tm + 1) / 2, apply = tm * tn;
    int64_t slots = gram + workgroups_for(z.tile, gram * sn);
    if (gram + workgroups_for(z.tile, gram * sm) > slots) slots = gram + workgroups_for(z.tile, gram * sm);
    if (apply + workgroups_for(z.tile, apply * sm) > slots) slots = apply + workgroups_for(z.tile, apply * sm);
    s.parts = c.take<float>((size_t)slots * z.tile * z.tile);
    s.norms = c.take<double>(kNormBlocks);
    s.bytes = c.used;
    return s;
}

cn_status product(const Product &g, int tile, int workgroups, int device, hipStream_t st) {
    static OncePerDevice configured;
    if (configured.first(device)) {
        CN_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&product_kernel<256>), hipFuncAttributeMaxDynamicSharedMemorySize, 4 * 256 * 128));
        CN_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&product_kernel<128>), hipFuncAttributeMaxDynamicSharedMemorySize, 4 * 128 * 128));
    }
    if (tile == 256)
        hipLaunchKernelGGL((product_kernel<256>), dim3(workgroups), dim3(threads_of<256>()), 4 * 256 * 128, st, g);
    else
        hipLaunchKernelGGL((product_kernel<128>), dim3(workgroups), dim3(threads_of<128>()), 4 * 128 * 128, st, g);
    CN_HIP(hipGetLastError());
    return CN_OK;
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
    const int64_t norm_tiles = ((src.cols + 255) / 256) * ((src.rows + 15) / 16);
    const int norm_blocks = (int)(norm_tiles < kNormBlocks ? norm_tiles : kNormBlocks);
    hipLaunchKernelGGL((norm_kernel<T>), dim3(norm_blocks), dim3(256), 0, st, src, s.norms);
    hipLaunchKernelGGL((split_kernel<T>), dim3((unsigned)((z.mp / 64) * (z.np / 64))), dim3(256), 0, st, src, s.norms, norm_blocks, z.flip,
                       z.mp, z.np, s.x, s.xt);
    CN_HIP(hipGetLastError());
    const int tm = (int)tiles_along(z.m, z.tile), tn = (int)tiles_along(z.n, z.tile);
    const int sm = (int)((z.m + kStage - 1) / kStage), sn = (int)((z.n + kStage - 1) / kStage);
    const int gram_tiles = tm * (tm + 1) / 2, side = z.tile / 64;
    for (int step = 0; step < steps; ++step) {
        for (int which = 0; which < 3; ++which) {  // A = X X^T, A A, X^T P
            Product g{};
            g.u = which == 0 ? s.x : which == 1 ? s.a : s.xt;
            g.v = which == 0 ? s.x : which == 1 ? s.a : s.p;
            g.u_cols = which == 0 ? z.np : z.mp;
            g.v_cols = g.u_cols;
            g.tiles_j = tm;
            g.symmetric = which != 2;
            g.tiles = which == 2 ? tn * tm : gram_tiles;
            g.stages = which == 0 ? sn : sm;
            g.parts = s.parts;
            const int64_t total = (int64_t)g.tiles * g.stages;
            const int W = workgroups_for(z.tile, total);
            cn_status status = product(g, z.tile, W, device, st);
            if (status != CN_OK) return status;
            FinishArgs f{};
            f.parts = s.parts;
            f.tile = z.tile; f.tiles_j = tm; f.symmetric = g.symmetric; f.stages = g.stages; f.workgroups = W;
            f.total = total;
            f.old = which == 1 ? s.a : s.xt;
            f.cols = z.mp;
            f.to = which == 0 ? s.a : which == 1 ? s.p : s.xt;
            f.to_t = which == 0 ? s.a : which == 1 ? s.p : s.x;
            f.cols_t = which == 2 ? z.np : z.mp;
            f.out = res.out; f.ldo = res.ldo; f.m = z.m; f.n = z.n; f.flip = z.flip;
            f.update = res.update; f.keep = res.keep; f.rate = res.rate;
            const dim3 grid((unsigned)(g.tiles * side * side));
            if (which == 0)             hipLaunchKernelGGL((finish_kernel<GRAM, float>), grid, dim3(256), 0, st, f);
            else if (which == 1)        hipLaunchKernelGGL((finish_kernel<POLY, float>), grid, dim3(256), 0, st, f);
            else if (step + 1 < steps)  hipLaunchKernelGGL((finish_kernel<STEP, float>), grid, dim3(256), 0, st, f);
            else if (res.dtype == CN_F32) hipLaunchKernelGGL((finish_kernel<LAST, float>), grid, dim3(256), 0, st, f);
            else if (res.dtype == CN_F16) hipLaunchKernelGGL((finish_kernel<LAST, f16_t>), grid, dim3(256), 0, st, f);
            else                        hipLaunchKernelGGL((finish_kernel<LAST, bf16_t>), grid, dim3(256), 0, st, f);
            CN_HIP(hipGetLastError());
        }
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
