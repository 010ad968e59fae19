// Weights in 4 bits with a scale per group of rows, gfx950: quantisation, its inverse, and the product of a few rows with such
// weights.  The sibling of the 8-bit codes (cn_codec.hip, cn_gemm_w8_rows.hip) for answers: a token's product reads every
// weight once, so half the bytes are half the time.
//
// W (K x N) = (q - z) s, q in 0 .. 15, one s (fp32) and one z (8, or stored) per group of 32, 64 or 128 rows of a column.
// Stored form: int32 words [N / 16][K / 128][64][4]; nibble i of word t of lane l = 16 h + c holds row 128 b + 32 t + 8 h + i
// of column 16 a + c.  Word t of the 64 lanes is then the B operand of one 16 x 16 x 32 matrix instruction (lane l supplies
// k = 8 h .. 8 h + 7 of column c), and a wavefront reads 1 KiB in a row for 128 rows of 16 columns.  Rows and columns are
// padded with code 0 to whole tiles.
//
// Product: out[M x N] = A W, bound by the codes' way from memory for up to a few dozen rows.
//   * 16-bit rows: codes become numbers without arithmetic.  Bits 3 .. 6 of the bf16 pattern of 16.0 (bits 6 .. 9 of the fp16 one)
//     set to q give exactly 16 + q, a shift and an and-or for two weights.  The 16 and the zero point leave again behind the sum:
//         sum a (q - z) = sum a (16 + q) - (16 + z) sum a,
//     where sum a comes from one more matrix instruction against ones, in the same fp32 accumulators and the same order.  For rows
//     with a mean the difference is far smaller than its two sums, and their roundings with it (5 10^-6 of the largest result
//     for maxout outputs, 1 x 4096): little beside a 16-bit result's rounding (21 of 16384 bf16 results are not the exact ones rounded,
//     8 in plain fp32), too much for fp32.
//   * So fp32 rows take q - z, exact in bf16 and 15 operations more for eight weights, which cost what the product with ones did
//     (13 x 5000 x 1999 13.4 us, with 16 + q 13.1; 64 x 8192 x 16384 91 and 86, 40 x 8192 x 8192 in groups of 32 67 and 72).
//     The errors are 0.16 to 0.31 of those of a plain fp32 product of the decoded weights (root mean square, rows of mean zero,
//     maxout and sigmoid outputs, rows near 1), where they were up to 35 times those.
//   * Where a may be as large as fp32 goes, the operands are 2^-13 (16 + q), 2^-13 in place of 1, and 2^-11 (q - z) (another
//     exponent in the same pattern): 128 of the largest fit fp32, where same-signed rows from 8 10^34 on would overflow.
//     The factor comes back in the write-out: all sums keep 2^-136, less than half a step of the smallest normal bf16
//     number.  (Given to the scales, which then need a place for those above 2^115: 5 % for groups of 32.)
//   * Products are exact: a 16-bit a times a whole number up to 31 fits fp32; a of fp32 enters as three bf16 numbers that add
//     up to it exactly (8 bits of it each).  The sums, the scales and everything behind them are fp32; a 16-bit result is
//     rounded once.
//   * Up to 16 rows cost one instruction per 32 k and 16 columns, more rows further ones on the same decoded weights.
//   * A workgroup's wavefronts share its columns and split K; their sums meet in LDS and are added in order, so the result
//     does not depend on scheduling.
#include "cn_dtypes.h"

namespace cn {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTileN = 16, kTileK = 128;
template <int N> struct Constant { static constexpr int value = N; };

int64_t tiles_n_of(int64_t N) { return (N + kTileN - 1) / kTileN; }
int64_t tiles_k_of(int64_t K) { return (K + kTileK - 1) / kTileK; }

// ---- product -----------------------------------------------------------------------------------------------------------
struct GemmW4Args {
    const void *a;
    const u32x4 *codes;
    const float *scales;   // [groups][N]
    const uint8_t *zeros;  // [groups][N] or NULL: 8 everywhere
    void *out;
    int64_t M, N, K, lda, ldo;
    int tiles_k, tiles_n;
    int vec_a;             // rows of A allow 16-byte loads; others go element by element, with nothing requested ahead (1 x 5000 x 16384
                           // bf16 12.7 us, 4999 24.0; 13 x 5000 x 1999 fp32 12.0, 5001 27.5; 64 x 8192 x 16384 bf16 51, 8191 154)
};

// A operand of one instruction as the words of its kind, and how many of them a number needs.
template <typename T> struct Kind;
template <> struct Kind<bf16_t> {
    static constexpr int kParts = 1;
    static constexpr uint32_t kMagic = 0x3b003b00u, kMask = 0x00780078u, kOnes = 0x39003900u;  // 2^-9 = 16 / kUnit, 1 / kUnit
    static constexpr float kUnit = 8192.0f;
    static constexpr int kShift = 3;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Kind<float> : Kind<bf16_t> {
    static constexpr int kParts = 3;
    static constexpr float kUnit = 2048.0f;
};
template <typename T> constexpr bool kCentred = sizeof(T) == 4;  // operands are q - z instead of 16 + q
template <> struct Kind<f16_t> {
    static constexpr int kParts = 1;
    static constexpr uint32_t kMagic = 0x4c004c00u, kMask = 0x03c003c0u, kOnes = 0x3c003c00u;
    static constexpr float kUnit = 1.0f;  // 128 * 31 of the largest fp16 number fit fp32
    static constexpr int kShift = 6;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Operand words from eight codes: word j takes nibbles j and j + 4, which lie 16 bits apart: one shift and one and-or for two
// weights.  So word j of the A operand has to hold the numbers j and j + 4 of the lane's eight as well; the sum over k does
// not mind.  (In the order 2 j, 2 j + 1 a word takes five operations.)
template <typename T>
__device__ __forceinline__ u32x4 expand(uint32_t w) {
    using Q = Kind<T>;
    u32x4 b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int down = 4 * j - Q::kShift;  // nibble j from bit 4 j to bit kShift
        b[j] = ((down >= 0 ? w >> down : w << -down) & Q::kMask) | Q::kMagic;
    }
    return b;
}

// The same of fp32 rows: (q - z) / kUnit, exact in bf16; zero: z / kUnit of the lane's column.  23 operations in place of 8.
template <typename T>
__device__ __forceinline__ u32x4 expand_centred(uint32_t w, float zero) {
    const uint32_t nibbles[2] = {w & 0x0f0f0f0fu, w >> 4 & 0x0f0f0f0fu};  // byte m: nibble 2 m, 2 m + 1
    auto weight = [&](int i) { return __builtin_fmaf((float)(nibbles[i & 1] >> (8 * (i >> 1)) & 255u), 1.0f / Kind<T>::kUnit, -zero); };
    u32x4 b;
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __builtin_amdgcn_perm(__float_as_uint(weight(j + 4)), __float_as_uint(weight(j)), 0x07060302u);
    return b;
}

// Eight consecutive elements of A as operand words.
template <typename T>
__device__ __forceinline__ void operand(const u32x4 (&raw)[sizeof(T) / 2], u32x4 (&part)[Kind<T>::kParts]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j)  // halves j of the eight and j + 4
            part[0][j] = __builtin_amdgcn_perm(raw[0][2 + (j >> 1)], raw[0][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t piece[3][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t x = raw[e][j];
                const uint32_t h = x & 0xffff0000u;  // the first eight bits
                const float r = __uint_as_float(x) - __uint_as_float(h);
                const uint32_t m = __float_as_uint(r) & 0xffff0000u;
                const float l = r - __uint_as_float(m);  // at most eight bits are left
                piece[0][e] = h;
                piece[1][e] = m;
                piece[2][e] = __float_as_uint(l);
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][j] = __builtin_amdgcn_perm(piece[p][1], piece[p][0], 0x07060302u);
        }
    }
}

// Eight k of a row, from k on, as stored words; element by element: zeros past K.
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_eight(const T *row, int64_t k, int64_t K, bool vec, u32x4 (&raw)[sizeof(T) / 2]) {
    constexpr int kRaw = sizeof(T) / 2;
    if (WHOLE || (vec && k + 8 <= K)) {
#pragma unroll
        for (int r = 0; r < kRaw; ++r) raw[r] = *(reinterpret_cast<const u32x4 *>(row + k) + r);
        return;
    }
    uint32_t words[4 * kRaw];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t v = k + e < K ? (uint32_t)reinterpret_cast<const uint16_t *>(row)[k + e] : 0u;
            words[e >> 1] = (e & 1) ? words[e >> 1] | v << 16 : v;
        } else {
            words[e] = k + e < K ? reinterpret_cast<const uint32_t *>(row)[k + e] : 0u;
        }
    }
#pragma unroll
    for (int r = 0; r < kRaw; ++r) raw[r] = u32x4{words[4 * r], words[4 * r + 1], words[4 * r + 2], words[4 * r + 3]};
}

// NT tiles of 16 columns and MB blocks of 16 rows per workgroup, WAVES wavefronts that split K, GROUPS scales per 128 rows.
// Codes and scales are requested kAhead tiles of 128 rows before they are used, A of a single block of rows one tile, of two
// blocks half a tile at a time (64 k: whole lines of a row of 16 bits at once, before the other wavefronts' rows push
// them out of the cache).
template <typename T, int NT, int MB, int WAVES, int GROUPS>
__global__ __launch_bounds__(WAVES * 64) void gemm_w4_kernel(GemmW4Args g) {
    using Q = Kind<T>;
    constexpr int kRaw = sizeof(T) / 2, kParts = Q::kParts, kAhead = 2, kSpan = 4 / GROUPS;
    constexpr bool kAheadA = MB == 1;
    extern __shared__ __attribute__((aligned(16))) float sums[];  // [WAVES][MB][NT][64][4]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int h = lane >> 4, c = lane & 15;
    const int tn0 = (int)blockIdx.x * NT;
    const int64_t m0 = (int64_t)blockIdx.y * (16 * MB);
    const int k0 = __builtin_amdgcn_readfirstlane((int)((int64_t)g.tiles_k * wave / WAVES));
    const int k1 = __builtin_amdgcn_readfirstlane((int)((int64_t)g.tiles_k * (wave + 1) / WAVES));

    const T *row[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {  // rows past the last read the last: nothing of theirs is stored
        const int64_t m = m0 + b * 16 + c;
        row[b] = (const T *)g.a + (m < g.M ? m : g.M - 1) * g.lda + 8 * h;
    }
    const u32x4 *codes[NT];
    int64_t column[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int tn = tn0 + t < g.tiles_n ? tn0 + t : g.tiles_n - 1;
        codes[t] = g.codes + (int64_t)tn * g.tiles_k * 64 + lane;
        const int64_t n = (int64_t)tn * kTileN + c;
        column[t] = n < g.N ? n : g.N - 1;
    }
    const int last_group = (int)((g.K - 1) / (32 * kSpan));  // a group that lies wholly past K has no scale; its sums are zero

    struct Slot {
        u32x4 w[NT];
        // Of group h % GROUPS of the tile: the lanes of a column hold all of them between them and exchange them at a group's
        // end.  (With every lane loading all: 16 rows of 8192 x 16384 in groups of 32 in 70 us instead of 34.)
        float scale[NT], zero[NT];
    };
    Slot slots[kAhead];
    u32x4 ahead_a[2][kAheadA ? 4 : 1][kRaw], half_a[2][MB][kRaw];
    const int64_t full = g.vec_a ? g.K / kTileK : 0;  // tiles of A that are read 16 bytes at a time; the others element by element
    const int kw = __builtin_amdgcn_readfirstlane((int)(full < k0 ? k0 : full < k1 ? full : k1));
    auto request = [&](Slot &s, int kb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            s.w[t] = codes[t][(int64_t)kb * 64];
            const int own = kb * GROUPS + h % GROUPS, group = own < last_group ? own : last_group;
            const int64_t at = (int64_t)group * g.N + column[t];
            s.scale[t] = g.scales[at];
            s.zero[t] = g.zeros ? (float)g.zeros[at] : 8.0f;
        }
    };
    auto request_a = [&](u32x4 (&a)[kAheadA ? 4 : 1][kRaw], int kb) {
        if constexpr (kAheadA) {
#pragma unroll
            for (int q = 0; q < 4; ++q) load_eight<true>(row[0], (int64_t)kb * kTileK + 32 * q, g.K - 8 * h, true, a[q]);
        }
    };
    auto request_half = [&](int64_t k) {
        if constexpr (!kAheadA) {
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) load_eight<true>(row[b], k + 32 * e, g.K - 8 * h, true, half_a[e][b]);
        }
    };

    f32x4 total[MB][NT];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) total[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = {Q::kOnes, Q::kOnes, Q::kOnes, Q::kOnes};

    auto consume = [&](const Slot &s, const u32x4 (&a)[kAheadA ? 4 : 1][kRaw], int kb, int next, auto whole) {
        constexpr bool kWhole = decltype(whole)::value != 0;
        f32x4 acc[MB][NT], sum_a[MB];
        float zero[NT];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            auto of_group = [&](float v) {
                return GROUPS == 1 ? v : __uint_as_float(__builtin_amdgcn_ds_bpermute((q / kSpan * 16 + c) * 4, (int)__float_as_uint(v)));
            };
            if (q % kSpan == 0) {
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    if (!kCentred<T>) sum_a[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                if (kCentred<T>)
#pragma unroll
                    for (int t = 0; t < NT; ++t) zero[t] = of_group(s.zero[t]) * (1.0f / Q::kUnit);
            }
            u32x4 bw[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (kCentred<T>) bw[t] = expand_centred<T>(s.w[t][q], zero[t]);
                else bw[t] = expand<T>(s.w[t][q]);
            }
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                u32x4 raw[kRaw], part[kParts];
                if constexpr (kWhole) {
#pragma unroll
                    for (int r = 0; r < kRaw; ++r) raw[r] = kAheadA ? a[kAheadA ? q : 0][r] : half_a[q & 1][b][r];
                } else {
                    load_eight<false>(row[b], (int64_t)kb * kTileK + 32 * q, g.K - 8 * h, g.vec_a != 0, raw);
                }
                operand<T>(raw, part);
#pragma unroll
                for (int p = kParts - 1; p >= 0; --p) {
                    if (!kCentred<T>) sum_a[b] = Q::mfma(part[p], ones, sum_a[b]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[b][t] = Q::mfma(part[p], bw[t], acc[b][t]);
                }
            }
            if (kWhole && (q & 1)) request_half(q == 1 ? (int64_t)kb * kTileK + 64 : (int64_t)next * kTileK);
            if (q % kSpan == kSpan - 1) {  // the end of a group
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float scale = of_group(s.scale[t]), offset = kCentred<T> ? 0.0f : 16.0f + of_group(s.zero[t]);
#pragma unroll
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float sum = kCentred<T> ? acc[b][t][r] : __builtin_fmaf(-offset, sum_a[b][r], acc[b][t][r]);
                            total[b][t][r] = __builtin_fmaf(scale, sum, total[b][t][r]);
                        }
                }
            }
        }
    };
    // a request past the last tile reads the last again (unused)
    auto last = [&](int kb) { return kb < kw ? kb : kw - 1; };
    if (k0 < kw) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) request(slots[d], last(k0 + d));
        request_a(ahead_a[0], k0);
        request_half((int64_t)k0 * kTileK);
    }
    static_assert(kAhead == 2, "the two buffers of A take turns with the slots");
    for (int kb = k0; kb < kw; kb += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            if (kb + d >= kw) break;
            request_a(ahead_a[d ^ 1], last(kb + d + 1));
            consume(slots[d], ahead_a[d], kb + d, last(kb + d + 1), Constant<1>{});
            request(slots[d], last(kb + d + kAhead));
        }
    }
#pragma unroll 1
    for (int kb = kw; kb < k1; ++kb) {
        request(slots[0], kb);
        consume(slots[0], ahead_a[0], kb, kb, Constant<0>{});
    }

    // Lane (h, c) holds rows 4 h .. 4 h + 3 of column c of each block.
    f32x4 *mine = reinterpret_cast<f32x4 *>(sums) + (size_t)wave * MB * NT * 64;
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) mine[(b * NT + t) * 64 + lane] = total[b][t];
    __syncthreads();
    const int64_t n0 = (int64_t)tn0 * kTileN;
    for (int i = threadIdx.x; i < MB * 16 * NT * 16; i += WAVES * 64) {
        const int n = i % (NT * 16), m = i / (NT * 16);
        if (m0 + m >= g.M || n0 + n >= g.N) continue;
        const int at = (((m >> 4) * NT + (n >> 4)) * 64 + ((m & 15) >> 2) * 16 + (n & 15)) * 4 + (m & 3);
        float v = sums[at];
#pragma unroll
        for (int wv = 1; wv < WAVES; ++wv) v += sums[wv * MB * NT * 256 + at];
        ((T *)g.out)[(m0 + m) * g.ldo + n0 + n] = (T)(v * Q::kUnit);
    }
}

template <typename T, int NT, int MB, int WAVES, int GROUPS>
cn_status launch_gemm(const GemmW4Args &g, hipStream_t st) {
    constexpr size_t lds = (size_t)WAVES * MB * NT * 256 * sizeof(float);
    static_assert(lds <= 65536, "no more than a launch may ask for by itself");
    const dim3 grid((unsigned)((g.tiles_n + NT - 1) / NT), (unsigned)((g.M + 16 * MB - 1) / (16 * MB)));
    hipLaunchKernelGGL((gemm_w4_kernel<T, NT, MB, WAVES, GROUPS>), grid, dim3(WAVES * 64), lds, st, g);
    CN_HIP(hipGetLastError());
    return CN_OK;
}

template <typename T, int GROUPS>
cn_status run_gemm(const GemmW4Args &g, hipStream_t st) {
    if (g.M > 16) {
        // Two blocks of rows per workgroup (four: 64 rows of 8192 x 16384 in 78 us instead of 61), and four tiles of columns where that
        // still makes a workgroup per compute unit: A comes from the L2 anew for every workgroup, and its lines are what bounds
        // this (64 rows of 8192 x 16384 61 us, 91 with two tiles; of 8192 x 8192 32 and 48; 32 rows of it, which would be 128
        // workgroups, 32 and 24).
        const int64_t workgroups = (int64_t)(g.tiles_n / 4) * ((g.M + 31) / 32);
        if constexpr (GROUPS < 4) {  // (four columns of groups of 32 would spill)
            if (workgroups >= 256) return launch_gemm<T, 4, 2, 8, GROUPS>(g, st);
        }
        return launch_gemm<T, 2, 2, 8, GROUPS>(g, st);
    }
    // Wide workgroups share A and its sums (one row of 16384 x 16384: 33.0 us, 38.3 us with narrow ones, 34.5 with four tiles of
    // columns, 34.0 with one tile of 128 rows ahead, 38.6 with four); narrow ones, with K among more wavefronts, fill the chip.
    if (g.tiles_n >= 512) return launch_gemm<T, 2, 1, 8, GROUPS>(g, st);
    if (g.tiles_n > 256) return launch_gemm<T, 1, 1, 8, GROUPS>(g, st);
    return launch_gemm<T, 1, 1, sizeof(T) == 2 ? 16 : 8, GROUPS>(g, st);  // (fp32 operands take too many registers for sixteen)
}

// ---- quantisation --------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows of 64 C columns, lane (h, l) rows 32 t + 8 h + i of C neighbouring ones: the codes of its four words
// each.  Workgroups that follow each other are neighbours along the rows of W.  (16384 x 8192 bf16, with workgroups going down
// the columns, one column a lane and every lane finding the scales by itself: 300 us.)
struct QuantArgs {
    int64_t K, N, ldw;
    int64_t tiles_k, tiles_n, blocks_n;
    int group;
};
constexpr float kLargest = 3.402823466e38f;

// Eight codes, round(v / scale) with ties to even, decided exactly: the product with the reciprocal is off by 10^-6 at most, so its
// rounding is the code or a neighbour of it, and the remainder tells which: the code is right while |remainder| is below
// scale / 2, or equal to it if the code is even.  The remainder has a single rounding that keeps this comparison (it is a
// multiple of scale's last place no larger than scale).  No branch for the rare doubtful ones: weights of 16 bits often
// are half of their group's largest, so that some lane always had one (135 us instead of 108 for 16384 x 8192 bf16; 16.4 instead of 17.1 for 4096 x 4096 fp32).  A scale of 0
// or NaN gives the code that stands for 0.
template <int C>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[8][C], int j, float scale, float zero) {
    const float lift = scale < 0x1p-90f ? 0x1p90f : 1.0f;  // keeps the reciprocal finite; exact either way
    const float s = scale * lift, inverse = 1.0f / s;
    const int half = (int)__float_as_uint(0.5f * s), z = (int)zero;
    uint32_t packed = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = v[i][j] * lift, q = rintf(x * inverse), rest = __builtin_fmaf(-q, s, x);
        const int n = (int)q, off = (int)__float_as_uint(rest);
        const float most = __uint_as_float((uint32_t)(half - (n & 1)));
        const int code = n + z + (fabsf(rest) > most ? off >> 31 | 1 : 0);
        packed |= (uint32_t)(code < 0 ? 0 : code > 15 ? 15 : code) << (4 * i);
    }
    return scale > 0.0f ? packed : (uint32_t)z * 0x11111111u;
}

template <typename T, bool ZP, int C>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs g, const T *__restrict__ w, u32x4 *__restrict__ codes,
                                                       float *__restrict__ scales, uint8_t *__restrict__ zeros) {
    constexpr int kCols = 64 * C;
    __shared__ float top[4][4][kCols], low[ZP ? 4 : 1][4][kCols];  // [t][h][column]: largest value (magnitude), smallest
    __shared__ float scale_of[4][kCols], zero_of[4][kCols];        // [group of the 128 rows][column]
    const int h = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t kb = blockIdx.x / g.blocks_n, n0 = blockIdx.x % g.blocks_n * kCols, n = n0 + l * C;
    const int64_t k0 = kb * kTileK + 8 * h;
    const bool inside = kb * kTileK + kTileK <= g.K && n0 + kCols <= g.N;  // of the whole workgroup
    float v[4][8][C];
    if (inside) {
        const T *at = w + k0 * g.ldw + n;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) load_f32<C>(at + (32 * t + i) * g.ldw, v[t][i]);
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int64_t k = k0 + 32 * t + i;
                if (k < g.K && n < g.N) {
                    load_f32<C>(w + k * g.ldw + n, v[t][i]);
                } else {
#pragma unroll
                    for (int j = 0; j < C; ++j) v[t][i][j] = 0.0f;  // zero changes no range: it belongs to every one
                }
            }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < C; ++j) {
            float hi = 0.0f, lo = 0.0f, odd = 0.0f;  // odd: NaN if something is not finite
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = v[t][i][j];
                odd = __builtin_fmaf(x, 0.0f, odd);
                hi = fmaxf(hi, ZP ? x : fabsf(x));
                if (ZP) lo = fminf(lo, x);
            }
            top[t][h][l * C + j] = odd == 0.0f ? hi : __uint_as_float(0x7f800000u);
            if (ZP) low[t][h][l * C + j] = lo;
        }
    __syncthreads();
    const int span = g.group / 32, groups = 4 / span;  // words of t per group: 1, 2 or 4
    for (int x = threadIdx.x; x < groups * kCols; x += 256) {
        const int group = x / kCols, col = x % kCols;
        float hi = 0.0f, lo = 0.0f;
        for (int t = group * span; t < group * span + span; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                hi = fmaxf(hi, top[t][q][col]);
                if (ZP) lo = fminf(lo, low[t][q][col]);
            }
        const bool finite = hi <= kLargest;
        // one rounding to fp32: quotients by 7 and 15 are never so near a midpoint that the one to 64 bits matters
        float scale = (float)(((double)hi - (double)lo) / (ZP ? 15.0 : 7.0));
        float zero = ZP ? (scale > 0.0f && finite ? (float)rint(-(double)lo / (double)scale) : 0.0f) : 8.0f;
        zero = fminf(fmaxf(zero, 0.0f), 15.0f);
        if (!finite) scale = __uint_as_float(0x7fc00000u);  // the whole group decodes to NaN
        scale_of[group][col] = scale;
        zero_of[group][col] = zero;
        const int64_t at = kb * groups + group;
        if (n0 + col < g.N && at * g.group < g.K) {
            scales[at * g.N + n0 + col] = scale;
            if (ZP) zeros[at * g.N + n0 + col] = (uint8_t)zero;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C; ++j) {
        u32x4 word;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float scale = scale_of[t / span][l * C + j], zero = zero_of[t / span][l * C + j];
            uint32_t packed = codes_of<C>(v[t], j, scale, zero);
            if (!inside) {
                const int64_t rows = g.K - (k0 + 32 * t);  // that there are
                if (n + j >= g.N || rows <= 0) packed = 0u;
                else if (rows < 8) packed &= (1u << (4 * rows)) - 1u;
            }
            word[t] = packed;
        }
        const int64_t a = (n + j) / kTileN;
        if (a < g.tiles_n) codes[(a * g.tiles_k + kb) * 64 + h * 16 + ((n + j) & 15)] = word;
    }
}

// STREAM: past the caches, for results that do not fit them (16384 x 8192 fp32 in 94.5 us instead of 103, and what runs next finds
// its data: quantising anew 76 instead of 108; 4096 x 4096, which fits, takes 13.8 instead of 13.2).
constexpr size_t kLastCache = (size_t)256 << 20;

template <typename T, bool ZP, int C, bool STREAM>
__global__ __launch_bounds__(256) void dequantize_kernel(QuantArgs g, const u32x4 *__restrict__ codes, const float *__restrict__ scales,
                                                         const uint8_t *__restrict__ zeros, T *__restrict__ out) {
    const int h = threadIdx.x >> 6, l = threadIdx.x & 63;
    const int64_t kb = blockIdx.x / g.blocks_n, n = blockIdx.x % g.blocks_n * (64 * C) + l * C;
    if (n >= g.N) return;
    u32x4 word[C];
#pragma unroll
    for (int j = 0; j < C; ++j) word[j] = codes[((n + j) / kTileN * g.tiles_k + kb) * 64 + h * 16 + ((n + j) & 15)];
    const int64_t k0 = kb * kTileK + 8 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t first = kb * kTileK + 32 * t;
        if (first >= g.K) break;
        const int64_t at = first / g.group * g.N + n;
        float scale[C], zero[C];
        load_f32<C>(scales + at, scale);
#pragma unroll
        for (int j = 0; j < C; ++j) zero[j] = ZP ? (float)zeros[at + j] : 8.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t k = k0 + 32 * t + i;
            float v[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
                v[j] = ((float)((word[j][t] >> (4 * i)) & 15u) - zero[j]) * scale[j];
                asm volatile("" : "+v"(v[j]));  // a product that becomes fp16 at once would skip its rounding to fp32
            }
            if (k < g.K) store_f32<C, STREAM>(out + k * g.ldw + n, v);
        }
    }
}

// Columns of a lane: two where their loads are whole words.
QuantArgs quant_args(int64_t K, int64_t N, int64_t ld, int group, int columns) {
    const int64_t wide = 64 * columns;
    return QuantArgs{K, N, ld, tiles_k_of(K), tiles_n_of(N), (N + wide - 1) / wide, group};
}

cn_status check_weights(const char *what, int64_t K, int64_t N, int group) {
    if (K < 0 || N < 0) { set_error("%s: negative dimension", what); return CN_ERR_SHAPE; }
    if (group != 32 && group != 64 && group != 128) { set_error("%s: groups of %d rows (32, 64 or 128)", what, group); return CN_ERR_ARG; }
    if (K > 0x7fffffffLL || N > 0x7fffffffLL || !launchable(tiles_k_of(K) * ((N + 63) / 64), 256)) {
        set_error("%s: too many weights for one launch", what);
        return CN_ERR_SHAPE;
    }
    return CN_OK;
}

}  // namespace

}  // namespace cn

using namespace cn;

extern "C" {

size_t cn_w4_code_words(int64_t K, int64_t N) {
    if (K <= 0 || N <= 0) return 0;
    return (size_t)tiles_n_of(N) * (size_t)tiles_k_of(K) * 256;
}

cn_status cn_quantize_4bit(const void *W, int dtype, int64_t K, int64_t N, int64_t ldw, int group, int32_t *codes, float *scales,
                           uint8_t *zeros, void *stream) {
    if (!known_dtype(dtype)) { set_error("quantize_4bit: unknown element type %d", dtype); return CN_ERR_ARG; }
    cn_status s = check_weights("quantize_4bit", K, N, group);
    if (s != CN_OK) return s;
    if (ldw < N) { set_error("quantize_4bit: leading dimension too small"); return CN_ERR_SHAPE; }
    if (K == 0 || N == 0) return CN_OK;
    if (!W || !codes || !scales) { set_error("quantize_4bit: NULL pointer"); return CN_ERR_NULL; }
    if (!aligned_to(codes, 16)) { set_error("quantize_4bit: the codes are not aligned to 16 bytes"); return CN_ERR_ARG; }
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto zero, auto columns) {
        typedef decltype(zero) T;
        constexpr int C = decltype(columns)::value;
        const QuantArgs g = quant_args(K, N, ldw, group, C);
        const dim3 grid((unsigned)(g.tiles_k * g.blocks_n));
        if (zeros) hipLaunchKernelGGL((quantize_kernel<T, true, C>), grid, dim3(256), 0, st, g, (const T *)W, (u32x4 *)codes, scales, zeros);
        else       hipLaunchKernelGGL((quantize_kernel<T, false, C>), grid, dim3(256), 0, st, g, (const T *)W, (u32x4 *)codes, scales, zeros);
    };
    const bool pairs = N % 2 == 0 && ldw % 2 == 0 && aligned_to(W, 2 * dtype_bytes(dtype));
    if (dtype == CN_F32) go(0.0f, Constant<1>{});
    else if (dtype == CN_F16) pairs ? go((f16_t)0, Constant<2>{}) : go((f16_t)0, Constant<1>{});
    else pairs ? go((bf16_t)0, Constant<2>{}) : go((bf16_t)0, Constant<1>{});
    CN_HIP(hipGetLastError());
    return CN_OK;
}

cn_status cn_dequantize_4bit(const int32_t *codes, const float *scales, const uint8_t *zeros, int64_t K, int64_t N, int group,
                             void *out, int dtype, int64_t ldo, void *stream) {
    if (!known_dtype(dtype)) { set_error("dequantize_4bit: unknown element type %d", dtype); return CN_ERR_ARG; }
    cn_status s = check_weights("dequantize_4bit", K, N, group);
    if (s != CN_OK) return s;
    if (ldo < N) { set_error("dequantize_4bit: leading dimension too small"); return CN_ERR_SHAPE; }
    if (K == 0 || N == 0) return CN_OK;
    if (!codes || !scales || !out) { set_error("dequantize_4bit: NULL pointer"); return CN_ERR_NULL; }
    if (!aligned_to(codes, 16)) { set_error("dequantize_4bit: the codes are not aligned to 16 bytes"); return CN_ERR_ARG; }
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto zero, auto columns) {
        typedef decltype(zero) T;
        constexpr int C = decltype(columns)::value;
        const QuantArgs g = quant_args(K, N, ldo, group, C);
        const dim3 grid((unsigned)(g.tiles_k * g.blocks_n));
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, g, (const u32x4 *)codes, scales, zeros, (T *)out);
        };
        const bool stream_out = C > 1 && (size_t)K * (size_t)N * sizeof(T) > kLastCache;
        if (stream_out) zeros ? launch(dequantize_kernel<T, true, C, (C > 1)>) : launch(dequantize_kernel<T, false, C, (C > 1)>);
        else zeros ? launch(dequantize_kernel<T, true, C, false>) : launch(dequantize_kernel<T, false, C, false>);
    };
    const bool pairs = N % 2 == 0 && ldo % 2 == 0 && aligned_to(out, 2 * dtype_bytes(dtype)) && aligned_to(scales, 8);
    if (dtype == CN_F32) pairs ? go(0.0f, Constant<2>{}) : go(0.0f, Constant<1>{});
    else if (dtype == CN_F16) pairs ? go((f16_t)0, Constant<2>{}) : go((f16_t)0, Constant<1>{});
    else pairs ? go((bf16_t)0, Constant<2>{}) : go((bf16_t)0, Constant<1>{});
    CN_HIP(hipGetLastError());
    return CN_OK;
}

cn_status cn_gemm_w4(int64_t M, int64_t N, int64_t K, const void *A, int dtype, int64_t lda, const int32_t *codes, const float *scales,
                     const uint8_t *zeros, int group, void *out, int64_t ldo, void *stream) {
    if (!known_dtype(dtype)) { set_error("gemm_w4: unknown element type %d", dtype); return CN_ERR_ARG; }
    cn_status s = check_weights("gemm_w4", K, N, group);
    if (s != CN_OK) return s;
    if (M < 0) { set_error("gemm_w4: negative dimension"); return CN_ERR_SHAPE; }
    if (lda < K || ldo < N) { set_error("gemm_w4: leading dimension too small"); return CN_ERR_SHAPE; }
    if ((M + 15) / 16 > 65535) { set_error("gemm_w4: more than 2^20 rows"); return CN_ERR_SHAPE; }
    if (M == 0 || N == 0) return CN_OK;
    if (!out || (K > 0 && (!A || !codes || !scales))) { set_error("gemm_w4: NULL pointer"); return CN_ERR_NULL; }
    if (!aligned_to(codes, 16)) { set_error("gemm_w4: the codes are not aligned to 16 bytes"); return CN_ERR_ARG; }
    if (out == A) { set_error("gemm_w4: the output is A"); return CN_ERR_ARG; }
    if (!launchable(tiles_n_of(N) / 2 + 1, 512)) { set_error("gemm_w4: too many columns for one launch"); return CN_ERR_SHAPE; }
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    GemmW4Args g{};
    g.a = A; g.codes = (const u32x4 *)codes; g.scales = scales; g.zeros = zeros; g.out = out;
    g.M = M; g.N = N; g.K = K; g.lda = lda; g.ldo = ldo;
    g.tiles_k = (int)tiles_k_of(K); g.tiles_n = (int)tiles_n_of(N);
    g.vec_a = aligned_to(A, 16) && lda % (16 / (int64_t)dtype_bytes(dtype)) == 0;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto zero) -> cn_status {
        typedef decltype(zero) T;
        return group == 128 ? run_gemm<T, 1>(g, st) : group == 64 ? run_gemm<T, 2>(g, st) : run_gemm<T, 4>(g, st);
    };
    return dtype == CN_F32 ? go(0.0f) : dtype == CN_F16 ? go((f16_t)0) : go((bf16_t)0);
}

}  // extern "C"
