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
//   * Codes become numbers without arithmetic: bits 3 .. 6 of the bf16 pattern of 16.0 (bits 6 .. 9 of the fp16 one) set to q
//     give exactly 16 + q, a shift and an and-or for two weights.  The 16 and the zero point leave again behind the sum:
//         sum a (q - z) = sum a (16 + q) - (16 + z) sum a,
//     where sum a comes from one more matrix instruction against ones, in the same fp32 accumulators and the same order.
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
    int group_shift;       // group = 1 << group_shift
    int vec_a;             // rows of A allow 16-byte loads
};

// A operand of one instruction as the words of its kind, and how many of them a number needs.
template <typename T> struct Kind;
template <> struct Kind<bf16_t> {
    static constexpr int kParts = 1;
    static constexpr uint32_t kMagic = 0x41804180u, kMask = 0x00780078u, kOnes = 0x3f803f80u;
    static constexpr int kShift = 3;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Kind<float> : Kind<bf16_t> {
    static constexpr int kParts = 3;
};
template <> struct Kind<f16_t> {
    static constexpr int kParts = 1;
    static constexpr uint32_t kMagic = 0x4c004c00u, kMask = 0x03c003c0u, kOnes = 0x3c003c00u;
    static constexpr int kShift = 6;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Words of the B operand from eight codes: word j holds k = 2 j and 2 j + 1 of the lane, so nibbles 2 j and 2 j + 1.  They are
// moved to the low and the high half: first the odd nibbles up by 12 bits (w << 12), then both to their place.
template <typename T>
__device__ __forceinline__ u32x4 expand(uint32_t w) {
    using Q = Kind<T>;
    u32x4 b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // nibble 2 j from bit 8 j to bit kShift, nibble 2 j + 1 from bit 8 j + 4 to bit 16 + kShift
        const int down = 8 * j - Q::kShift, up = 12 + Q::kShift - 8 * j;
        const uint32_t lo = down >= 0 ? w >> down : w << -down;
        const uint32_t hi = up >= 0 ? w << up : w >> -up;
        b[j] = (lo & (Q::kMask & 0xffffu)) | (hi & (Q::kMask & 0xffff0000u)) | Q::kMagic;
    }
    return b;
}

// Eight consecutive elements of A as operand words.
template <typename T>
__device__ __forceinline__ void operand(const u32x4 (&raw)[sizeof(T) / 2], u32x4 (&part)[Kind<T>::kParts]) {
    if constexpr (sizeof(T) == 2) {
        part[0] = raw[0];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t piece[3][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t x = raw[(2 * j + e) >> 2][(2 * j + e) & 3];
                const uint32_t h = x & 0xffff0000u;  // the first eight bits
                const float r = __uint_as_float(x) - __uint_as_float(h);
                const uint32_t m = __float_as_uint(r) & 0xffff0000u;
                const float l = r - __uint_as_float(m);  // at most eight bits are left
                piece[0][e] = h;
                piece[1][e] = m;
                piece[2][e] = __float_as_uint(l);
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) part[p][j] = (piece[p][0] >> 16) | (piece[p][1] & 0xffff0000u);
        }
    }
}

// NT tiles of 16 columns and MB blocks of 16 rows per workgroup, WAVES wavefronts that split K.
template <typename T, int NT, int MB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gemm_w4_kernel(GemmW4Args g) {
    using Q = Kind<T>;
    constexpr int kRaw = sizeof(T) / 2, kParts = Q::kParts;
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
        row[b] = (const T *)g.a + (m < g.M ? m : g.M - 1) * g.lda;
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

    f32x4 total[MB][NT];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t) total[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = {Q::kOnes, Q::kOnes, Q::kOnes, Q::kOnes};

    u32x4 w[NT];
    if (k0 < k1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = codes[t][(int64_t)k0 * 64];
    }
    for (int kb = k0; kb < k1; ++kb) {
        u32x4 next[NT];
        const int ahead = kb + 1 < k1 ? kb + 1 : kb;
#pragma unroll
        for (int t = 0; t < NT; ++t) next[t] = codes[t][(int64_t)ahead * 64];
        u32x4 raw[MB][4][kRaw];
        const int64_t kk = (int64_t)kb * kTileK + 8 * h;
        if (g.vec_a && (int64_t)kb * kTileK + kTileK <= g.K) {
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int r = 0; r < kRaw; ++r) raw[b][s][r] = *(reinterpret_cast<const u32x4 *>(row[b] + kk + 32 * s) + r);
        } else {  // element by element, zeros past K
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t words[4 * kRaw];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int64_t k = kk + 32 * s + e;
                        if constexpr (sizeof(T) == 2) {
                            const uint32_t v = k < g.K ? (uint32_t)reinterpret_cast<const uint16_t *>(row[b])[k] : 0u;
                            words[e >> 1] = (e & 1) ? words[e >> 1] | v << 16 : v;
                        } else {
                            words[e] = k < g.K ? reinterpret_cast<const uint32_t *>(row[b])[k] : 0u;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < kRaw; ++r) raw[b][s][r] = u32x4{words[4 * r], words[4 * r + 1], words[4 * r + 2], words[4 * r + 3]};
                }
        }
        f32x4 acc[MB][NT], sum_a[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            sum_a[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[b][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 bw[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) bw[t] = expand<T>(w[t][s]);
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                u32x4 part[kParts];
                operand<T>(raw[b][s], part);
#pragma unroll
                for (int p = kParts - 1; p >= 0; --p) {
                    sum_a[b] = Q::mfma(part[p], ones, sum_a[b]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[b][t] = Q::mfma(part[p], bw[t], acc[b][t]);
                }
            }
            if (((s + 1) << 5 & ((1 << g.group_shift) - 1)) == 0) {  // the end of a group
                // a group that lies wholly past K has no scale; its sums are zero
                int64_t group = ((int64_t)kb * kTileK + 32 * s) >> g.group_shift;
                const int64_t last = (g.K - 1) >> g.group_shift;
                group = group < last ? group : last;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int64_t at = group * g.N + column[t];
                    const float scale = g.scales[at];
                    const float offset = 16.0f + (g.zeros ? (float)g.zeros[at] : 8.0f);
#pragma unroll
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            total[b][t][r] += scale * (acc[b][t][r] - offset * sum_a[b][r]);
                            acc[b][t][r] = 0.0f;
                        }
                }
#pragma unroll
                for (int b = 0; b < MB; ++b) sum_a[b] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = next[t];
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
        ((T *)g.out)[(m0 + m) * g.ldo + n0 + n] = (T)v;
    }
}

template <typename T, int NT, int MB, int WAVES>
cn_status launch_gemm(const GemmW4Args &g, int device, hipStream_t st) {
    const size_t lds = (size_t)WAVES * MB * NT * 256 * sizeof(float);
    static OncePerDevice configured;
    if (lds > 65536 && configured.first(device))
        CN_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&gemm_w4_kernel<T, NT, MB, WAVES>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    const dim3 grid((unsigned)((g.tiles_n + NT - 1) / NT), (unsigned)((g.M + 16 * MB - 1) / (16 * MB)));
    hipLaunchKernelGGL((gemm_w4_kernel<T, NT, MB, WAVES>), grid, dim3(WAVES * 64), lds, st, g);
    CN_HIP(hipGetLastError());
    return CN_OK;
}

template <typename T>
cn_status run_gemm(const GemmW4Args &g, int device, hipStream_t st) {
    if (g.M > 16) return g.M > 32 ? launch_gemm<T, 2, 4, 8>(g, device, st) : launch_gemm<T, 2, 2, 8>(g, device, st);
    // wide workgroups read A less often, narrow ones are enough to fill the chip
    if (g.tiles_n >= 2048) return launch_gemm<T, 4, 1, 8>(g, device, st);
    if (g.tiles_n >= 1024) return launch_gemm<T, 2, 1, 8>(g, device, st);
    return launch_gemm<T, 1, 1, 8>(g, device, st);
}

// ---- quantisation --------------------------------------------------------------------------------------------------------
// A workgroup takes 128 rows of 64 columns, lane (h, column) rows 32 t + 8 h + i: the codes of its four words.
struct QuantArgs {
    int64_t K, N, ldw;
    int64_t tiles_k, tiles_n;
    int group;
};

template <typename T, bool ZP>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs g, const T *__restrict__ w, u32x4 *__restrict__ codes,
                                                       float *__restrict__ scales, uint8_t *__restrict__ zeros) {
    __shared__ float top[4][4][64], low[4][4][64];  // [t][h][column]: largest value (magnitude), smallest
    const int h = threadIdx.x >> 6, col = threadIdx.x & 63;
    const int64_t kb = blockIdx.x % g.tiles_k, n = blockIdx.x / g.tiles_k * 64 + col;
    const int64_t k0 = kb * kTileK + 8 * h;
    float v[4][8];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t k = k0 + 32 * t + i;
            v[t][i] = k < g.K && n < g.N ? (float)w[k * g.ldw + n] : 0.0f;  // zero changes no range: it belongs to every one
        }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        float hi = 0.0f, lo = 0.0f;
        bool odd = false;  // something is not finite
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            odd |= !(fabsf(v[t][i]) <= 3.402823466e38f);
            if (ZP) {
                hi = fmaxf(hi, v[t][i]);
                lo = fminf(lo, v[t][i]);
            } else {
                hi = fmaxf(hi, fabsf(v[t][i]));
            }
        }
        top[t][h][col] = odd ? __uint_as_float(0x7f800000u) : hi;
        if (ZP) low[t][h][col] = lo;
    }
    __syncthreads();
    u32x4 word;
    float scale = 0.0f, inverse = 0.0f, lift = 1.0f, zero = 8.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int span = g.group / 32;  // words of t per group: 1, 2 or 4
        if (t % span == 0) {
            float hi = 0.0f, lo = 0.0f;
            for (int s = t; s < t + span; ++s)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    hi = fmaxf(hi, top[s][q][col]);
                    if (ZP) lo = fminf(lo, low[s][q][col]);
                }
            const bool finite = hi <= 3.402823466e38f;
            // one rounding to fp32: quotients by 7 and 15 are never so near a midpoint that the one to 64 bits matters
            scale = (float)(((double)hi - (double)lo) / (ZP ? 15.0 : 7.0));
            zero = ZP ? (scale > 0.0f && finite ? (float)rint(-(double)lo / (double)scale) : 0.0f) : 8.0f;
            zero = fminf(fmaxf(zero, 0.0f), 15.0f);
            if (!finite) scale = __uint_as_float(0x7fc00000u);  // the whole group decodes to NaN
            lift = scale < 0x1p-90f ? 0x1p90f : 1.0f;  // keeps the reciprocal finite; exact either way
            inverse = scale > 0.0f ? 1.0f / (scale * lift) : 0.0f;
            const int64_t group = (kb * kTileK + 32 * t) / g.group;
            if (h == 0 && n < g.N && group * g.group < g.K) {
                scales[group * g.N + n] = scale;
                if (ZP) zeros[group * g.N + n] = (uint8_t)zero;
            }
        }
        uint32_t packed = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // round(v / scale), ties to even, decided exactly: the remainder of the candidate has a single rounding that keeps its
            // comparison with scale / 2 (it is a multiple of scale's last place no larger than scale)
            const float x = v[t][i] * lift, s = scale * lift;
            float q = rintf(x * inverse);
            const float rest = __builtin_fmaf(-q, s, x), twice = rest + rest;
            if (twice > s || (twice == s && ((int)q & 1))) q += 1.0f;
            else if (-twice > s || (-twice == s && ((int)q & 1))) q -= 1.0f;
            q = fminf(fmaxf(q + zero, 0.0f), 15.0f);
            const int64_t k = k0 + 32 * t + i;
            const uint32_t code = inverse > 0.0f ? (uint32_t)q : (uint32_t)zero;
            packed |= (k < g.K && n < g.N ? code : 0u) << (4 * i);
        }
        word[t] = packed;
    }
    const int64_t a = n / kTileN;
    if (a < g.tiles_n) codes[(a * g.tiles_k + kb) * 64 + h * 16 + (col & 15)] = word;
}

template <typename T, bool ZP>
__global__ __launch_bounds__(256) void dequantize_kernel(QuantArgs g, const u32x4 *__restrict__ codes, const float *__restrict__ scales,
                                                         const uint8_t *__restrict__ zeros, T *__restrict__ out) {
    const int h = threadIdx.x >> 6, col = threadIdx.x & 63;
    const int64_t kb = blockIdx.x % g.tiles_k, n = blockIdx.x / g.tiles_k * 64 + col;
    if (n >= g.N) return;
    const u32x4 word = codes[(n / kTileN * g.tiles_k + kb) * 64 + h * 16 + (col & 15)];
    const int64_t k0 = kb * kTileK + 8 * h;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int64_t first = kb * kTileK + 32 * t;
        if (first >= g.K) break;
        const int64_t at = first / g.group * g.N + n;
        const float scale = scales[at], zero = ZP ? (float)zeros[at] : 8.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t k = k0 + 32 * t + i;
            float v = ((float)((word[t] >> (4 * i)) & 15u) - zero) * scale;
            asm volatile("" : "+v"(v));  // a product that becomes fp16 at once would skip its rounding to fp32
            if (k < g.K) out[k * g.ldw + n] = (T)v;
        }
    }
}

cn_status check_weights(const char *what, int64_t K, int64_t N, int group) {
    if (K < 0 || N < 0) { set_error("%s: negative dimension", what); return CN_ERR_SHAPE; }
    if (group != 32 && group != 64 && group != 128) { set_error("%s: groups of %d rows (32, 64 or 128)", what, group); return CN_ERR_ARG; }
    if (K > 0x7fffffffLL || N > 0x7fffffffLL || tiles_k_of(K) * ((N + 63) / 64) > 0x7fffffffLL) {
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
    const QuantArgs g{K, N, ldw, tiles_k_of(K), tiles_n_of(N), group};
    const dim3 grid((unsigned)(g.tiles_k * ((N + 63) / 64)));
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        if (zeros) hipLaunchKernelGGL((quantize_kernel<T, true>), grid, dim3(256), 0, (hipStream_t)stream, g, (const T *)W, (u32x4 *)codes, scales, zeros);
        else       hipLaunchKernelGGL((quantize_kernel<T, false>), grid, dim3(256), 0, (hipStream_t)stream, g, (const T *)W, (u32x4 *)codes, scales, zeros);
    };
    if (dtype == CN_F32) go(0.0f); else if (dtype == CN_F16) go((f16_t)0); else go((bf16_t)0);
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
    const QuantArgs g{K, N, ldo, tiles_k_of(K), tiles_n_of(N), group};
    const dim3 grid((unsigned)(g.tiles_k * ((N + 63) / 64)));
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        if (zeros) hipLaunchKernelGGL((dequantize_kernel<T, true>), grid, dim3(256), 0, (hipStream_t)stream, g, (const u32x4 *)codes, scales, zeros, (T *)out);
        else       hipLaunchKernelGGL((dequantize_kernel<T, false>), grid, dim3(256), 0, (hipStream_t)stream, g, (const u32x4 *)codes, scales, zeros, (T *)out);
    };
    if (dtype == CN_F32) go(0.0f); else if (dtype == CN_F16) go((f16_t)0); else go((bf16_t)0);
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
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    GemmW4Args g{};
    g.a = A; g.codes = (const u32x4 *)codes; g.scales = scales; g.zeros = zeros; g.out = out;
    g.M = M; g.N = N; g.K = K; g.lda = lda; g.ldo = ldo;
    g.tiles_k = (int)tiles_k_of(K); g.tiles_n = (int)tiles_n_of(N);
    g.group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
    g.vec_a = aligned_to(A, 16) && lda % (16 / (int64_t)dtype_bytes(dtype)) == 0;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == CN_F32) return run_gemm<float>(g, ctx->device, st);
    if (dtype == CN_F16) return run_gemm<f16_t>(g, ctx->device, st);
    return run_gemm<bf16_t>(g, ctx->device, st);
}

}  // extern "C"
