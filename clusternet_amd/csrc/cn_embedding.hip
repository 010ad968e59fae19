// Rows of a table by token number, and the gradient of that lookup, gfx950.  The reference gathers and scatters the
// vocabulary of its window language model with one atomic per element (kConstructVocabMatrix, kUpdateVocabWithGradient,
// source/clusterKernels.cu:1497-1712); here the gradient's sums run over sorted tokens, so they do not depend on scheduling.
//
// Lookup      out[t] = round(scale * E[tok[t]]).  Bound by memory: every row read once, every output written once.  16 bytes an
//             access where the width, both leading dimensions and both addresses are multiples of that; one element an access
//             otherwise, which 16-bit rows feel most (65536 tokens: 120 fp32 columns 9.6 us, 121 17.5; 2048 bf16 columns 61, 2047
//             327; the whole gradient of 2048 285, of 2047 795).
//
// Gradient    dE[v] = scale * sum over {t : tok[t] = v} of dY[t], in fp32.
//   Up to kDirectItems positions and rows that are not wide: see grad_direct_kernel.  Otherwise:
//   1. The positions are sorted by token, stably, by a radix sort of my own digits: ceil(log2(rows + 1)) bits in as many
//      passes as digits of at most kMaxDigit bits need (two for a table of up to 2^18 rows).  A token outside the table
//      takes the key `rows` and so comes last.  Up to kSmallItems positions one workgroup does all passes in LDS; beyond,
//      a pass is three launches (count digits per block, prefix sums per digit over the blocks, scatter).
//   2. The sorted list is cut into chunks of equal length, so a token that makes up a large share of the text costs no more
//      than any other.  A group of lanes walks its chunk, adds the rows of dY in sorted order and writes each run of one
//      token as it ends.  A run that crosses a chunk's border leaves its part in the workspace instead.
//   3. The parts of such runs are added in chunk order and written.
//   Rows that no token names are filled with zeros by further workgroups of step 2, each finding out by a binary search in
//   the sorted list (unless the gradient is added to what is there).
//   Bound by memory: dY read once, dE written once.
#include "cn_dtypes.h"

namespace cn {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kSmallRounds = 8;                               // items per lane of the sort in one workgroup, at most
constexpr int kSmallItems = kSortThreads * kSmallRounds;      // 8192
// Of the sort over many workgroups: a lane's items are ranked one after the other, so few of them and more workgroups (eight
// a lane and 8 workgroups for 65536 tokens: 15 us a scatter).
constexpr int kManyRounds = 2;
constexpr int kManyItems = kSortThreads * kManyRounds;
constexpr int kMaxDigit = 9;                                  // bits of a digit
constexpr int kMaxBins = 1 << kMaxDigit;

// ---- lookup -----------------------------------------------------------------------------------------------------------
constexpr int kRowsAhead = 4;  // rows of a lane in flight

template <typename T, typename I, int VEC>
__global__ __launch_bounds__(256) void embedding_kernel(const T *__restrict__ table, int64_t rows, int64_t cols, int64_t ld,
                                                        const I *__restrict__ tokens, int64_t count, float scale,
                                                        T *__restrict__ out, int64_t ldo, int lanes) {
    const int per = 256 / lanes, sub = threadIdx.x / lanes, lane = threadIdx.x - sub * lanes;
    const int64_t col = ((int64_t)blockIdx.y * lanes + lane) * VEC;
    if (col >= cols) return;
    const int64_t first = (int64_t)blockIdx.x * per * kRowsAhead + sub;
    float v[kRowsAhead][VEC];
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) {
        const int64_t t = first + (int64_t)j * per;
        const int64_t row = t < count ? (int64_t)tokens[t] : -1;
        if (row >= 0 && row < rows) {
            load_f32<VEC>(table + row * ld + col, v[j]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) {
        const int64_t t = first + (int64_t)j * per;
        if (t >= count) continue;
        const int64_t row = (int64_t)tokens[t];
        if (row >= 0 && row < rows) {  // a scale that is not finite leaves the zeros of unnamed rows alone
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] *= scale;
        }
        // past the caches, which then hold the table's frequent rows (65536 x 2048 bf16: 59 us instead of 91)
        store_f32<VEC, true>(out + t * ldo + col, v[j]);
    }
}

// ---- sorting ------------------------------------------------------------------------------------------------------------
// Lanes of the wavefront whose digit equals this lane's (inactive lanes carry a digit of their own class: `live` false).
__device__ __forceinline__ uint64_t lanes_alike(uint32_t digit, int bits, bool live) {
    uint64_t mask = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1u);
        mask &= ((digit >> b) & 1u) ? set : ~set;
    }
    return mask;
}

// Ranks the workgroup's items stably by digit.  In: digit[r] of item (wave * R + r) * 64 + lane (live[r]: it exists).
// Out: rank[r] = number of the workgroup's items of the same digit that come before it; counts[w][d] = exclusive prefix over
// the wavefronts, totals[d] = the workgroup's items of digit d.
template <int R>
__device__ __forceinline__ void rank_items(const uint32_t (&digit)[R], const bool (&live)[R], int bits,
                                           uint32_t (*counts)[kMaxBins], uint32_t *totals, uint32_t (&rank)[R]) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, bins = 1 << bits;
    for (int i = tid; i < kSortWaves * kMaxBins; i += kSortThreads) (&counts[0][0])[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t alike = lanes_alike(digit[r], bits, live[r]);
        uint32_t before = 0u;
        if (live[r]) before = counts[wave][digit[r]];
        __builtin_amdgcn_wave_barrier();  // every lane has read before the first of its digit writes
        const int ahead = __popcll(alike & ((1ull << lane) - 1ull));
        if (live[r] && ahead == 0) counts[wave][digit[r]] = before + (uint32_t)__popcll(alike);
        __builtin_amdgcn_wave_barrier();
        rank[r] = before + (uint32_t)ahead;
    }
    __syncthreads();
    for (int d = tid; d < bins; d += kSortThreads) {
        uint32_t sum = 0u;
        for (int w = 0; w < kSortWaves; ++w) {
            const uint32_t c = counts[w][d];
            counts[w][d] = sum;
            sum += c;
        }
        totals[d] = sum;
    }
    __syncthreads();
}

// In place: v[0 .. bins) becomes its exclusive prefix sums.  bins <= kMaxBins <= kSortThreads; scratch: kSortWaves words.
__device__ __forceinline__ void exclusive_scan(uint32_t *v, int bins, uint32_t *scratch) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const uint32_t mine = tid < bins ? v[tid] : 0u;
    uint32_t sum = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)sum, off, 64);
        if (lane >= off) sum += o;
    }
    if (lane == 63) scratch[wave] = sum;
    __syncthreads();
    uint32_t base = 0u;
    for (int w = 0; w < wave; ++w) base += scratch[w];
    if (tid < bins) v[tid] = base + sum - mine;
    __syncthreads();
}

template <typename I>
__device__ __forceinline__ uint32_t key_of(const I *tokens, int64_t i, int64_t rows) {
    const int64_t t = (int64_t)tokens[i];
    return (uint32_t)(t >= 0 && t < rows ? t : rows);
}

// All passes for up to R * kSortThreads positions in one workgroup.
template <typename I, int R>
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(const I *__restrict__ tokens, int count, int64_t rows,
                                                                  int passes, int bits, uint32_t *__restrict__ keys,
                                                                  uint32_t *__restrict__ positions) {
    __shared__ uint32_t key[R * kSortThreads];
    __shared__ uint16_t order[R * kSortThreads];
    __shared__ uint32_t counts[kSortWaves][kMaxBins];
    __shared__ uint32_t totals[kMaxBins];
    __shared__ uint32_t scratch[kSortWaves];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int i = tid; i < count; i += kSortThreads) {
        key[i] = key_of(tokens, i, rows);
        order[i] = (uint16_t)i;
    }
    __syncthreads();
    for (int p = 0; p < passes; ++p) {
        uint32_t digit[R], rank[R];
        uint16_t item[R];
        bool live[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = (wave * R + r) * 64 + lane;
            live[r] = i < count;
            item[r] = live[r] ? order[i] : (uint16_t)0;
            digit[r] = live[r] ? (key[item[r]] >> (p * bits)) & ((1u << bits) - 1u) : 0u;
        }
        rank_items(digit, live, bits, counts, totals, rank);
        exclusive_scan(totals, 1 << bits, scratch);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (live[r]) order[totals[digit[r]] + counts[wave][digit[r]] + rank[r]] = item[r];
        __syncthreads();
    }
    for (int i = tid; i < count; i += kSortThreads) {
        const int item = order[i];
        keys[i] = key[item];
        positions[i] = (uint32_t)item;
    }
}

// One pass over many positions.  The first pass takes the tokens in order, later ones the lists of the pass before.
template <typename I>
struct SortArgs {
    const I *tokens;  // first pass, else NULL
    const uint32_t *keys_in, *positions_in;
    uint32_t *keys_out, *positions_out;
    uint32_t *counts;  // [bin][blocks]
    uint32_t *totals;  // [bin]
    int64_t count, rows;
    int blocks, shift, bits;
};

template <typename I>
__device__ __forceinline__ uint32_t sort_key(const SortArgs<I> &a, int64_t i) {
    return a.tokens ? key_of(a.tokens, i, a.rows) : a.keys_in[i];
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs<I> a) {
    __shared__ uint32_t bin[kMaxBins];
    const int tid = threadIdx.x, bins = 1 << a.bits;
    for (int d = tid; d < bins; d += kSortThreads) bin[d] = 0u;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kManyRounds; ++r) {
        const int64_t i = (int64_t)blockIdx.x * kManyItems + r * kSortThreads + tid;
        if (i < a.count) atomicAdd(&bin[(sort_key(a, i) >> a.shift) & (uint32_t)(bins - 1)], 1u);  // whole numbers: any order
    }
    __syncthreads();
    for (int d = tid; d < bins; d += kSortThreads) a.counts[(size_t)d * a.blocks + blockIdx.x] = bin[d];
}

// A workgroup per digit: its counts over the blocks become exclusive prefix sums.
__global__ __launch_bounds__(256) void sort_prefix_kernel(uint32_t *counts, uint32_t *totals, int blocks) {
    __shared__ uint32_t scratch[4];
    uint32_t *c = counts + (size_t)blockIdx.x * blocks;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    uint32_t carry = 0u;
    for (int base = 0; base < blocks; base += 256) {
        const uint32_t mine = base + tid < blocks ? c[base + tid] : 0u;
        uint32_t sum = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)sum, off, 64);
            if (lane >= off) sum += o;
        }
        if (lane == 63) scratch[wave] = sum;
        __syncthreads();
        uint32_t before = carry, all = 0u;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) before += scratch[w];
            all += scratch[w];
        }
        if (base + tid < blocks) c[base + tid] = before + sum - mine;
        carry += all;
        __syncthreads();
    }
    if (tid == 0) totals[blockIdx.x] = carry;
}

template <typename I>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs<I> a) {
    __shared__ uint32_t counts[kSortWaves][kMaxBins];
    __shared__ uint32_t totals[kMaxBins];
    __shared__ uint32_t base[kMaxBins];
    __shared__ uint32_t scratch[kSortWaves];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, bins = 1 << a.bits;
    uint32_t key[kManyRounds], position[kManyRounds], digit[kManyRounds], rank[kManyRounds];
    bool live[kManyRounds];
#pragma unroll
    for (int r = 0; r < kManyRounds; ++r) {
        const int64_t i = (int64_t)blockIdx.x * kManyItems + wave * (64 * kManyRounds) + r * 64 + lane;
        live[r] = i < a.count;
        key[r] = live[r] ? sort_key(a, i) : 0u;
        position[r] = live[r] ? (a.tokens ? (uint32_t)i : a.positions_in[i]) : 0u;
        digit[r] = (key[r] >> a.shift) & (uint32_t)(bins - 1);
    }
    if (tid < bins) base[tid] = a.totals[tid];
    __syncthreads();
    exclusive_scan(base, bins, scratch);
    if (tid < bins) base[tid] += a.counts[(size_t)tid * a.blocks + blockIdx.x];
    rank_items(digit, live, a.bits, counts, totals, rank);
#pragma unroll
    for (int r = 0; r < kManyRounds; ++r)
        if (live[r]) {
            const uint32_t to = base[digit[r]] + counts[wave][digit[r]] + rank[r];
            a.keys_out[to] = key[r];
            a.positions_out[to] = position[r];
        }
}

// ---- sums over runs of one token --------------------------------------------------------------------------------------
constexpr int kAhead = 4;      // rows of dY in flight per lane (eight: 270 us instead of 245 for 65536 x 2048, fewer wavefronts fit)
constexpr int kZeroRows = 32;  // rows of dE per zero-filling workgroup

struct GradArgs {
    const uint32_t *keys, *positions;
    float *parts;  // [chunks][2][cols]: the part of a run that came in from the chunk before, the part of one that goes on
    int64_t count, rows, cols, ldy, lde;
    int64_t chunks, chunk_blocks;
    int chunk;  // positions per chunk
    int lanes;  // lanes that share a row of dE, one slab of columns
    float scale;
    int accumulate;
};

template <int VEC, typename E>
__device__ __forceinline__ void finish_row(E *at, const float (&sum)[VEC], float scale, bool accumulate) {
    float v[VEC];
    if (accumulate) {
        load_f32<VEC>(at, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = v[e] + scale * sum[e];
        store_f32<VEC>(at, v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = scale * sum[e];
        store_f32<VEC, true>(at, v);
    }
}

// Zeros for the rows of dE from row0 on that are not named: this workgroup's slab of columns, 16 bytes a lane (one element where
// rows are not made of whole vectors).
template <typename E, int VEC>
__device__ __forceinline__ void fill_unnamed(const GradArgs &a, const uint8_t *named, int64_t row0, E *__restrict__ de) {
    constexpr int kPiece = VEC == 1 ? 1 : 16 / (int)sizeof(E);
    const float zero[kPiece] = {};
    const int64_t slab = (int64_t)blockIdx.y * a.lanes * VEC;
    const int64_t width = a.cols - slab < (int64_t)a.lanes * VEC ? a.cols - slab : (int64_t)a.lanes * VEC;
    const int pieces = (int)(width / kPiece);
    const int per = pieces >= 256 ? 1 : 256 / pieces, sub = threadIdx.x / pieces < per ? threadIdx.x / pieces : -1;
    for (int r = pieces >= 256 ? 0 : sub; r >= 0 && r < kZeroRows; r += per)
        if (!named[r])
            for (int x = pieces >= 256 ? threadIdx.x : threadIdx.x - sub * pieces; x < pieces; x += 256)
                store_f32<kPiece, true>(de + (row0 + r) * a.lde + slab + (int64_t)x * kPiece, zero);
}

// UNIFORM: a wavefront's lanes share their chunk (64 lanes and more a row), so that keys and positions are scalar loads.
template <typename T, typename E, int VEC, bool UNIFORM>
__global__ __launch_bounds__(256) void grad_chunks_kernel(GradArgs a, const T *__restrict__ dy, E *__restrict__ de) {
    if ((int64_t)blockIdx.x >= a.chunk_blocks) {  // zeros for the rows that no token names
        __shared__ uint8_t named[kZeroRows];
        const int64_t row0 = ((int64_t)blockIdx.x - a.chunk_blocks) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const int64_t row = row0 + threadIdx.x;
            int64_t lo = 0, hi = a.count;  // first sorted place whose key is not below row
            while (lo < hi) {
                const int64_t mid = (lo + hi) >> 1;
                if ((int64_t)a.keys[mid] < row) lo = mid + 1; else hi = mid;
            }
            named[threadIdx.x] = row >= a.rows || (lo < a.count && (int64_t)a.keys[lo] == row);
        }
        __syncthreads();
        fill_unnamed<E, VEC>(a, named, row0, de);
        return;
    }
    const int per = 256 / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x - sub * a.lanes;
    int64_t chunk = (int64_t)blockIdx.x * per + sub;
    if (UNIFORM) chunk = __builtin_amdgcn_readfirstlane((int)chunk);
    const int64_t col = ((int64_t)blockIdx.y * a.lanes + lane) * VEC;
    if (chunk >= a.chunks || col >= a.cols) return;
    const int64_t first = chunk * a.chunk;
    const int64_t end = first + a.chunk < a.count ? first + a.chunk : a.count;
    const uint32_t none = (uint32_t)a.rows;

    uint32_t run = a.keys[first];
    bool came_in = first > 0 && a.keys[first - 1] == run;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
    auto close = [&](bool goes_on) {
        if (run == none) return;
        if (came_in || goes_on) {
            float *p = a.parts + (size_t)(chunk * 2 + (came_in ? 0 : 1)) * a.cols + col;
            store_f32<VEC>(p, sum);
        } else {
            finish_row<VEC>(de + (int64_t)run * a.lde + col, sum, a.scale, a.accumulate != 0);
        }
    };
    for (int64_t i = first; i < end; i += kAhead) {
        uint32_t key[kAhead];
        float v[kAhead][VEC];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int64_t at = i + j < end ? i + j : end - 1;
            key[j] = a.keys[at];
            const uint32_t row = a.positions[at];
            if (key[j] != none) {
                load_f32<VEC>(dy + (int64_t)row * a.ldy + col, v[j]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] = 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (i + j >= end) break;
            if (key[j] != run) {
                close(false);
                run = key[j];
                came_in = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += v[j][e];
        }
    }
    close(end < a.count && a.keys[end] == run);
}

// Few positions and rows that are not wide, in one launch and without sorting: workgroup t compares token t with all others.  If
// an earlier one is the same it ends; else it has its list of positions, in order, from the ballots, its groups of lanes add
// every per-th of them, and the groups' sums are added in order.  At most 32 lanes a row, so that per is 8 or more: even if all
// positions name one row, no more than 256 are added one after the other, kDirectAhead in flight.  (128 windows of 11 words x
// 120, fp32: 7.6 us, 19.9 by sorting; 2048 positions 8 and 21, all of them the same row 28.5 and 23.3.)  Every slab of
// columns compares anew: two at most where 16 bytes a lane are taken (four: 2048 x 1024 bf16 in 17 us, by sorting in 20, all the
// same row in 65 and 25).  Rows of up to 256 elements always go this way, so that such calls need no workspace, even where they are
// not made of whole vectors and a lane takes one element: up to eight slabs then (2048 x 65 fp32 12 us, all the same row 31;
// x 129 17 and 34; x 255 24 and 39, where 257 columns are sorted in 20 and 24: a few microseconds at the far end, not worth a
// second contract for the workspace).  Wider rows go this way where 16 bytes a lane cover them in two slabs.
constexpr int kDirectItems = 2048, kDirectLanes = 32, kDirectSlabs = 2, kDirectAhead = 8;

template <typename T, typename E, typename I, int VEC>
__global__ __launch_bounds__(256) void grad_direct_kernel(GradArgs a, const I *__restrict__ tokens, const T *__restrict__ dy,
                                                          E *__restrict__ de) {
    __shared__ uint64_t words[kDirectItems / 64];
    __shared__ uint16_t list[kDirectItems];
    __shared__ float partial[256 * VEC];
    __shared__ uint8_t named[kZeroRows];
    const int n = (int)a.count, wave = threadIdx.x >> 6, lane64 = threadIdx.x & 63;
    if ((int)blockIdx.x >= n) {  // zeros for the rows that no token names
        const int64_t row0 = (int64_t)((int)blockIdx.x - n) * kZeroRows;
        if (threadIdx.x < kZeroRows) named[threadIdx.x] = row0 + threadIdx.x >= a.rows;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += 256) {
            const int64_t row = (int64_t)tokens[j];
            if (row >= row0 && row < row0 + kZeroRows) named[row - row0] = 1;
        }
        __syncthreads();
        fill_unnamed<E, VEC>(a, named, row0, de);
        return;
    }
    const int t = (int)blockIdx.x;
    const int64_t token = (int64_t)tokens[t];
    if (token < 0 || token >= a.rows) return;
    constexpr int kScans = kDirectItems / 256;
    I other[kScans];
#pragma unroll
    for (int i = 0; i < kScans; ++i) {
        const int j = (i * 4 + wave) * 64 + lane64;
        other[i] = tokens[j < n ? j : n - 1];
    }
#pragma unroll
    for (int i = 0; i < kScans; ++i) {
        const int w = i * 4 + wave;
        const uint64_t same = __ballot(w * 64 + lane64 < n && (int64_t)other[i] == token);
        if (lane64 == 0) words[w] = same;
    }
    __syncthreads();
    // every wavefront by itself; a lane has a word
    uint64_t mine = lane64 < kDirectItems / 64 ? words[lane64] : 0u;
    const uint64_t earlier = lane64 < t / 64 ? mine : lane64 == t / 64 ? mine & (((uint64_t)1 << (t & 63)) - 1) : 0u;
    if (__ballot(earlier != 0)) return;  // the first of them does it
    int upto = __popcll(mine);
    for (int off = 1; off < 64; off <<= 1) {
        const int before = __shfl_up(upto, off, 64);
        if (lane64 >= off) upto += before;
    }
    const int matches = __shfl(upto, 63, 64);
    if (wave == 0) {
        int at = upto - __popcll(mine);
        for (; mine; mine &= mine - 1) list[at++] = (uint16_t)(lane64 * 64 + __builtin_ctzll(mine));
    }
    __syncthreads();

    const int per = 256 / a.lanes, sub = threadIdx.x / a.lanes, lane = threadIdx.x - sub * a.lanes;
    const int64_t col = ((int64_t)blockIdx.y * a.lanes + lane) * VEC;
    const bool in = col < a.cols;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
    if (in) {
        for (int r = sub; r < matches; r += per * kDirectAhead) {
            float v[kDirectAhead][VEC];
#pragma unroll
            for (int j = 0; j < kDirectAhead; ++j)
                if (r + j * per < matches) load_f32<VEC>(dy + (int64_t)list[r + j * per] * a.ldy + col, v[j]);
#pragma unroll
            for (int j = 0; j < kDirectAhead; ++j)
                if (r + j * per < matches) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) sum[e] += v[j][e];
                }
        }
    }
    const int groups = matches < per ? matches : per;
    if (groups > 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) partial[e * 256 + threadIdx.x] = sum[e];
        __syncthreads();
        if (sub == 0)
            for (int g = 1; g < groups; ++g)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] += partial[e * 256 + g * a.lanes + lane];
    }
    if (sub == 0 && in) finish_row<VEC>(de + token * a.lde + col, sum, a.scale, a.accumulate != 0);
}

// The runs that cross chunk borders.  Workgroup c takes the run that begins in chunk c and goes on into the next, if there is
// one: its wavefronts add every fourth part, and the four sums are added in order.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void grad_join_kernel(GradArgs a, E *__restrict__ de) {
    __shared__ float partial[4][64][VEC];
    const int64_t chunk = blockIdx.x, first = chunk * a.chunk, end = first + a.chunk;
    if (end >= a.count) return;
    const uint32_t run = a.keys[end - 1];
    if (run == (uint32_t)a.rows || a.keys[end] != run) return;
    if (a.keys[first] == run && first > 0 && a.keys[first - 1] == run) return;  // began before this chunk
    // the chunks behind this one that begin with the run: first chunk that does not, by binary search
    int64_t lo = chunk + 1, hi = a.chunks;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (a.keys[mid * a.chunk] == run) lo = mid + 1; else hi = mid;
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t col = ((int64_t)blockIdx.y * 64 + lane) * VEC;
    const bool in = col < a.cols;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
    if (in) {
#pragma unroll 4
        for (int64_t j = chunk + wave; j < lo; j += 4) {
            float v[VEC];
            load_f32<VEC>(a.parts + (size_t)(j * 2 + (j == chunk ? 1 : 0)) * a.cols + col, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) partial[wave][lane][e] = sum[e];
    __syncthreads();
    if (wave == 0 && in) {
#pragma unroll
        for (int w = 1; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += partial[w][lane][e];
        finish_row<VEC>(de + (int64_t)run * a.lde + col, sum, a.scale, a.accumulate != 0);
    }
}

// Lanes per row: a power of two that covers the row, at most a workgroup.
int lanes_for(int64_t cols, int vec) {
    int lanes = 16;
    while (lanes < 256 && (int64_t)lanes * vec < cols) lanes *= 2;
    return lanes;
}

// Positions per chunk: short ones for few positions (a chunk's rows are read one batch after the other), longer ones (fewer parts
// to store and join) where 256 K lanes are busy all the same: 64 at 65536 x 2048 (32: the join takes 13.5 us instead of 8),
// 16 at 262144 x 120 (256, as for wide rows: 219 us in all instead of 97).
int chunk_for(int64_t count, int64_t cols) {
    int c = 8;
    while (c < 256 && (int64_t)c * (256 * 1024) < count * lanes_for(cols, 8)) c *= 2;
    return c;
}

struct GradPlan {
    int passes, bits, blocks, chunk;
    int64_t chunks;
};
GradPlan plan_grad(int64_t count, int64_t rows, int64_t cols) {
    GradPlan p;
    int total = 1;
    while (total < 32 && (rows >> total) != 0) ++total;  // bits of the largest key, `rows`
    p.passes = (total + kMaxDigit - 1) / kMaxDigit;
    p.bits = (total + p.passes - 1) / p.passes;
    p.blocks = count <= kSmallItems ? 1 : (int)((count + kManyItems - 1) / kManyItems);
    p.chunk = chunk_for(count, cols);
    p.chunks = (count + p.chunk - 1) / p.chunk;
    return p;
}

// Whatever the type and the alignment: such calls need no workspace.
bool never_sorted(int64_t count, int64_t cols) { return count > 0 && count <= kDirectItems && cols <= kDirectSlabs * kDirectLanes * 4; }

struct GradSpace {
    uint32_t *keys[2], *positions[2], *counts, *totals;
    float *parts;
    size_t bytes;
};
GradSpace lay_out(void *workspace, const GradPlan &p, int64_t count, int64_t cols) {
    Carver c(workspace);
    GradSpace s;
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = c.take<uint32_t>((size_t)count);
        s.positions[i] = c.take<uint32_t>((size_t)count);
    }
    s.counts = c.take<uint32_t>((size_t)p.blocks << p.bits);
    s.totals = c.take<uint32_t>((size_t)kMaxBins);
    s.parts = c.take<float>((size_t)p.chunks * 2 * (size_t)cols);
    s.bytes = c.used;
    return s;
}

template <typename I>
cn_status sort_tokens(const I *tokens, int64_t count, int64_t rows, const GradPlan &p, GradSpace &s, int *sorted, hipStream_t st) {
    if (p.blocks <= 1) {
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(1), dim3(kSortThreads), 0, st, tokens, (int)count, rows, p.passes, p.bits, s.keys[0], s.positions[0]);
        };
        if (count <= kSortThreads) go(sort_small_kernel<I, 1>);
        else if (count <= 2 * kSortThreads) go(sort_small_kernel<I, 2>);
        else if (count <= 4 * kSortThreads) go(sort_small_kernel<I, 4>);
        else go(sort_small_kernel<I, kSmallRounds>);
        CN_HIP(hipGetLastError());
        *sorted = 0;
        return CN_OK;
    }
    for (int pass = 0; pass < p.passes; ++pass) {
        const int to = pass & 1, from = to ^ 1;
        SortArgs<I> a{pass == 0 ? tokens : nullptr, s.keys[from], s.positions[from], s.keys[to], s.positions[to],
                      s.counts, s.totals, count, rows, p.blocks, pass * p.bits, p.bits};
        hipLaunchKernelGGL((sort_count_kernel<I>), dim3(p.blocks), dim3(kSortThreads), 0, st, a);
        hipLaunchKernelGGL(sort_prefix_kernel, dim3(1 << p.bits), dim3(256), 0, st, s.counts, s.totals, p.blocks);
        hipLaunchKernelGGL((sort_scatter_kernel<I>), dim3(p.blocks), dim3(kSortThreads), 0, st, a);
        CN_HIP(hipGetLastError());
        *sorted = to;
    }
    return CN_OK;
}

template <typename T, typename E, int VEC>
cn_status run_grad(GradArgs a, const void *tokens, int token_bits, bool direct, const void *dy, void *de, hipStream_t st) {
    a.lanes = lanes_for(a.cols, VEC);
    if (direct && a.lanes > kDirectLanes) a.lanes = kDirectLanes;
    const int64_t slabs = (a.cols + (int64_t)a.lanes * VEC - 1) / ((int64_t)a.lanes * VEC);
    const int per = 256 / a.lanes;
    a.chunk_blocks = (a.chunks + per - 1) / per;
    const int64_t zero_blocks = a.accumulate ? 0 : (a.rows + kZeroRows - 1) / kZeroRows;
    const int64_t join_slabs = (a.cols + 64 * VEC - 1) / (64 * VEC);
    if (a.chunk_blocks + zero_blocks == 0) return CN_OK;
    if (direct) {
        const dim3 grid((unsigned)(a.count + zero_blocks), (unsigned)slabs);
        if (token_bits == 32)
            hipLaunchKernelGGL((grad_direct_kernel<T, E, int32_t, VEC>), grid, dim3(256), 0, st, a, (const int32_t *)tokens, (const T *)dy, (E *)de);
        else
            hipLaunchKernelGGL((grad_direct_kernel<T, E, int64_t, VEC>), grid, dim3(256), 0, st, a, (const int64_t *)tokens, (const T *)dy, (E *)de);
        CN_HIP(hipGetLastError());
        return CN_OK;
    }
    const dim3 grid((unsigned)(a.chunk_blocks + zero_blocks), (unsigned)slabs);
    if (a.lanes >= 64)
        hipLaunchKernelGGL((grad_chunks_kernel<T, E, VEC, true>), grid, dim3(256), 0, st, a, (const T *)dy, (E *)de);
    else
        hipLaunchKernelGGL((grad_chunks_kernel<T, E, VEC, false>), grid, dim3(256), 0, st, a, (const T *)dy, (E *)de);
    if (a.chunks > 1)
        hipLaunchKernelGGL((grad_join_kernel<E, VEC>), dim3((unsigned)(a.chunks - 1), (unsigned)join_slabs), dim3(256), 0, st, a, (E *)de);
    CN_HIP(hipGetLastError());
    return CN_OK;
}

template <typename T, int VEC>
cn_status run_lookup(const void *table, int64_t rows, int64_t cols, int64_t ld, const void *tokens, int bits, int64_t count,
                     float scale, void *out, int64_t ldo, hipStream_t st) {
    const int lanes = lanes_for(cols, VEC);
    const int64_t per = (int64_t)(256 / lanes) * kRowsAhead;
    const int64_t blocks = (count + per - 1) / per, slabs = (cols + (int64_t)lanes * VEC - 1) / ((int64_t)lanes * VEC);
    const dim3 grid((unsigned)blocks, (unsigned)slabs);
    if (bits == 32)
        hipLaunchKernelGGL((embedding_kernel<T, int32_t, VEC>), grid, dim3(256), 0, st, (const T *)table, rows, cols, ld,
                           (const int32_t *)tokens, count, scale, (T *)out, ldo, lanes);
    else
        hipLaunchKernelGGL((embedding_kernel<T, int64_t, VEC>), grid, dim3(256), 0, st, (const T *)table, rows, cols, ld,
                           (const int64_t *)tokens, count, scale, (T *)out, ldo, lanes);
    CN_HIP(hipGetLastError());
    return CN_OK;
}

cn_status check_tokens(const char *what, int64_t rows, int64_t cols, int64_t ld, int token_bits, int64_t count) {
    if (rows < 0 || cols < 0 || count < 0) { set_error("%s: negative dimension", what); return CN_ERR_SHAPE; }
    if (ld < cols) { set_error("%s: leading dimension too small", what); return CN_ERR_SHAPE; }
    if (token_bits != 32 && token_bits != 64) { set_error("%s: tokens have 32 or 64 bits", what); return CN_ERR_ARG; }
    if (rows > 0x7fffffffLL || count > 0x7fffffffLL) { set_error("%s: more than 2^31 - 1 rows or tokens", what); return CN_ERR_SHAPE; }
    return CN_OK;
}

}  // namespace

}  // namespace cn

using namespace cn;

extern "C" {

cn_status cn_embedding(const void *table, int dtype, int64_t rows, int64_t cols, int64_t ld, const void *tokens, int token_bits,
                       int64_t count, float scale, void *out, int64_t ldo, void *stream) {
    if (!known_dtype(dtype)) { set_error("embedding: unknown element type %d", dtype); return CN_ERR_ARG; }
    cn_status s = check_tokens("embedding", rows, cols, ld, token_bits, count);
    if (s != CN_OK) return s;
    if (ldo < cols) { set_error("embedding: leading dimension too small"); return CN_ERR_SHAPE; }
    if (count == 0 || cols == 0) return CN_OK;
    if ((rows > 0 && !table) || !tokens || !out) { set_error("embedding: NULL pointer"); return CN_ERR_NULL; }
    if (table == out) { set_error("embedding: the output is the table"); return CN_ERR_ARG; }
    const int64_t vec = 16 / (int64_t)dtype_bytes(dtype);
    const bool wide = cols % vec == 0 && ld % vec == 0 && ldo % vec == 0 && aligned_to(table, 16) && aligned_to(out, 16);
    const int64_t lanes = lanes_for(cols, wide ? vec : 1), per = 256 / lanes * kRowsAhead;
    if (!launchable((count + per - 1) / per, 256, cols / (lanes * (wide ? vec : 1)) + 1)) {
        set_error("embedding: too many tokens or columns for one launch");
        return CN_ERR_SHAPE;
    }
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto zero) -> cn_status {
        typedef decltype(zero) T;
        constexpr int kWide = 16 / (int)sizeof(T);
        return wide ? run_lookup<T, kWide>(table, rows, cols, ld, tokens, token_bits, count, scale, out, ldo, st)
                    : run_lookup<T, 1>(table, rows, cols, ld, tokens, token_bits, count, scale, out, ldo, st);
    };
    return dtype == CN_F32 ? go(0.0f) : dtype == CN_F16 ? go((f16_t)0) : go((bf16_t)0);
}

size_t cn_embedding_grad_workspace_bytes(int64_t count, int64_t rows, int64_t cols) {
    if (count <= 0 || rows < 0 || cols <= 0 || count > 0x7fffffffLL || rows > 0x7fffffffLL) return 0;
    return never_sorted(count, cols) ? 0 : lay_out(nullptr, plan_grad(count, rows, cols), count, cols).bytes;
}

cn_status cn_embedding_grad(const void *dy, int dy_dtype, int64_t ldy, const void *tokens, int token_bits, int64_t count,
                            int64_t rows, int64_t cols, float scale, int accumulate, void *de, int de_dtype, int64_t lde,
                            void *workspace, size_t workspace_bytes, void *stream) {
    if (!known_dtype(dy_dtype) || (de_dtype != CN_F32 && de_dtype != dy_dtype)) {
        set_error("embedding_grad: the gradient is fp32 or of the errors' type (got %d for %d)", de_dtype, dy_dtype);
        return CN_ERR_ARG;
    }
    cn_status s = check_tokens("embedding_grad", rows, cols, lde, token_bits, count);
    if (s != CN_OK) return s;
    if (ldy < cols) { set_error("embedding_grad: leading dimension too small"); return CN_ERR_SHAPE; }
    if (rows == 0 || cols == 0 || (accumulate && count == 0)) return CN_OK;
    const size_t needed = cn_embedding_grad_workspace_bytes(count, rows, cols);
    if (!de || (count > 0 && (!dy || !tokens)) || (needed > 0 && !workspace)) { set_error("embedding_grad: NULL pointer"); return CN_ERR_NULL; }
    if (workspace_bytes < needed) {
        set_error("embedding_grad: workspace of %zu bytes, %zu needed", workspace_bytes, needed);
        return CN_ERR_WORKSPACE;
    }
    if (needed > 0 && !aligned_to(workspace, 256)) { set_error("embedding_grad: the workspace is not aligned to 256 bytes"); return CN_ERR_ARG; }
    if (count > 0 && de == dy) { set_error("embedding_grad: the gradient is the errors"); return CN_ERR_ARG; }
    const GradPlan p = plan_grad(count, rows, cols);
    const int64_t most = (p.chunks < kDirectItems ? kDirectItems : p.chunks) + (accumulate ? 0 : rows / kZeroRows + 1);
    if (!launchable(most, 256, cols / 64 + 1)) {
        set_error("embedding_grad: too many rows or columns for one launch");
        return CN_ERR_SHAPE;
    }
    Context *ctx;
    s = current_context(&ctx);
    if (s != CN_OK) return s;
    hipStream_t st = (hipStream_t)stream;
    GradSpace space = lay_out(workspace, p, count, cols);
    // whole vectors: 16 bytes of dY; the parts and dE hold as many elements
    const int64_t vec = 16 / (int64_t)dtype_bytes(dy_dtype);
    const bool wide = cols % vec == 0 && ldy % vec == 0 && lde % vec == 0 && aligned_to(dy, 16) &&
                      aligned_to(de, (size_t)vec * dtype_bytes(de_dtype));
    const bool direct = never_sorted(count, cols) || (count > 0 && count <= kDirectItems && cols <= kDirectSlabs * kDirectLanes * (wide ? vec : 1));
    int sorted = 0;
    if (count > 0 && !direct) {
        s = token_bits == 32 ? sort_tokens((const int32_t *)tokens, count, rows, p, space, &sorted, st)
                             : sort_tokens((const int64_t *)tokens, count, rows, p, space, &sorted, st);
        if (s != CN_OK) return s;
    }
    GradArgs a{};
    a.keys = space.keys[sorted];
    a.positions = space.positions[sorted];
    a.parts = space.parts;
    a.count = count; a.rows = rows; a.cols = cols; a.ldy = ldy; a.lde = lde;
    a.chunks = p.chunks; a.chunk = p.chunk;
    a.scale = scale; a.accumulate = accumulate != 0;
    auto go = [&](auto in, auto to) -> cn_status {
        typedef decltype(in) T;
        typedef decltype(to) E;
        constexpr int kWide = 16 / (int)sizeof(T);
        return wide ? run_grad<T, E, kWide>(a, tokens, token_bits, direct, dy, de, st)
                    : run_grad<T, E, 1>(a, tokens, token_bits, direct, dy, de, st);
    };
    if (dy_dtype == CN_F32) return go(0.0f, 0.0f);
    if (dy_dtype == CN_F16) return de_dtype == CN_F32 ? go((f16_t)0, 0.0f) : go((f16_t)0, (f16_t)0);
    return de_dtype == CN_F32 ? go((bf16_t)0, 0.0f) : go((bf16_t)0, (bf16_t)0);
}

}  // extern "C"
