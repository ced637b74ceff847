// Token embedding and its gradient:
//     out[i] = scale W[t_i],    dW[v] (+)= scale sum_{i: t_i = v} dout[i].
//
// Bound: HBM -- the looked-up rows and the outputs once; for the gradient dout once and the whole table
// once (twice where it is added to).  A thread of the lookup has four vectors of 16 bytes in flight: 16384 rows of
// 20480 x 640 fp32 take 13.4 us, 6.3 TB/s (they fit the memory-side cache).
//
// The gradient's sums run over each token's positions in an order that sizes and ids fix, not timing: no
// atomics on values.  Three to five launches:
//   sort:  a workgroup owns a range of tokens and lists its positions by token.  Its waves take runs of
//          positions: each counts its tokens, and after a scan over tokens and waves places its positions, in order.
//          Of few positions the workgroup reads all ids (and counts those below the range, which
//          gives where the range's positions begin without asking another workgroup).  Of many, a launch before
//          writes the number of each id's range as a byte and counts them by blocks of positions, and the
//          workgroup picks its positions by comparing 16 bytes at a time.  Of very many, ranges with a large share of
//          them are picked and counted by several workgroups, and placed by a launch behind.
//   sum:   a wave walks a chunk of the sorted positions for up to 64 vectors of columns and writes a
//          token's row where its run ends.  Runs that leave the chunk go to the workspace as fp32 parts.
//          Further waves clear the rows of tokens that do not occur.
//   join:  the parts of such a run: up to 16 in order, more as eight sums of every eighth, which are added in order.
// us of the sort, the sum and the join: 16384 of 20480 x 640 fp32, added, 16, 17.5, 4.7; 262144 of 20480 x 1024 bf16,
// with a token that has 3.7 % of them, 47, 133 (4.4 TB/s of rows in random order) and 10; 4111 of 673 x 333 bf16,
// where each is a chain of latencies, 6.7, 8.8, 4.5.
#include "common.h"

#include <algorithm>

namespace yuf {
namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kUnits = 4;         // vectors of a thread of the lookup
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortRanges = 256;  // workgroups of the sort: one per CU
constexpr int kRangeMost = 960;   // tokens of a range: their counters fill 60 KB of LDS
// Of more than kManyPositions positions the ranges are written down first, where they are at most kNoRange of at
// most kWidthMost tokens each, that is for up to 130560 tokens.  Both forms, us without and with: 4111 of 673 6.7 and 12.0,
// 16384 of 20480 24 and 15.6, of 130560 27 and 16.2; 262144 of 130560 355 and 39.  Without, each range's workgroup reads
// all ids, so that a larger table costs as much, and one of millions of narrow rows more than anything else (16384 of 2^24 x 8 1.6 ms).
constexpr int kManyPositions = 8192;
constexpr int kNoRange = 255, kWidthMost = 512;
constexpr int kBlocksMost = 256, kBlockRun = 1024;  // blocks of positions, and positions that a wave reads at a time
constexpr int kPicks = 4;         // such reads of a wave in flight
constexpr int kHeld = 12288;      // positions of a range that are kept in LDS (96 KB), beside 32 KB of counters
// Of more than kSplitPositions positions, ranges with more than kHeavy of them (or a kHeavyShare-th of all) are shared
// by helpers of half as many each, which costs a launch.  The sort of 187747 of 673, one of them in 44 % of the places:
// 125 us without and 39 with; with even frequencies 22 and 29.  262144 of 20480, the heaviest range 10500: 41.5 and 47, the
// helpers having nothing to do.
constexpr int64_t kSplitPositions = 65536;
constexpr int kHeavy = 16384, kHeavyShare = 64;
constexpr int kBatch = 8;         // rows of a wave in flight
static_assert(kSortWaves * kBatch * kWave >= kManyPositions, "a batch of each wave holds them");
constexpr int kWalks = 5120;      // 20 waves a CU, which run together (4096 of bf16 32 x 8192 x 1024: 140 -> 132 us)
constexpr int kClearRows = 8;     // table rows that a wave looks over for tokens without positions
constexpr int kJoinWaves = 8, kJoinAlone = 16;  // and parts that a wave joins alone
constexpr int kVocabMost = 1 << 24, kColsMost = 1 << 24;

// Vectors with the alignment of their elements: rows of odd widths start anywhere.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8_u __attribute__((ext_vector_type(8), aligned(2)));

template <typename T> struct Vec;
template <> struct Vec<float> { static constexpr int kN = 4; using type = f32x4_u; };
template <> struct Vec<uint16_t> { static constexpr int kN = 8; using type = u16x8_u; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ void narrow(float x, float &out) { out = x; }
__device__ __forceinline__ void narrow(float x, uint16_t &out) {
    // Round to nearest even; NaN stays a (quiet) NaN.
    const uint32_t u = __float_as_uint(x);
    out = x != x ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ int64_t token_at(const void *tokens, bool wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(tokens)[i] : (int64_t)static_cast<const int32_t *>(tokens)[i];
}

// A lane's columns of a row of `cols`: kN from `at` on, of which those from `own` to `end` are its own.  The last
// vector of a row is moved back to end with it (its first columns are its neighbour's), unless the row is
// shorter than a vector.
template <typename T> struct Columns {
    int at, own, end;
    __device__ __forceinline__ Columns(int first, int cols) {
        constexpr int kN = Vec<T>::kN;
        at = max(0, min(first, cols - kN));
        own = min(first, cols) - at;
        end = min(kN, cols - at);
        if (first >= cols) own = end;
    }
    __device__ __forceinline__ bool any() const { return own < end; }
    __device__ __forceinline__ void load(const T *row, typename Vec<T>::type &x) const {
        constexpr int kN = Vec<T>::kN;
        if (end == kN) {
            x = *reinterpret_cast<const typename Vec<T>::type *>(row + at);
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) x[e] = e < end ? row[at + e] : T(0);
        }
    }
    __device__ __forceinline__ void load(const T *row, float (&x)[Vec<T>::kN]) const {
        typename Vec<T>::type v;
        load(row, v);
#pragma unroll
        for (int e = 0; e < Vec<T>::kN; ++e) x[e] = widen(v[e]);
    }
    __device__ __forceinline__ void store(T *row, const float (&x)[Vec<T>::kN]) const {
        constexpr int kN = Vec<T>::kN;
        if (own == 0 && end == kN) {
            typename Vec<T>::type v;
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                T t;
                narrow(x[e], t);
                v[e] = t;
            }
            *reinterpret_cast<typename Vec<T>::type *>(row + at) = v;
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                T t;
                narrow(x[e], t);
                if (e >= own && e < end) row[at + e] = t;
            }
        }
    }
};

// ------------------------------------------------------------------------------ lookup
template <typename T> struct LookupParams {
    int64_t count;  // vectors of the output
    int row_vecs;   // of a row
    int cols, vocab;
    const void *tokens;
    bool wide;
    const T *table;
    float scale;
    T *out;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) embedding_kernel(LookupParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    const int64_t base = (int64_t)blockIdx.x * (kThreads * kUnits);
    const int64_t row0 = base / p.row_vecs;
    const uint32_t rest = (uint32_t)(base - row0 * p.row_vecs) + threadIdx.x;
    float x[kUnits][kN];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t at = rest + u * kThreads, row = at / (uint32_t)p.row_vecs;
        if (base + threadIdx.x + u * kThreads >= p.count) break;
        const int64_t token = token_at(p.tokens, p.wide, row0 + row);
        const Columns<T> c((int)(at - row * p.row_vecs) * kN, p.cols);
        if (token >= 0 && token < p.vocab) {
            c.load(p.table + token * p.cols, x[u]);
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) x[u][e] = NAN;
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const uint32_t at = rest + u * kThreads, row = at / (uint32_t)p.row_vecs;
        if (base + threadIdx.x + u * kThreads >= p.count) break;
        const Columns<T> c((int)(at - row * p.row_vecs) * kN, p.cols);
#pragma unroll
        for (int e = 0; e < kN; ++e) x[u][e] *= p.scale;
        c.store(p.out + (row0 + row) * p.cols, x[u]);
    }
}

template <typename T>
int embedding(int64_t M, int V, int D, const T *table, const void *tokens, int token_bits, double scale, T *out, void *stream) {
    if (M < 0 || V < 0 || D < 0) return fail(YUF_ERR_INVALID, "embedding: negative size");
    if (token_bits != 32 && token_bits != 64) return fail(YUF_ERR_INVALID, "embedding: token_bits must be 32 or 64");
    if (V > kVocabMost || D > kColsMost) return fail(YUF_ERR_INVALID, "embedding: V and D may not exceed 2^24");
    if (M == 0 || D == 0) return YUF_OK;
    if (M >= (int64_t)1 << 31) return fail(YUF_ERR_INVALID, "embedding: 2^31 tokens or more");
    const int row_vecs = ceil_div(D, Vec<T>::kN);
    const int64_t blocks = (M * row_vecs + kThreads * kUnits - 1) / (kThreads * kUnits);
    if (blocks * kThreads >= (int64_t)1 << 32) return fail(YUF_ERR_INVALID, "embedding: too many elements");  // threads of a launch
    if (!tokens || !out || (!table && V > 0)) return fail(YUF_ERR_INVALID, "embedding: null table, tokens or output");
    const size_t row = (size_t)D * sizeof(T);
    if (outputs_overlap<2, 1>({{table, V * row}, {tokens, (size_t)M * (token_bits / 8)}}, {{out, M * row}}))
        return fail(YUF_ERR_INVALID, "embedding: the output may not be the table or the tokens, nor a part of them");
    LookupParams<T> p{};
    p.row_vecs = row_vecs;
    p.count = M * row_vecs;
    p.cols = D; p.vocab = V;
    p.tokens = tokens; p.wide = token_bits == 64;
    p.table = table; p.scale = (float)scale; p.out = out;
    hipLaunchKernelGGL((embedding_kernel<T>), dim3((uint32_t)blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), p);
    YUF_LAUNCH_CHECK("embedding");
    return YUF_OK;
}

// ---------------------------------------------------------------------------- gradient
struct Place {
    int position, token;
};

// Tokens are numbered by their ranges: a range holds `width` numbers, some of the last ones unused.  Of many positions
// range r holds the tokens r + 255 j, so that frequent neighbours fall into different ranges.
struct Numbering {
    int width;
    bool spread;
    __device__ __forceinline__ int number(int token) const { return spread ? token % kNoRange * width + token / kNoRange : token; }
};

struct SortParams {
    int64_t M;
    int vocab, width, bits;  // tokens of a range, bits of an index into it
    int numbers;             // of all ranges
    const void *tokens;
    bool wide;
    int64_t padding;  // or -1
    Place *order;     // [M]
    int *start;       // [numbers + 1]
    // Of many positions:
    int64_t block;    // positions of a block
    int blocks;
    uint8_t *ranges;  // [blocks block]
    int *below;       // [blocks][256]
    Place *picked;    // [M]: a range's positions, if they are more than LDS holds
    int heavy;        // a range with more positions than this is shared by helpers, two for each `heavy` of them
    int helpers;      // the most there can be; 0: no range is shared
    int *shares;      // [helpers][width]: a helper's positions of each token
    int *assigned;    // [helpers][3]: a helper's range (or -1), part and parts
};

// The token of a position, or -1: not to be counted.
__device__ __forceinline__ int counted_token(const SortParams &p, int64_t at) {
    const int64_t t = token_at(p.tokens, p.wide, at);
    return t >= 0 && t < p.vocab && t != p.padding ? (int)t : -1;
}

// Lanes with the same j as this one, among those that are `in`.
__device__ __forceinline__ uint64_t same_lanes(bool in, int j, int bits) {
    uint64_t same = __ballot(in);
    for (int bit = 0; bit < bits; ++bit) {
        const uint64_t set = __ballot(in && (j >> bit & 1));
        same &= j >> bit & 1 ? set : ~set;
    }
    return same;
}

// counts [waves][p.width] of the range's tokens -> where each wave's first position of each token goes, the range's
// positions beginning at `first`; p.start of the range.  The workgroup, between barriers.  Helper `part` of `parts` has its
// counts here and those of all in `shares`.
__device__ __forceinline__ void sort_places(const SortParams &p, int range, int first, int *counts, int *sums,
                                            const int *shares = nullptr, int part = 0, int parts = 1) {
    const int low = range * p.width, width = min(p.width, p.numbers - low);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    for (int base = 0; base < width; base += kSortThreads) {
        const int j = base + threadIdx.x;
        int here = 0, earlier = 0;  // of all helpers, and of those before this one
        int mine[kSortWaves];
        if (j < width)
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) mine[w] = counts[w * p.width + j];
        if (j < width && shares) {
            for (int q = 0; q < parts; ++q) {
                const int n = shares[q * p.width + j];
                here += n;
                if (q < part) earlier += n;
            }
        } else if (j < width) {
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) here += mine[w];
        }
        int upto = here;  // inclusive scan over the workgroup
        for (int step = 1; step < kWave; step *= 2) {
            const int other = __shfl_up(upto, step);
            if (lane >= step) upto += other;
        }
        if (lane == kWave - 1) sums[wave] = upto;
        __syncthreads();
        int before = first, all = 0;
        for (int w = 0; w < kSortWaves; ++w) {
            if (w < wave) before += sums[w];
            all += sums[w];
        }
        int next = before + upto - here;
        if (j < width) {
            if (part == 0) p.start[low + j] = next;
            next += earlier;
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                counts[w * p.width + j] = next;
                next += mine[w];
            }
        }
        first += all;
        __syncthreads();
    }
    if (low + width < p.numbers || part > 0) return;
    if (threadIdx.x == 0) p.start[p.numbers] = first;
    for (int64_t i = first + threadIdx.x; i < p.M; i += kSortThreads) p.order[i] = {0, -1};  // positions that are not counted
}

// Lanes of the same token rank themselves by comparing its bits; `mine`: the wave's places.
__device__ __forceinline__ void sort_place(const SortParams &p, bool in, int j, int token, int position, int *mine) {
    const uint64_t same = same_lanes(in, j, p.bits);
    const int lane = threadIdx.x % kWave;
    if (in) {
        const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
        const int at = mine[j];
        __builtin_amdgcn_wave_barrier();
        p.order[at + rank] = {position, token};
        if (rank == 0) mine[j] = at + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
}

// ONCE: a wave's positions are one batch, whose tokens stay in registers (M <= kManyPositions; 4111 of 673 8.5 -> 6.7 us,
// 8192 of 20480 12.8 -> 11.1).
template <bool ONCE>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(SortParams p) {
    extern __shared__ int counts[];  // [waves][width]
    __shared__ int below[kSortWaves], sums[kSortWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int low = blockIdx.x * p.width, width = min(p.width, p.vocab - low);
    int *mine = counts + wave * p.width;
    for (int i = threadIdx.x; i < kSortWaves * p.width; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    // This wave's run of positions, in whole waves of them.
    const int64_t tiles = (p.M + kWave - 1) / kWave;
    const int64_t first = tiles * wave / kSortWaves * kWave, last = min(p.M, tiles * (wave + 1) / kSortWaves * kWave);
    int t[kBatch];
    const auto read = [&](int64_t from) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t at = from + u * kWave + lane;
            t[u] = at < last ? counted_token(p, at) : -1;
        }
    };
    if (ONCE) read(first);
    int less = 0;
    for (int64_t at = first; at < (ONCE ? first + 1 : last); at += kBatch * kWave) {
        if (!ONCE) read(at);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            less += t[u] >= 0 && t[u] < low;
            if (t[u] >= low && t[u] < low + width) atomicAdd(&mine[t[u] - low], 1);
        }
    }
    for (int step = 1; step < kWave; step *= 2) less += __shfl_xor(less, step);
    if (lane == 0) below[wave] = less;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < kSortWaves; ++w) total += below[w];
    sort_places(p, blockIdx.x, total, counts, sums);
    for (int64_t at = first; at < (ONCE ? first + 1 : last); at += kBatch * kWave) {
        if (!ONCE) read(at);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const bool in = t[u] >= low && t[u] < low + width;
            if (__ballot(in) != 0) sort_place(p, in, t[u] - low, t[u], (int)(at + u * kWave) + lane, mine);
        }
    }
}

// The byte of each position: its range, or 255, of 16 positions e in word e % 4 and byte e / 4; and for each block of
// positions, how many lie in ranges below each.
__global__ void __launch_bounds__(kThreads) embedding_ranges_kernel(SortParams p) {
    __shared__ int counts[kThreads], sums[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    counts[tid] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * p.block;
    for (int64_t at = first + tid * 4; at < first + p.block; at += kThreads * 4) {
        uint8_t *to = p.ranges + at / 16 * 16 + at % 16 / 4;
        int t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = at + e < p.M ? counted_token(p, at + e) : -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int range = t[e] < 0 ? kNoRange : t[e] % kNoRange;
            if (t[e] >= 0) atomicAdd(&counts[range], 1);
            to[e * 4] = (uint8_t)range;
        }
    }
    __syncthreads();
    const int here = counts[tid];
    int upto = here;
    for (int step = 1; step < kWave; step *= 2) {
        const int other = __shfl_up(upto, step);
        if (lane >= step) upto += other;
    }
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += sums[w];
    p.below[blockIdx.x * kThreads + tid] = upto - here;
}

// Where the range's positions begin, and where each block's do among them (offsets, with their number at the end).
__device__ __forceinline__ int range_offsets(const SortParams &p, int range, int *offsets, int *sums, int *bases) {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    int before = 0, here = 0;
    if (tid < p.blocks) {
        before = p.below[tid * kThreads + range];
        here = p.below[tid * kThreads + range + 1] - before;
    }
    int upto = here;
    for (int step = 1; step < kWave; step *= 2) {
        const int other = __shfl_up(upto, step);
        if (lane >= step) upto += other;
        before += __shfl_xor(before, step);
    }
    if (lane == kWave - 1) sums[wave] = upto;
    if (lane == 0) bases[wave] = before;
    __syncthreads();
    int first = 0, n = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        first += bases[w];
        if (w < wave) upto += sums[w];
        n += sums[w];
    }
    if (tid < p.blocks) offsets[tid] = upto - here;
    if (tid == 0) offsets[p.blocks] = n;
    __syncthreads();
    return first;
}

// A wave's blocks' positions of the range, in order, from list[next] on.
__device__ __forceinline__ void pick_positions(const SortParams &p, int range, int block0, int block1, int next, Place *list) {
    const int lane = threadIdx.x % kWave;
    const uint32_t pattern = (uint32_t)range * 0x01010101u;
    for (int64_t at = block0 * p.block; at < block1 * p.block; at += kPicks * kBlockRun) {
        uint4 bytes[kPicks];
#pragma unroll
        for (int u = 0; u < kPicks; ++u)
            bytes[u] = *reinterpret_cast<const uint4 *>(p.ranges + min(at + u * kBlockRun, block1 * p.block - kBlockRun) + lane * 16);
#pragma unroll
        for (int u = 0; u < kPicks; ++u) {
            if (at + u * kBlockRun >= block1 * p.block) break;
            // Bit 8 b + w of match: byte b of word w is the range.  In ascending order they are the positions 4 b + w.
            const uint32_t words[4] = {bytes[u].x, bytes[u].y, bytes[u].z, bytes[u].w};
            uint32_t match = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t x = words[w] ^ pattern;
                match |= (~(((x & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | x) & 0x80808080u) >> (7 - w);
            }
            if (__ballot(match != 0) == 0) continue;
            int upto = __popc(match);
            const int own = upto;
            for (int step = 1; step < kWave; step *= 2) {
                const int other = __shfl_up(upto, step);
                if (lane >= step) upto += other;
            }
            int to = next + upto - own;
            for (; match; match &= match - 1, ++to) {
                const int bit = __ffs(match) - 1;
                list[to].position = (int)(at + u * kBlockRun) + lane * 16 + (bit >> 3) * 4 + (bit & 7);
            }
            next += __builtin_amdgcn_readlane(upto, kWave - 1);
        }
    }
}

// A wave's positions from list[from] to list[end]: their tokens (numbered in the range) are looked up, if LOOK, and counted.
template <bool LOOK>
__device__ __forceinline__ void count_positions(const SortParams &p, Place *list, int from, int end, int *mine) {
    const int lane = threadIdx.x % kWave;
    for (int at = from; at < end; at += kBatch * kWave) {
        int j[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const Place &place = list[min(at + u * kWave + lane, end - 1)];
            j[u] = LOOK ? place.position : place.token;
        }
        if (LOOK)
#pragma unroll
            for (int u = 0; u < kBatch; ++u) j[u] = (int)token_at(p.tokens, p.wide, j[u]) / kNoRange;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = at + u * kWave + lane;
            const bool in = i < end;
            if (LOOK && in) list[i].token = j[u];
            const uint64_t same = same_lanes(in, j[u], p.bits);
            if (in && (same & (((uint64_t)1 << lane) - 1)) == 0) mine[j[u]] += __popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
    }
}

__device__ __forceinline__ void place_positions(const SortParams &p, int range, const Place *list, int from, int end, int *mine) {
    const int lane = threadIdx.x % kWave;
    for (int at = from; at < end; at += kBatch * kWave) {
        Place place[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) place[u] = list[min(at + u * kWave + lane, end - 1)];
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (at + u * kWave < end)
                sort_place(p, at + u * kWave + lane < end, place[u].token, place[u].token * kNoRange + range, place[u].position, mine);
    }
}

// Sorts a range's positions by token: into `list`, where the wave's blocks begin at `next`, and from there into p.order.
__device__ __forceinline__ void sort_range(const SortParams &p, int range, int first, int n, int block0, int block1, int next,
                                           Place *list, int *counts, int *sums) {
    const int wave = threadIdx.x / kWave, tiles = (n + kWave - 1) / kWave;
    const int from = tiles * wave / kSortWaves * kWave, end = min(n, tiles * (wave + 1) / kSortWaves * kWave);
    int *mine = counts + wave * p.width;
    pick_positions(p, range, block0, block1, next, list);
    __syncthreads();
    count_positions<true>(p, list, from, end, mine);
    __syncthreads();
    sort_places(p, range, first, counts, sums);
    place_positions(p, range, list, from, end, mine);
}

// A helper's range and its part of it.  Helpers are numbered through the heavy ranges; at most 3 M / heavy are needed, since
// ceil(2 n / heavy) < 3 n / heavy for n > heavy.
struct Share {
    int range, part, parts;
};
__device__ __forceinline__ Share find_share(const SortParams &p, int helper, int *firsts, int *sums) {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    if (tid < kThreads) firsts[tid] = 0;
    __syncthreads();
    constexpr int kQuarters = kSortThreads / kThreads, kReads = 16;
    int first = 0;  // positions of ranges below this thread's, in a quarter of the blocks
    for (int b0 = tid / kThreads; b0 < p.blocks; b0 += kReads * kQuarters) {
        int below[kReads];
#pragma unroll
        for (int u = 0; u < kReads; ++u) below[u] = p.below[min(b0 + u * kQuarters, p.blocks - 1) * kThreads + tid % kThreads];
#pragma unroll
        for (int u = 0; u < kReads; ++u)
            if (b0 + u * kQuarters < p.blocks) first += below[u];
    }
    atomicAdd(&firsts[tid % kThreads], first);
    __syncthreads();
    const int n = tid < kThreads - 1 ? firsts[tid + 1] - firsts[tid] : 0;
    const int here = n > p.heavy ? min((int)((2 * (int64_t)n + p.heavy - 1) / p.heavy), p.blocks) : 0;
    int upto = here;
    for (int step = 1; step < kWave; step *= 2) {
        const int other = __shfl_up(upto, step);
        if (lane >= step) upto += other;
    }
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += sums[w];
    __syncthreads();
    if (tid == 0) sums[0] = -1;
    __syncthreads();
    if (helper >= upto - here && helper < upto) {  // one thread at most
        sums[0] = tid;
        sums[1] = helper - (upto - here);
        sums[2] = here;
    }
    __syncthreads();
    const Share share{sums[0], sums[1], sums[2]};
    if (tid < 3) p.assigned[helper * 3 + tid] = sums[tid];
    __syncthreads();
    return share;
}

// Range blockIdx.x - helpers, unless helpers share it; of a helper's part the positions with their tokens and the counts.
__global__ void __launch_bounds__(kSortThreads) embedding_pick_kernel(SortParams p) {
    __shared__ int counts[kSortWaves * kWidthMost];  // [waves][width]
    __shared__ int sums[kSortWaves], offsets[kBlocksMost + 1], bases[kSortWaves];
    __shared__ Place held[kHeld];
    const int tid = threadIdx.x, wave = tid / kWave;
    for (int i = tid; i < kSortWaves * p.width; i += kSortThreads) counts[i] = 0;
    if ((int)blockIdx.x >= p.helpers) {
        const int range = blockIdx.x - p.helpers;
        const int first = range_offsets(p, range, offsets, sums, bases), n = offsets[p.blocks];
        if (p.helpers && n > p.heavy) return;
        const int block0 = p.blocks * wave / kSortWaves, block1 = p.blocks * (wave + 1) / kSortWaves;
        if (n <= kHeld) {
            sort_range(p, range, first, n, block0, block1, offsets[block0], held, counts, sums);
        } else {
            sort_range(p, range, first, n, block0, block1, offsets[block0], p.picked + first, counts, sums);
        }
        return;
    }
    const Share share = find_share(p, blockIdx.x, offsets, sums);
    if (share.range < 0) return;
    const int first = range_offsets(p, share.range, offsets, sums, bases);
    const int begin = p.blocks * share.part / share.parts, blocks = p.blocks * (share.part + 1) / share.parts - begin;
    const int block0 = begin + blocks * wave / kSortWaves, block1 = begin + blocks * (wave + 1) / kSortWaves;
    const int base = offsets[begin], n = offsets[begin + blocks] - base, tiles = (n + kWave - 1) / kWave;
    const int from = tiles * wave / kSortWaves * kWave, end = min(n, tiles * (wave + 1) / kSortWaves * kWave);
    Place *list = p.picked + first + base;
    pick_positions(p, share.range, block0, block1, offsets[block0] - base, list);
    __syncthreads();
    count_positions<true>(p, list, from, end, counts + wave * p.width);
    __syncthreads();
    for (int j = tid; j < p.width; j += kSortThreads) {
        int here = 0;
        for (int w = 0; w < kSortWaves; ++w) here += counts[w * p.width + j];
        p.shares[blockIdx.x * p.width + j] = here;
    }
}

// The helpers' second half: their places, from the counts of all.
__global__ void __launch_bounds__(kSortThreads) embedding_share_kernel(SortParams p) {
    __shared__ int counts[kSortWaves * kWidthMost];  // [waves][width]
    __shared__ int sums[kSortWaves], offsets[kBlocksMost + 1], bases[kSortWaves];
    const int tid = threadIdx.x, wave = tid / kWave;
    const int *assigned = p.assigned + blockIdx.x * 3;
    const Share share{assigned[0], assigned[1], assigned[2]};
    if (share.range < 0) return;
    for (int i = tid; i < kSortWaves * p.width; i += kSortThreads) counts[i] = 0;
    const int first = range_offsets(p, share.range, offsets, sums, bases);
    const int begin = p.blocks * share.part / share.parts, after = p.blocks * (share.part + 1) / share.parts;
    const int base = offsets[begin], n = offsets[after] - base, tiles = (n + kWave - 1) / kWave;
    const int from = tiles * wave / kSortWaves * kWave, end = min(n, tiles * (wave + 1) / kSortWaves * kWave);
    Place *list = p.picked + first + base;
    int *mine = counts + wave * p.width;
    count_positions<false>(p, list, from, end, mine);
    __syncthreads();
    sort_places(p, share.range, first, counts, sums, p.shares + (blockIdx.x - share.part) * p.width, share.part, share.parts);
    place_positions(p, share.range, list, from, end, mine);
}

template <typename T> struct SumParams {
    int64_t M;
    int vocab, cols, slices;  // slices: of the columns, one vector a lane
    Numbering numbering;
    int chunk, chunks;        // sorted positions of a wave's walk, and the most such walks
    int clears;               // waves that look for tokens without positions
    float scale;
    const Place *order;
    const int *start;
    const T *dout;
    float *parts;  // [chunks][2][slices][lanes' columns]: of a run that began before the chunk, and of one that goes on behind it
    T *out;
    bool add;
};

// A lane's part of a run that enters (0) or leaves (1) a chunk.
template <typename T>
__device__ __forceinline__ floatx4 *part_at(const SumParams<T> &p, int64_t chunk, int which, int slice, int lane) {
    return reinterpret_cast<floatx4 *>(p.parts + (((chunk * 2 + which) * p.slices + slice) * kWave + lane) * Vec<T>::kN);
}
template <typename T>
__device__ __forceinline__ void store_part(floatx4 *to, const float (&x)[Vec<T>::kN]) {
#pragma unroll
    for (int e = 0; e < Vec<T>::kN; e += 4) to[e / 4] = floatx4{x[e], x[e + 1], x[e + 2], x[e + 3]};
}

// Writes a token's finished row: scale x sum, added to what is there where `old` is given.
template <typename T, bool ADD>
__device__ __forceinline__ void write_row(const SumParams<T> &p, const Columns<T> &c, int token, float (&sum)[Vec<T>::kN],
                                          const typename Vec<T>::type &old) {
#pragma unroll
    for (int e = 0; e < Vec<T>::kN; ++e) sum[e] = ADD ? fmaf(p.scale, sum[e], widen(old[e])) : p.scale * sum[e];
    c.store(p.out + (int64_t)token * p.cols, sum);
}

template <typename T, bool ADD>
__global__ void __launch_bounds__(kThreads, 5) embedding_sum_kernel(SumParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    const int lane = threadIdx.x % kWave;
    const int64_t task = (int64_t)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t walks = (int64_t)p.chunks * p.slices;
    if (task >= walks) {  // the rows of tokens that have no position
        const int64_t clear = task - walks;
        if (ADD || clear >= p.clears) return;  // the last workgroup's spare waves
        const int row0 = (int)clear * kClearRows, mine = min(row0 + lane, p.vocab - 1);
        uint64_t empty = __ballot(lane < kClearRows && row0 + lane < p.vocab && p.start[p.numbering.number(mine) + 1] == p.start[p.numbering.number(mine)]);
        float zero[kN] = {};
        for (; empty; empty &= empty - 1) {
            T *row = p.out + (int64_t)(row0 + __ffsll((unsigned long long)empty) - 1) * p.cols;
            for (int first = lane * kN; first < p.cols; first += kWave * kN) Columns<T>(first, p.cols).store(row, zero);
        }
        return;
    }
    const int chunk = (int)(task / p.slices), slice = (int)(task - (int64_t)chunk * p.slices);
    const int begin = chunk * p.chunk, end = (int)min(p.M, (int64_t)begin + p.chunk);
    const Columns<T> c((slice * kWave + lane) * kN, p.cols);
    const int previous = begin > 0 ? p.order[begin - 1].token : -1;
    bool came = false, goes_on = false;  // the present run began before the chunk; the last one goes on behind it
    float sum[kN] = {};
    for (int base = begin; base < end; base += kWave) {
        const Place place = p.order[min(base + lane, end - 1)];
        const int next = (int64_t)base + lane + 1 < p.M ? p.order[base + lane + 1].token : -1;
        const bool in = base + lane < end && place.token >= 0;
        const int n = __popcll(__ballot(in));  // the counted positions come first
        if (n == 0) break;
        if (base == begin) came = __builtin_amdgcn_readlane(place.token, 0) == previous;
        // The positions that end their token's run; the chunk's last one leaves it unfinished where it goes on.
        const uint64_t more = __ballot(in && next == place.token);
        goes_on = base + n == end && (more >> (n - 1) & 1);
        const uint64_t ends = __ballot(in) & ~more;
        for (int j0 = 0; j0 < n; j0 += kBatch) {
            typename Vec<T>::type row[kBatch], old[kBatch];  // as they are, until they are summed
            const bool finishes = ADD && (ends >> j0 & ((1u << kBatch) - 1));
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int j = min(j0 + u, n - 1);
                const T *from = p.dout + (int64_t)__builtin_amdgcn_readlane(place.position, j) * p.cols;
                if (c.any()) c.load(from, row[u]);
                if (finishes) {  // where no row is finished, dout's own row once more, which is near
                    const T *there = p.out + (int64_t)__builtin_amdgcn_readlane(place.token, j) * p.cols;
                    if (c.any()) c.load(ends >> j & 1 ? there : from, old[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int j = j0 + u;
                if (j >= n) break;
#pragma unroll
                for (int e = 0; e < kN; ++e) sum[e] += widen(row[u][e]);
                if (ends >> j & 1) {
                    if (c.any()) {
                        if (came) {
                            store_part<T>(part_at(p, chunk, 0, slice, lane), sum);
                        } else {
                            write_row<T, ADD>(p, c, __builtin_amdgcn_readlane(place.token, j), sum, old[u]);
                        }
                    }
                    came = false;
#pragma unroll
                    for (int e = 0; e < kN; ++e) sum[e] = 0.0f;
                }
            }
        }
    }
    // A run through the whole chunk counts as begun before it.
    if (goes_on && c.any()) store_part<T>(part_at(p, chunk, came ? 0 : 1, slice, lane), sum);
}

// The number of parts of a run that began in a chunk and left it, or 0.
template <typename T> __device__ __forceinline__ int parts_of(const SumParams<T> &p, int chunk) {
    const int64_t begin = (int64_t)chunk * p.chunk, end = begin + p.chunk;
    if (end >= p.M) return 0;
    const int token = p.order[end - 1].token;
    if (token < 0 || p.order[end].token != token || (begin > 0 && p.order[begin - 1].token == token)) return 0;
    return (p.start[p.numbering.number(token) + 1] - 1) / p.chunk - chunk + 1;
}

// The parts of such runs.  A wave joins the few of its own; many are shared by the workgroup, each wave summing every
// kJoinWaves-th.  8 waves: a run of 80 thousand positions 44 -> 27 us against 4 waves that share every run.
template <typename T, bool ADD>
__global__ void __launch_bounds__(kJoinWaves * kWave) embedding_join_kernel(SumParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    __shared__ float joined[kJoinWaves][kN][kWave];
    __shared__ int many[kJoinWaves];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int first = blockIdx.x * kJoinWaves, tasks = p.chunks * p.slices;  // a long run's slices in different workgroups
    const auto sum_parts = [&](int chunk, int slice, int from, int step, int count, float (&sum)[kN]) {
        for (int k0 = from; k0 < count; k0 += kBatch * step) {
            floatx4 x[kBatch][kN / 4];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int k = min(k0 + u * step, count - 1);
                const floatx4 *at = part_at(p, chunk + k, k == 0, slice, lane);
#pragma unroll
                for (int e = 0; e < kN / 4; ++e) x[u][e] = at[e];
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    if (k0 + u * step < count) sum[e] += x[u][e / 4][e % 4];
        }
    };
    const auto write = [&](const Columns<T> &c, int chunk, float (&sum)[kN]) {
        const int token = p.order[(int64_t)(chunk + 1) * p.chunk - 1].token;
        typename Vec<T>::type old{};
        if (ADD) c.load(p.out + (int64_t)token * p.cols, old);
        write_row<T, ADD>(p, c, token, sum, old);
    };
    const int task = first + wave, slice = task / p.chunks, chunk = task - slice * p.chunks;
    const int count = task < tasks ? parts_of(p, chunk) : 0;
    const Columns<T> c((slice * kWave + lane) * kN, p.cols);
    if (count > 0 && count <= kJoinAlone && c.any()) {
        float sum[kN] = {};
        sum_parts(chunk, slice, 0, 1, count, sum);
        write(c, chunk, sum);
    }
    if (lane == 0) many[wave] = count > kJoinAlone ? count : 0;
    __syncthreads();
    for (int w = 0; w < kJoinWaves; ++w) {
        const int count = many[w];
        if (count == 0) continue;
        const int slice = (first + w) / p.chunks, chunk = first + w - slice * p.chunks;
        const Columns<T> c((slice * kWave + lane) * kN, p.cols);
        float sum[kN] = {};
        if (c.any()) sum_parts(chunk, slice, wave, kJoinWaves, count, sum);
#pragma unroll
        for (int e = 0; e < kN; ++e) joined[wave][e][lane] = sum[e];
        __syncthreads();
        if (wave == 0 && c.any()) {
#pragma unroll
            for (int e = 0; e < kN; ++e)
                for (int v = 1; v < kJoinWaves; ++v) sum[e] += joined[v][e][lane];
            write(c, chunk, sum);
        }
        __syncthreads();
    }
}

struct GradPlan {
    int width, ranges, bits, numbers, slices, chunk, chunks, clears;
    int blocks;                     // 0: the ranges are not written down
    int64_t block;
    int heavy, helpers;             // no helpers: no range is shared
    int64_t sums, joins;            // workgroups
    size_t order, start, parts, bytes_of, below, picked, shares, assigned, bytes;  // offsets into the workspace, and its size
};

// Sorted positions of a wave's walk: as many as leave kWalks waves, so that short batches still fill the card and long ones
// do so in one round.
GradPlan grad_plan(int64_t M, int V, int D, int vec) {
    GradPlan g{};
    g.ranges = std::max(std::min(V, kSortRanges), ceil_div(V, kRangeMost));
    g.width = ceil_div(V, g.ranges);
    g.ranges = ceil_div(V, g.width);
    if (M > kManyPositions && V <= kNoRange * kWidthMost) {
        g.ranges = std::min(V, kNoRange);
        g.width = ceil_div(V, kNoRange);
        const int64_t run = (M + kBlocksMost - 1) / kBlocksMost;
        g.block = (run + kBlockRun - 1) / kBlockRun * kBlockRun;
        g.blocks = (int)((M + g.block - 1) / g.block);
        if (M > kSplitPositions) {
            g.heavy = (int)std::max<int64_t>(kHeavy, M / kHeavyShare);
            g.helpers = (int)(3 * M / g.heavy);
        }
    }
    while (1 << g.bits < g.width) ++g.bits;
    g.numbers = g.blocks ? g.ranges * g.width : V;
    g.slices = ceil_div(D, kWave * vec);
    const int64_t each = (M * g.slices + kWalks - 1) / kWalks;
    g.chunk = (int)std::min<int64_t>(256, std::max<int64_t>(8, (each + 7) / 8 * 8));
    g.chunks = (int)((M + g.chunk - 1) / g.chunk);
    g.clears = ceil_div(V, kClearRows);
    g.joins = (int64_t)g.chunks * g.slices;
    g.sums = (g.joins + g.clears + kThreads / kWave - 1) / (kThreads / kWave);
    const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    g.order = 0;
    g.start = round((size_t)M * sizeof(Place));
    g.parts = g.start + round(((size_t)g.numbers + 1) * sizeof(int));
    g.bytes_of = g.parts + round((size_t)g.chunks * 2 * g.slices * kWave * vec * sizeof(float));
    g.below = g.bytes_of + round((size_t)(g.blocks * g.block));
    g.picked = g.below + round((size_t)g.blocks * kThreads * sizeof(int));
    g.shares = g.picked + (g.blocks ? round((size_t)M * sizeof(Place)) : 0);
    g.assigned = g.shares + round((size_t)g.helpers * g.width * sizeof(int));
    g.bytes = g.assigned + round((size_t)g.helpers * 3 * sizeof(int));
    return g;
}

// Why the operator refuses sizes, or null.
const char *grad_refusal(int64_t M, int V, int D, int vec) {
    if (M < 0 || V < 0 || D < 0) return "embedding gradient: negative size";
    if (V > kVocabMost || D > kColsMost) return "embedding gradient: V and D may not exceed 2^24";
    if (M > (int64_t)1 << 30) return "embedding gradient: more than 2^30 tokens";
    if (V == 0 || D == 0) return nullptr;
    const GradPlan g = grad_plan(M, V, D, vec);
    if (std::max(g.sums, g.joins) * kThreads >= (int64_t)1 << 32) return "embedding gradient: too many elements";  // threads of a launch
    return nullptr;
}

template <typename T, bool ADD>
int launch_grad(const GradPlan &g, const SortParams &sort, const SumParams<T> &sum, hipStream_t s) {
    const size_t counters = kSortWaves * g.width * sizeof(int);
    if (g.blocks) {
        hipLaunchKernelGGL(embedding_ranges_kernel, dim3(g.blocks), dim3(kThreads), 0, s, sort);
        hipLaunchKernelGGL(embedding_pick_kernel, dim3(g.helpers + g.ranges), dim3(kSortThreads), 0, s, sort);
        if (g.helpers) hipLaunchKernelGGL(embedding_share_kernel, dim3(g.helpers), dim3(kSortThreads), 0, s, sort);
    } else {
        const auto kernel = sort.M <= kManyPositions ? embedding_sort_kernel<true> : embedding_sort_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(g.ranges), dim3(kSortThreads), counters, s, sort);
    }
    const int64_t sums = ADD ? (g.joins + kThreads / kWave - 1) / (kThreads / kWave) : g.sums;
    hipLaunchKernelGGL((embedding_sum_kernel<T, ADD>), dim3((uint32_t)sums), dim3(kThreads), 0, s, sum);
    if (g.chunks > 1) hipLaunchKernelGGL((embedding_join_kernel<T, ADD>), dim3((uint32_t)((g.joins + kJoinWaves - 1) / kJoinWaves)), dim3(kJoinWaves * kWave), 0, s, sum);
    YUF_LAUNCH_CHECK("embedding gradient");
    return YUF_OK;
}

template <typename T>
int embedding_grad(int64_t M, int V, int D, const void *tokens, int token_bits, const T *dout, double scale, int64_t padding,
                   int accumulate, T *out, void *workspace, void *stream) {
    if (const char *why = grad_refusal(M, V, D, Vec<T>::kN)) return fail(YUF_ERR_INVALID, why);
    if (token_bits != 32 && token_bits != 64) return fail(YUF_ERR_INVALID, "embedding gradient: token_bits must be 32 or 64");
    if (accumulate != 0 && accumulate != 1) return fail(YUF_ERR_INVALID, "embedding gradient: accumulate must be 0 or 1");
    if (V == 0 || D == 0 || (M == 0 && accumulate)) return YUF_OK;
    if (!out || (M > 0 && (!tokens || !dout))) return fail(YUF_ERR_INVALID, "embedding gradient: null tokens, gradient or output");
    if (!workspace || !scratch_aligned(workspace))
        return fail(YUF_ERR_INVALID, "embedding gradient: the workspace must be given and 256-byte aligned");
    const GradPlan g = grad_plan(M, V, D, Vec<T>::kN);
    const size_t row = (size_t)D * sizeof(T);
    if (outputs_overlap<2, 2>({{tokens, (size_t)M * (token_bits / 8)}, {dout, M * row}}, {{out, V * row}, {workspace, g.bytes}}))
        return fail(YUF_ERR_INVALID, "embedding gradient: the output and the workspace may not be an input or each other, nor a part of them");
    char *space = static_cast<char *>(workspace);
    SortParams sort{};
    sort.M = M; sort.vocab = V; sort.width = g.width; sort.bits = g.bits; sort.numbers = g.numbers;
    sort.block = g.block; sort.blocks = g.blocks;
    sort.ranges = reinterpret_cast<uint8_t *>(space + g.bytes_of);
    sort.below = reinterpret_cast<int *>(space + g.below);
    sort.picked = reinterpret_cast<Place *>(space + g.picked);
    sort.heavy = g.heavy; sort.helpers = g.helpers; sort.shares = reinterpret_cast<int *>(space + g.shares);
    sort.assigned = reinterpret_cast<int *>(space + g.assigned);
    sort.tokens = tokens; sort.wide = token_bits == 64; sort.padding = padding;
    sort.order = reinterpret_cast<Place *>(space + g.order);
    sort.start = reinterpret_cast<int *>(space + g.start);
    SumParams<T> sum{};
    sum.numbering = {g.width, g.blocks > 0};
    sum.M = M; sum.vocab = V; sum.cols = D; sum.slices = g.slices; sum.chunk = g.chunk; sum.chunks = g.chunks;
    sum.clears = g.clears;
    sum.scale = (float)scale;
    sum.order = sort.order; sum.start = sort.start; sum.dout = dout;
    sum.parts = reinterpret_cast<float *>(space + g.parts);
    sum.out = out;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return accumulate ? launch_grad<T, true>(g, sort, sum, s) : launch_grad<T, false>(g, sort, sum, s);
}

}  // namespace
}  // namespace yuf

extern "C" int yuf_embedding_f32(int64_t M, int V, int D, const float *table, const void *tokens, int token_bits, double scale,
                                 float *out, void *stream) {
    return yuf::embedding<float>(M, V, D, table, tokens, token_bits, scale, out, stream);
}

extern "C" int yuf_embedding_bf16(int64_t M, int V, int D, const uint16_t *table, const void *tokens, int token_bits,
                                  double scale, uint16_t *out, void *stream) {
    return yuf::embedding<uint16_t>(M, V, D, table, tokens, token_bits, scale, out, stream);
}

extern "C" size_t yuf_embedding_grad_workspace(int64_t M, int V, int D) {
    size_t bytes = 0;  // for either type
    for (int vec : {4, 8})
        if (V > 0 && D > 0 && !yuf::grad_refusal(M, V, D, vec)) bytes = std::max(bytes, yuf::grad_plan(M, V, D, vec).bytes);
    return bytes;
}

extern "C" int yuf_embedding_grad_f32(int64_t M, int V, int D, const void *tokens, int token_bits, const float *dout,
                                      double scale, int64_t padding, int accumulate, float *out, void *workspace, void *stream) {
    return yuf::embedding_grad<float>(M, V, D, tokens, token_bits, dout, scale, padding, accumulate, out, workspace, stream);
}

extern "C" int yuf_embedding_grad_bf16(int64_t M, int V, int D, const void *tokens, int token_bits, const uint16_t *dout,
                                       double scale, int64_t padding, int accumulate, uint16_t *out, void *workspace, void *stream) {
    return yuf::embedding_grad<uint16_t>(M, V, D, tokens, token_bits, dout, scale, padding, accumulate, out, workspace, stream);
}
