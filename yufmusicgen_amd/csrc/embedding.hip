// Token embedding and its gradient:
//     out[i] = scale W[t_i],    dW[v] (+)= scale sum_{i: t_i = v} dout[i].
//
// Bound: HBM -- the looked-up rows and the outputs once; for the gradient dout once and the whole table
// once (twice where it is added to).
//
// The gradient's sums run over each token's positions in order, so they do not depend on timing: no
// atomics on values.  Three launches:
//   sort:  a workgroup owns a range of tokens and reads all ids twice.  Each of its waves takes a run of
//          positions: it counts the tokens of the range, and the ids below it (which gives where the range's
//          positions begin without asking another workgroup); after a scan over tokens and waves it
//          places its positions, in order.
//   sum:   a wave walks a chunk of the sorted positions for up to 64 vectors of columns and writes a
//          token's row where its run ends.  Runs that leave the chunk go to the workspace as fp32 parts.
//          Further waves clear the rows of tokens that do not occur.
//   join:  the parts of such a run, in order.
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
constexpr int kBatch = 8;         // rows of a wave in flight
constexpr int kClearRows = 8;     // table rows that a wave looks over for tokens without positions
constexpr int kJoinWaves = kThreads / kWave;
constexpr int kVocabMost = 1 << 24, kColsMost = 1 << 24;

// Vectors with the alignment of their elements: rows of odd widths start anywhere.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
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
    __device__ __forceinline__ void load(const T *row, float (&x)[Vec<T>::kN]) const {
        constexpr int kN = Vec<T>::kN;
        if (end == kN) {
            const auto v = *reinterpret_cast<const typename Vec<T>::type *>(row + at);
#pragma unroll
            for (int e = 0; e < kN; ++e) x[e] = widen(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) x[e] = e < end ? widen(row[at + e]) : 0.0f;
        }
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

struct SortParams {
    int64_t M;
    int vocab, width, bits;  // tokens of a range, bits of an index into it
    const void *tokens;
    bool wide;
    int64_t padding;  // or -1
    Place *order;     // [M]
    int *start;       // [V + 1]
};

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(SortParams p) {
    extern __shared__ int counts[];  // [waves][width]: counts, then where a wave's next position goes
    __shared__ int below[kSortWaves], sums[kSortWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int low = blockIdx.x * p.width, width = min(p.width, p.vocab - low);
    int *mine = counts + wave * p.width;
    for (int i = threadIdx.x; i < kSortWaves * p.width; i += kSortThreads) counts[i] = 0;
    __syncthreads();
    // This wave's run of positions, in whole waves of them.
    const int64_t tiles = (p.M + kWave - 1) / kWave;
    const int64_t first = tiles * wave / kSortWaves * kWave, last = min(p.M, tiles * (wave + 1) / kSortWaves * kWave);
    const auto read = [&](int64_t at) -> int {  // the token, or -1: not to be counted
        if (at + lane >= last) return -1;
        const int64_t t = token_at(p.tokens, p.wide, at + lane);
        return t >= 0 && t < p.vocab && t != p.padding ? (int)t : -1;
    };
    int less = 0;
    for (int64_t at = first; at < last; at += kBatch * kWave) {
        int t[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) t[u] = read(at + u * kWave);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            less += t[u] >= 0 && t[u] < low;
            if (t[u] >= low && t[u] < low + width) atomicAdd(&mine[t[u] - low], 1);
        }
    }
    for (int step = 1; step < kWave; step *= 2) less += __shfl_xor(less, step);
    if (lane == 0) below[wave] = less;
    __syncthreads();
    // Counts of a token before each wave, then of the tokens before each token.
    int total = 0;
    for (int w = 0; w < kSortWaves; ++w) total += below[w];
    for (int base = 0; base < width; base += kSortThreads) {
        const int j = base + threadIdx.x;
        int here = 0;
        if (j < width)
            for (int w = 0; w < kSortWaves; ++w) here += counts[w * p.width + j];
        int upto = here;  // inclusive scan over the workgroup
        for (int step = 1; step < kWave; step *= 2) {
            const int other = __shfl_up(upto, step);
            if (lane >= step) upto += other;
        }
        if (lane == kWave - 1) sums[wave] = upto;
        __syncthreads();
        int before = total, all = 0;
        for (int w = 0; w < kSortWaves; ++w) {
            if (w < wave) before += sums[w];
            all += sums[w];
        }
        int next = before + upto - here;
        if (j < width) {
            p.start[low + j] = next;
            for (int w = 0; w < kSortWaves; ++w) {
                const int n = counts[w * p.width + j];
                counts[w * p.width + j] = next;
                next += n;
            }
        }
        total += all;
        __syncthreads();
    }
    if (low + width == p.vocab && threadIdx.x == 0) p.start[p.vocab] = total;
    // Places, in the order of positions: lanes of the same token rank themselves by comparing its bits.
    for (int64_t at = first; at < last; at += kBatch * kWave) {
        int t[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) t[u] = read(at + u * kWave);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const bool in = t[u] >= low && t[u] < low + width;
            uint64_t same = __ballot(in);
            if (same == 0) continue;
            const int j = t[u] - low;
            for (int bit = 0; bit < p.bits; ++bit) {
                const uint64_t set = __ballot(in && (j >> bit & 1));
                same &= j >> bit & 1 ? set : ~set;
            }
            if (in) {
                const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
                const int at0 = mine[j];
                __builtin_amdgcn_wave_barrier();
                p.order[at0 + rank] = {(int)(at + u * kWave) + lane, t[u]};
                if (rank == 0) mine[j] = at0 + __popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <typename T> struct SumParams {
    int vocab, cols, slices;  // slices: of the columns, one vector a lane
    int chunk, chunks;        // sorted positions of a wave's walk, and the most such walks
    int clears;               // waves that look for tokens without positions
    float scale;
    const Place *order;
    const int *start;
    const T *dout;
    float *parts;  // [chunks][2][cols]: of a run that began before the chunk, and of one that goes on behind it
    T *out;
    bool add;
};

// Writes a token's finished row: scale x sum, added to what is there where `old` is given.
template <typename T, bool ADD>
__device__ __forceinline__ void write_row(const SumParams<T> &p, const Columns<T> &c, int token, float (&sum)[Vec<T>::kN],
                                          const float (&old)[Vec<T>::kN]) {
#pragma unroll
    for (int e = 0; e < Vec<T>::kN; ++e) sum[e] = ADD ? fmaf(p.scale, sum[e], old[e]) : p.scale * sum[e];
    c.store(p.out + (int64_t)token * p.cols, sum);
}

template <typename T, bool ADD>
__global__ void __launch_bounds__(kThreads) embedding_sum_kernel(SumParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    const int lane = threadIdx.x % kWave;
    const int64_t task = (int64_t)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t walks = (int64_t)p.chunks * p.slices;
    if (task >= walks) {  // the rows of tokens that have no position
        const int64_t clear = task - walks;
        if (ADD || clear >= p.clears) return;  // the last workgroup's spare waves
        for (int r = 0; r < kClearRows; ++r) {
            const int row = (int)clear * kClearRows + r;
            if (row >= p.vocab) return;
            if (p.start[row + 1] != p.start[row]) continue;
            float zero[kN] = {};
            for (int first = lane * kN; first < p.cols; first += kWave * kN)
                Columns<T>(first, p.cols).store(p.out + (int64_t)row * p.cols, zero);
        }
        return;
    }
    const int chunk = (int)(task / p.slices), slice = (int)(task - (int64_t)chunk * p.slices);
    const int all = p.start[p.vocab];
    const int begin = chunk * p.chunk, end = min(all, begin + p.chunk);
    if (begin >= end) return;
    const Columns<T> c((slice * kWave + lane) * kN, p.cols);
    const bool goes_on = end < all && p.order[end].token == p.order[end - 1].token;
    bool came = begin > 0 && p.order[begin - 1].token == p.order[begin].token;  // the present run began before the chunk
    float sum[kN] = {};
    for (int base = begin; base < end; base += kWave) {
        const int n = min(kWave, end - base);
        const Place place = p.order[min(base + lane, end - 1)];
        // Whether this lane's position ends its token's run.
        const int next = __shfl_down(place.token, 1);
        const bool closes = base + lane == end - 1 ? !goes_on : lane == kWave - 1 ? p.order[base + kWave].token != place.token : next != place.token;
        const uint64_t ends = __ballot(lane < n && closes);
        for (int j0 = 0; j0 < n; j0 += kBatch) {
            float row[kBatch][kN], old[kBatch][kN];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int j = min(j0 + u, n - 1);
                const T *from = p.dout + (int64_t)__builtin_amdgcn_readlane(place.position, j) * p.cols;
                if (c.any()) c.load(from, row[u]);
                if (ADD) {  // where no row is finished, dout's own row once more, which is near
                    const T *there = p.out + (int64_t)__builtin_amdgcn_readlane(place.token, j) * p.cols;
                    if (c.any()) c.load(ends >> j & 1 ? there : from, old[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int j = j0 + u;
                if (j >= n) break;
#pragma unroll
                for (int e = 0; e < kN; ++e) sum[e] += row[u][e];
                if (ends >> j & 1) {
                    if (c.any()) {
                        if (came) {
                            float *part = p.parts + (int64_t)chunk * 2 * p.cols + c.at;
#pragma unroll
                            for (int e = 0; e < kN; ++e)
                                if (e >= c.own && e < c.end) part[e] = sum[e];
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
    if (goes_on && c.any()) {  // a run through the whole chunk counts as begun before it
        float *part = p.parts + ((int64_t)chunk * 2 + (came ? 0 : 1)) * p.cols + c.at;
#pragma unroll
        for (int e = 0; e < kN; ++e)
            if (e >= c.own && e < c.end) part[e] = sum[e];
    }
}

// The parts of a run that began in this workgroup's chunk: each wave sums every kJoinWaves-th, then they are joined.
template <typename T, bool ADD>
__global__ void __launch_bounds__(kThreads) embedding_join_kernel(SumParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    __shared__ float joined[kJoinWaves][kN][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int chunk = blockIdx.x / p.slices, slice = blockIdx.x - chunk * p.slices;
    const int64_t end = (int64_t)(chunk + 1) * p.chunk;
    if (end >= p.start[p.vocab]) return;
    const int token = p.order[end - 1].token;
    const int from = p.start[token], to = p.start[token + 1];
    if (from < end - p.chunk || to <= end) return;
    const int last = (to - 1) / p.chunk;  // its last chunk
    const Columns<T> c((slice * kWave + lane) * kN, p.cols);
    const auto part = [&](int k, float (&x)[kN]) {  // the run's k-th part
        const float *at = p.parts + ((int64_t)(chunk + k) * 2 + (k == 0 ? 1 : 0)) * p.cols + c.at;
#pragma unroll
        for (int e = 0; e < kN; ++e) x[e] = e >= c.own && e < c.end ? at[e] : 0.0f;
    };
    const int count = last - chunk + 1;
    float sum[kN] = {};
    if (c.any()) {
        for (int k0 = wave; k0 < count; k0 += kBatch * kJoinWaves) {
            float x[kBatch][kN];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) part(min(k0 + u * kJoinWaves, count - 1), x[u]);
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    if (k0 + u * kJoinWaves < count) sum[e] += x[u][e];
        }
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) joined[wave][e][lane] = sum[e];
    __syncthreads();
    if (wave != 0 || !c.any()) return;
    float old[kN] = {};
    if (ADD) c.load(p.out + (int64_t)token * p.cols, old);
#pragma unroll
    for (int e = 0; e < kN; ++e)
        for (int w = 1; w < kJoinWaves; ++w) sum[e] += joined[w][e][lane];
    write_row<T, ADD>(p, c, token, sum, old);
}

struct GradPlan {
    int width, ranges, slices, chunk, chunks, clears;
    int64_t sums, joins;            // workgroups
    size_t order, start, parts, bytes;  // offsets into the workspace, and its size
};

// Sorted positions of a wave's walk: as many as leave 16 waves a CU, so that short batches still fill the card.
GradPlan grad_plan(int64_t M, int V, int D, int vec) {
    GradPlan g{};
    g.ranges = std::max(std::min(V, kSortRanges), ceil_div(V, kRangeMost));
    g.width = ceil_div(V, g.ranges);
    g.ranges = ceil_div(V, g.width);
    g.slices = ceil_div(D, kWave * vec);
    g.chunk = 16;
    while (g.chunk < 256 && (M + 2 * g.chunk - 1) / (2 * g.chunk) * g.slices >= 4096) g.chunk *= 2;
    g.chunks = (int)((M + g.chunk - 1) / g.chunk);
    g.clears = ceil_div(V, kClearRows);
    g.joins = (int64_t)g.chunks * g.slices;
    g.sums = (g.joins + g.clears + kThreads / kWave - 1) / (kThreads / kWave);
    const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    g.order = 0;
    g.start = round((size_t)M * sizeof(Place));
    g.parts = g.start + round(((size_t)V + 1) * sizeof(int));
    g.bytes = g.parts + round((size_t)g.chunks * 2 * D * sizeof(float));
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
    hipLaunchKernelGGL(embedding_sort_kernel, dim3(g.ranges), dim3(kSortThreads), kSortWaves * g.width * sizeof(int), s, sort);
    const int64_t sums = ADD ? (g.joins + kThreads / kWave - 1) / (kThreads / kWave) : g.sums;
    hipLaunchKernelGGL((embedding_sum_kernel<T, ADD>), dim3((uint32_t)sums), dim3(kThreads), 0, s, sum);
    if (g.chunks > 1) hipLaunchKernelGGL((embedding_join_kernel<T, ADD>), dim3((uint32_t)g.joins), dim3(kThreads), 0, s, sum);
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
    sort.M = M; sort.vocab = V; sort.width = g.width;
    while (1 << sort.bits < g.width) ++sort.bits;
    sort.tokens = tokens; sort.wide = token_bits == 64; sort.padding = padding;
    sort.order = reinterpret_cast<Place *>(space + g.order);
    sort.start = reinterpret_cast<int *>(space + g.start);
    SumParams<T> sum{};
    sum.vocab = V; sum.cols = D; sum.slices = g.slices; sum.chunk = g.chunk; sum.chunks = g.chunks;
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
