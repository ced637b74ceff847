// Cross-entropy of logits and token ids, with the logits' gradient in the same pass:
//     lse = log sum_j exp(x_j),  loss = lse - x_target,
//     dx_j = (exp(x_j - lse) - [j = target]) * scale,
// scale = upstream gradient (/ number of rows that count, for a mean).  Rows whose
// target is ignore_index have loss 0 and gradient 0 and are not read.
//
// Bound: HBM -- the logits read once, their gradient written once.  A row stays in
// registers between the two (a wave per row for short rows, up to 16 waves for long
// ones), so the maximum, the sum and the gradient cost one read; rows beyond 16
// waves' registers are read twice.  Each wave takes its own maximum and sum, and
// the waves of a row join them through LDS with one barrier.  Everything is summed
// in fp32 inside a row and in fp64 over the rows, always in the same order.
// 16384 x 20480 fp32 with the gradient, 5 % of the rows ignored: 506 us, and 10 us to count
// the rows before and to sum their losses behind; 527 in all with none ignored = 5.1 TB/s (a copy of
// that size 5.1, a multiplication 6.2; a GPU that was idle takes 575 to 600 for its first 20 passes).
#include "common.h"

#include <algorithm>

namespace yuf {
namespace {

constexpr int kWave = 64;
constexpr int kRowsPerWg = 4;    // rows of a workgroup where a row is one wave
constexpr int kMaxWaves = 16;
constexpr int kBatch = 8;        // loads of a lane in flight where rows are counted and summed
// Up to kCountInline / (a row's waves) rows each workgroup counts the valid targets itself.  The whole call so
// and with a count before it, rows x vocabulary: a wave, 673: 6144 17.5 and 20.0, 8192 20.2 and 20.2, 16384 44 and
// 25 us; 4 waves, 2048: 2048 17.1 and 19.9, 4096 22.8 and 21.5; 8 waves, 20480 bf16: 1024 33.3 and 33.6,
// 2048 54 and 52; 16 waves, 20480: 512 26.6 and 25.9, 1024 47 and 42, 4096 171 and 151.
constexpr int kCountInline = 8192;

// Vectors with the alignment of their elements: a row of an odd vocabulary starts anywhere.
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
template <typename T> struct MinusInf;
template <> struct MinusInf<float> { static __device__ float get() { return -INFINITY; } };
template <> struct MinusInf<uint16_t> { static __device__ uint16_t get() { return 0xFF80; } };

struct LossParams {
    int M, V;
    int row0;  // first row of this launch
    const void *logits;
    int64_t ld;
    const void *targets;
    int64_t ignore;
    bool wide;           // targets are int64
    int reduction;
    float *row_loss;     // [M] or nullptr
    const float *count;  // [1]: valid rows, or nullptr (a mean counts them itself)
    const float *dloss;  // [1] or [M] (no reduction), or nullptr: 1
    void *dlogits;       // or nullptr
    int64_t ld_out;
};

__device__ __forceinline__ int64_t target_of(const void *targets, bool wide, int row) {
    return wide ? static_cast<const int64_t *>(targets)[row] : (int64_t)static_cast<const int32_t *>(targets)[row];
}

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_move<dpp::kQuadXor1>(x));
    x = fmaxf(x, dpp_move<dpp::kQuadXor2>(x));
    x = fmaxf(x, dpp_move<dpp::kRowHalfMirror>(x));
    x = fmaxf(x, dpp_move<dpp::kRowMirror>(x));
    const float a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 0));
    const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16));
    const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 32));
    const float d = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 48));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// A maximum that an exponent can be taken against: a part without any finite
// logit has exp(x - 0) = 0 everywhere.
__device__ __forceinline__ float finite_base(float m) { return m == -INFINITY ? 0.0f : m; }

// exp(m - all): what a part's exponentials are multiplied by where the maximum of
// all of them is `all` (its sum is 0 and has to stay so where it saw no finite logit).
__device__ __forceinline__ float rescale(float m, float all) { return m == -INFINITY ? 0.0f : expf(m - all); }

template <typename I> __device__ __forceinline__ int count_mine(const I *targets, uint32_t M, int64_t ignore) {
    int mine = 0;
    // kBatch loads in flight: one at a time, each waits for memory (16384 rows: 10.5 us, so 6.2).  Unsigned,
    // since the last step goes beyond M, which may be 2^31 - 1.
    for (uint32_t i0 = threadIdx.x; i0 < M; i0 += kBatch * blockDim.x) {
        I t[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) t[e] = targets[min(i0 + e * blockDim.x, M - 1)];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) mine += i0 + e * blockDim.x < M && (int64_t)t[e] != ignore;
    }
    return mine;
}

// Rows whose target counts, seen by every lane of the workgroup (all its threads call this).
__device__ __forceinline__ float count_valid(const LossParams &p, int *partial) {
    int mine = p.wide ? count_mine(static_cast<const int64_t *>(p.targets), p.M, p.ignore)
                      : count_mine(static_cast<const int32_t *>(p.targets), p.M, p.ignore);
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) mine += __shfl_xor(mine, s);
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = mine;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) all += partial[w];
    __syncthreads();
    return (float)all;
}

// WAVES waves per row (one: kRowsPerWg rows a workgroup), NV vectors per lane;
// NV = 0: rows of any length, read twice.
template <typename T, int WAVES, int NV>
__global__ void __launch_bounds__(WAVES == 1 ? kRowsPerWg * kWave : WAVES * kWave) loss_kernel(LossParams p) {
    constexpr int kN = Vec<T>::kN;
    using V = typename Vec<T>::type;
    constexpr int kLanes = WAVES * kWave;
    __shared__ float part[2 * kMaxWaves + 1];
    __shared__ int counts[kMaxWaves];
    float count = 1.0f;
    if (p.reduction == YUF_LOSS_MEAN && p.dlogits)
        count = p.count ? *p.count : count_valid(p, counts);
    const int row = p.row0 + (WAVES == 1 ? (int)blockIdx.x * kRowsPerWg + (int)(threadIdx.x >> 6) : (int)blockIdx.x);
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    if (row >= p.M) return;  // whole waves of a one-wave form, which has no barrier below
    const int64_t target = target_of(p.targets, p.wide, row);
    T *out = p.dlogits ? static_cast<T *>(p.dlogits) + (int64_t)row * p.ld_out : nullptr;
    const int full = p.V / kN, vecs = (p.V + kN - 1) / kN;  // whole vectors; with the ragged last one

    auto store = [&](int i, V v) {
        if (i < full) {
            *reinterpret_cast<V *>(out + (int64_t)i * kN) = v;
        } else if (i < vecs) {
#pragma unroll
            for (int e = 0; e < kN; ++e)
                if (i * kN + e < p.V) out[(int64_t)i * kN + e] = v[e];
        }
    };
    if (target == p.ignore) {
        if (lane == 0 && p.row_loss) p.row_loss[row] = 0.0f;
        if (out)
            for (int i = lane; i < vecs; i += kLanes) store(i, V{});
        return;
    }
    const bool in_range = target >= 0 && target < p.V;
    const T *x = static_cast<const T *>(p.logits) + (int64_t)row * p.ld;
    auto load = [&](int i) {
        V v;
        if (i < full) {
            v = *reinterpret_cast<const V *>(x + (int64_t)i * kN);
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = i * kN + e < p.V ? x[(int64_t)i * kN + e] : MinusInf<T>::get();
        }
        return v;
    };
    // Read, and waited for, before any lane writes: dlogits may be the logits themselves.
    float at_target = lane == 0 && in_range ? widen(x[target]) : NAN;

    // This wave's maximum and sum of exponentials against it.
    constexpr int kHeld = NV ? NV : 1;
    V held[kHeld];
    float top = -INFINITY, sum = 0.0f;
    if constexpr (NV > 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u) held[u] = load(lane + u * kLanes);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < kN; ++e) top = fmaxf(top, widen(held[u][e]));
        top = wave_max(top);
        const float base = finite_base(top);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                const float y = expf(widen(held[u][e]) - base);
                sum += y;
                if constexpr (sizeof(T) == 4) held[u][e] = y;  // fp32 keeps the exponential, bf16 the logit
            }
    } else {
        for (int i = lane; i < vecs; i += kLanes) {
            const V v = load(i);
            float m = widen(v[0]);
#pragma unroll
            for (int e = 1; e < kN; ++e) m = fmaxf(m, widen(v[e]));
            if (m > top) {
                sum *= rescale(top, m);
                top = m;
            }
            const float base = finite_base(top);
#pragma unroll
            for (int e = 0; e < kN; ++e) sum += expf(widen(v[e]) - base);
        }
        const float m = wave_max(top);
        sum *= rescale(top, m);
        top = m;
    }
    sum = wave_sum(sum);
    float all_top = top, all = sum;
    if constexpr (WAVES > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            part[2 * wave] = top;
            part[2 * wave + 1] = sum;
        }
        if (threadIdx.x == 0) part[2 * kMaxWaves] = at_target;
        __syncthreads();  // every read of the row is done
        at_target = part[2 * kMaxWaves];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) all_top = fmaxf(all_top, part[2 * w]);
        all = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            all += part[2 * w + 1] * rescale(part[2 * w], all_top);
    }
    const float base = finite_base(all_top);
    if (lane == 0 && p.row_loss) p.row_loss[row] = logf(all) - (at_target - base);
    if (!out) return;

    float scale = p.dloss ? p.dloss[p.reduction == YUF_LOSS_NONE ? row : 0] : 1.0f;
    scale /= count;
    if (!in_range) scale = NAN;  // a target outside the vocabulary: loss and gradient are NaN
    // p_j = exp(x_j - base) / all; a wave that holds exponentials has them against its own maximum.
    const float inv = 1.0f / all, mine = NV > 0 && sizeof(T) == 4 ? rescale(top, all_top) * inv : inv;
    auto grad = [&](V v, int i, bool exponentials) {
        V g;
        const int64_t hit = target - (int64_t)i * kN;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
            float q = exponentials ? widen(v[e]) * mine : expf(widen(v[e]) - base) * mine;
            if (hit == e) q -= 1.0f;
            T t;
            narrow(q * scale, t);
            g[e] = t;
        }
        store(i, g);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            if (lane + u * kLanes < vecs) grad(held[u], lane + u * kLanes, sizeof(T) == 4);
    } else {
        for (int i = lane; i < vecs; i += kLanes) grad(load(i), i, false);
    }
}

constexpr int kReduceThreads = 1024;

__global__ void __launch_bounds__(kReduceThreads) loss_count_kernel(LossParams p, float *count) {
    __shared__ int partial[kReduceThreads / kWave];
    const float n = count_valid(p, partial);
    if (threadIdx.x == 0) *count = n;
}

// Sum or mean of the row losses, in fp64 and one order.
__global__ void __launch_bounds__(kReduceThreads) loss_sum_kernel(LossParams p, float *loss) {
    __shared__ double sums[kReduceThreads / kWave];
    __shared__ int partial[kReduceThreads / kWave];
    double s = 0.0;
    const uint32_t M = p.M;  // unsigned, as where the rows are counted
    for (uint32_t i0 = threadIdx.x; i0 < M; i0 += kBatch * kReduceThreads) {
        float v[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) v[e] = p.row_loss[min(i0 + e * kReduceThreads, M - 1)];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) s += i0 + e * kReduceThreads < M ? (double)v[e] : 0.0;
    }
    s = wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    float n = 1.0f;
    if (p.reduction == YUF_LOSS_MEAN) n = p.count ? *p.count : count_valid(p, partial);
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < kReduceThreads / kWave; ++w) t += sums[w];
        *loss = (float)(t / (double)n);
    }
}

template <typename T, int WAVES, int NV>
void launch_form(LossParams p, hipStream_t s) {
    constexpr int kPerWg = WAVES == 1 ? kRowsPerWg : 1;
    constexpr int kRows = 1 << 21;  // of a launch, which has at most 2^32 threads
    for (; p.row0 < p.M; p.row0 += kRows) {
        const int rows = std::min(p.M - p.row0, kRows);
        hipLaunchKernelGGL((loss_kernel<T, WAVES, NV>), dim3((rows + kPerWg - 1) / kPerWg), dim3(kPerWg * WAVES * kWave), 0, s, p);
        if (p.M - p.row0 <= kRows) break;
    }
}

// The fewest waves whose registers hold the row.
int row_waves(int vecs) { return vecs <= 4 * kWave ? 1 : vecs <= 4 * 4 * kWave ? 4 : vecs <= 8 * 5 * kWave ? 8 : 16; }
template <typename T> int row_vecs(int V) { return (V + Vec<T>::kN - 1) / Vec<T>::kN; }

template <typename T>
void launch_rows(const LossParams &p, hipStream_t s) {
    const int vecs = row_vecs<T>(p.V), waves = row_waves(vecs);
    if (vecs <= 1 * kWave) launch_form<T, 1, 1>(p, s);
    else if (vecs <= 2 * kWave) launch_form<T, 1, 2>(p, s);
    else if (waves == 1) launch_form<T, 1, 4>(p, s);
    else if (waves == 4) launch_form<T, 4, 4>(p, s);
    else if (waves == 8) launch_form<T, 8, 5>(p, s);
    else if (vecs <= 16 * 5 * kWave) launch_form<T, 16, 5>(p, s);
    else if (vecs <= 16 * 8 * kWave) launch_form<T, 16, 8>(p, s);
    else {
        // Twice the registers hold fp32 rows only: bf16 rows of that length, widened, spill.
        if constexpr (sizeof(T) == 4)
            if (vecs <= 16 * 16 * kWave) return launch_form<T, 16, 16>(p, s);
        launch_form<T, 16, 0>(p, s);
    }
}

// Whether M rows of `bytes` at each of two places, a stride apart, share memory.  Rows of one stride may lie
// between each other's; of two strides, places that reach into each other are taken to overlap.
bool rows_overlap(int M, size_t bytes, const void *a, size_t stride_a, const void *b, size_t stride_b) {
    if (!overlap({a, (M - 1) * stride_a + bytes}, {b, (M - 1) * stride_b + bytes})) return false;
    if (stride_a != stride_b) return true;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    const size_t apart = (x < y ? y - x : x - y) % stride_a;
    return apart < bytes || stride_a - apart < bytes;
}

template <typename T>
int cross_entropy(int M, int V, const T *logits, int64_t ld, const void *targets, int target_bits, int64_t ignore,
                  int reduction, float *loss, const float *dloss, T *dlogits, int64_t ld_out, float *workspace,
                  void *stream) {
    if (M < 0 || V < 0) return fail(YUF_ERR_INVALID, "cross entropy: negative size");
    if (reduction != YUF_LOSS_NONE && reduction != YUF_LOSS_MEAN && reduction != YUF_LOSS_SUM)
        return fail(YUF_ERR_INVALID, "cross entropy: reduction must be YUF_LOSS_NONE, _MEAN or _SUM");
    if (target_bits != 32 && target_bits != 64) return fail(YUF_ERR_INVALID, "cross entropy: target_bits must be 32 or 64");
    if (ld < V || (dlogits && ld_out < V)) return fail(YUF_ERR_INVALID, "cross entropy: row stride below V");
    if (V > 1 << 30) return fail(YUF_ERR_INVALID, "cross entropy: V above 2^30");
    if (M > 0 && V == 0) return fail(YUF_ERR_INVALID, "cross entropy: rows without logits");
    if (M > 0 && (!logits || !targets)) return fail(YUF_ERR_INVALID, "cross entropy: null logits or targets");
    if (!loss && M == 0) return YUF_OK;  // the gradient of no rows, whose pointer may well be null
    if (!loss && !dlogits) return fail(YUF_ERR_INVALID, "cross entropy: neither a loss nor a gradient asked for");
    if (dlogits == logits && dlogits && ld_out != ld)
        return fail(YUF_ERR_INVALID, "cross entropy: a gradient in place of the logits has their row stride");
    if (dlogits && dlogits != logits && M > 0 && rows_overlap(M, V * sizeof(T), logits, ld * sizeof(T), dlogits, ld_out * sizeof(T)))
        return fail(YUF_ERR_INVALID, "cross entropy: the gradient may take the logits' place, but not overlap them otherwise");
    const bool reduced = reduction != YUF_LOSS_NONE;
    if (reduced && !workspace) return fail(YUF_ERR_INVALID, "cross entropy: mean and sum need the workspace");
    hipStream_t s = static_cast<hipStream_t>(stream);
    LossParams p{};
    p.M = M; p.V = V; p.logits = logits; p.ld = ld;
    p.targets = targets; p.wide = target_bits == 64; p.ignore = ignore;
    p.reduction = reduction;
    p.row_loss = loss ? (reduced ? workspace + 1 : loss) : nullptr;
    p.dloss = dloss; p.dlogits = dlogits; p.ld_out = ld_out;
    // A mean's gradient needs the number of rows before any is written.
    if (reduction == YUF_LOSS_MEAN && M > kCountInline / row_waves(row_vecs<T>(V))) {
        hipLaunchKernelGGL(loss_count_kernel, dim3(1), dim3(kReduceThreads), 0, s, p, workspace);
        p.count = workspace;
    }
    if (M > 0) launch_rows<T>(p, s);
    if (loss && reduced) hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(kReduceThreads), 0, s, p, loss);
    YUF_LAUNCH_CHECK("cross entropy");
    return YUF_OK;
}

}  // namespace
}  // namespace yuf

extern "C" size_t yuf_cross_entropy_workspace(int M) { return M < 0 ? 0 : ((size_t)M + 1) * sizeof(float); }

extern "C" int yuf_cross_entropy_f32(int M, int V, const float *logits, int64_t ld, const void *targets, int target_bits,
                                     int64_t ignore_index, int reduction, float *loss, const float *dloss,
                                     float *dlogits, int64_t ld_out, void *workspace, void *stream) {
    return yuf::cross_entropy<float>(M, V, logits, ld, targets, target_bits, ignore_index, reduction, loss, dloss,
                                     dlogits, ld_out, static_cast<float *>(workspace), stream);
}

extern "C" int yuf_cross_entropy_bf16(int M, int V, const uint16_t *logits, int64_t ld, const void *targets,
                                      int target_bits, int64_t ignore_index, int reduction, float *loss,
                                      const float *dloss, uint16_t *dlogits, int64_t ld_out, void *workspace,
                                      void *stream) {
    return yuf::cross_entropy<uint16_t>(M, V, logits, ld, targets, target_bits, ignore_index, reduction, loss, dloss,
                                        dlogits, ld_out, static_cast<float *>(workspace), stream);
}
