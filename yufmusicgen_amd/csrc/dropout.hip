// Dropout with a mask that is generated, not stored:
//     out_i = keep_i ? x_i / (1 - p) : 0   (+ residual_i)
// keep_i is a function of (seed, counter, i) alone, so the gradient regenerates the
// mask of the forward pass: dx = the same operator on dout without the residual.
//
// The generator is Philox 4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011): one 128-bit counter
// (i / 4, counter) under a 64-bit key gives four 32-bit words, one per element,
// and an element is dropped where its word is below p 2^32.
//
// Bound: memory, 8 or 12 bytes an element in fp32 (half of it in bf16).  Philox costs
// 20 32 x 32 -> 64-bit products per four elements.  A thread handles kUnits groups
// of a 16-byte vector, all loads issued before the first product.  16384 x 640 fp32
// with the residual: 19.0 us = 6.6 TB/s, as long as an addition of the two tensors
// (they fit the memory-side cache).  In bf16 the products are twice as many per byte and bound it:
// 14.8 us with the residual, 12.4 without (an addition: 10.1).
#include "common.h"

#include <cmath>

namespace yuf {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // 16-byte vectors of a thread

// Vectors with the alignment of their elements: tensors may start at any element.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8_u __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ void philox(uint64_t index, uint64_t counter, uint64_t seed, uint32_t (&c)[4]) {
    c[0] = (uint32_t)index; c[1] = (uint32_t)(index >> 32);
    c[2] = (uint32_t)counter; c[3] = (uint32_t)(counter >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

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

template <typename T> struct DropoutParams {
    int64_t n;
    const T *x, *residual;
    T *out;
    uint64_t seed, counter;
    const uint64_t *counter_dev;
    uint32_t threshold;  // a word below it drops its element
    bool keep_none;      // p = 1
    float scale;         // 1 / (1 - p)
};

template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(DropoutParams<T> p) {
    constexpr int kN = Vec<T>::kN;
    using V = typename Vec<T>::type;
    const uint64_t counter = p.counter + (p.counter_dev ? *p.counter_dev : 0);
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kUnits) + threadIdx.x;
    V x[kUnits], r[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = (first + u * kThreads) * kN;
        if (at + kN <= p.n) {
            x[u] = *reinterpret_cast<const V *>(p.x + at);
            if (p.residual) r[u] = *reinterpret_cast<const V *>(p.residual + at);
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                x[u][e] = at + e < p.n ? p.x[at + e] : T(0);
                r[u][e] = p.residual && at + e < p.n ? p.residual[at + e] : T(0);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = (first + u * kThreads) * kN;
        if (at >= p.n) break;
        V o;
#pragma unroll
        for (int e = 0; e < kN; e += 4) {
            uint32_t word[4];
            philox((uint64_t)(at + e) >> 2, counter, p.seed, word);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // A dropped element is 0 whatever it holds (an infinity times 0 would not be).
                const bool keep = word[i] >= p.threshold && !p.keep_none;
                float y = keep ? widen(x[u][e + i]) * p.scale : 0.0f;
                if (p.residual) y += widen(r[u][e + i]);
                T t;
                narrow(y, t);
                o[e + i] = t;
            }
        }
        if (at + kN <= p.n) {
            *reinterpret_cast<V *>(p.out + at) = o;
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e)
                if (at + e < p.n) p.out[at + e] = o[e];
        }
    }
}

template <typename T>
int dropout(int64_t n, const T *x, const T *residual, double p, uint64_t seed, uint64_t counter,
            const uint64_t *counter_dev, T *out, void *stream) {
    if (n < 0) return fail(YUF_ERR_INVALID, "dropout: negative size");
    if (!(p >= 0.0 && p <= 1.0)) return fail(YUF_ERR_INVALID, "dropout: p must be in [0, 1]");
    if (n == 0) return YUF_OK;
    if (!x || !out) return fail(YUF_ERR_INVALID, "dropout: null input/output pointer");
    // A thread reads its elements, and no others, before it writes them.
    const Span to{out, (size_t)n * sizeof(T)};
    for (const T *from : {x, residual})
        if (from != out && overlap({from, to.bytes}, to))
            return fail(YUF_ERR_INVALID, "dropout: out may be x or residual, but not a part of them");
    constexpr int64_t kPerBlock = (int64_t)kThreads * kUnits * Vec<T>::kN;
    const int64_t blocks = (n + kPerBlock - 1) / kPerBlock;
    if (blocks * kThreads >= (int64_t)1 << 32) return fail(YUF_ERR_INVALID, "dropout: too many elements");  // threads of a launch
    DropoutParams<T> q{};
    q.n = n; q.x = x; q.residual = residual; q.out = out;
    q.seed = seed; q.counter = counter; q.counter_dev = counter_dev;
    q.keep_none = p >= 1.0;
    q.threshold = q.keep_none ? 0u : (uint32_t)(p * 4294967296.0);
    q.scale = q.keep_none ? 0.0f : (float)(1.0 / (1.0 - p));
    hipLaunchKernelGGL((dropout_kernel<T>), dim3((uint32_t)blocks), dim3(kThreads), 0, static_cast<hipStream_t>(stream), q);
    YUF_LAUNCH_CHECK("dropout");
    return YUF_OK;
}

}  // namespace
}  // namespace yuf

extern "C" int yuf_dropout_f32(int64_t n, const float *x, const float *residual, double p, uint64_t seed,
                               uint64_t counter, const uint64_t *counter_dev, float *out, void *stream) {
    return yuf::dropout<float>(n, x, residual, p, seed, counter, counter_dev, out, stream);
}

extern "C" int yuf_dropout_bf16(int64_t n, const uint16_t *x, const uint16_t *residual, double p, uint64_t seed,
                                uint64_t counter, const uint64_t *counter_dev, uint16_t *out, void *stream) {
    return yuf::dropout<uint16_t>(n, x, residual, p, seed, counter, counter_dev, out, stream);
}
