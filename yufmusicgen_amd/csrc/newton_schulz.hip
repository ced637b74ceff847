// Orthogonalising matrices by Newton-Schulz products, and the weight update around it:
//     X <- x / (|x|_F + eps);   `steps` times:  A = X X^T,  X <- a X + (b A + c A A) X,
// of the transpose where x has more rows than columns (p: the smaller side, q: the larger).
//
// Bound: the matrix cores.  Per step p^2 q + p^3 + 2 p^2 q operations, since A and A A are symmetric: only
// tiles on and above the diagonal are multiplied, and each is written to both its places.
//
// Operands are fp16 pairs.  A value v scaled by a power of two is held as hi = fp16(v), lo = fp16(v - hi),
// |v - hi - lo| <= 2^-22 |v|.  The scale of each matrix follows from a bound of its singular values (X starts
// with a Frobenius norm of 1, and the polynomial's largest value bounds each next step), which bounds its elements, so
// nothing overflows and what is lost below fp16's subnormals is under 2^-38 of the bound.
// A product of two is three of theirs, hi hi + hi lo + lo hi (the one left out is below 2^-22): the polynomial amplifies what
// a step's rounding adds, along small singular values by up to a each step and near 1 by slopes of up to 4, and by how much
// in all depends on the matrix (2-norm errors of 640 x 640: 1.8e-6; of fp32 products 2.9e-6).  bf16 matrices take the
// same: hi hi alone, 11 bits, is enough for many noisy directions (2e-4, against the 3.9e-3 of the output's half step), but was
// off by 6e-3 for 333 equal singular values, 9.6e-3 for equal elements, 8.5e-2 with steeper coefficients, and no rule on
// sizes, steps and coefficients tells these apart.
//
// Layout: every operand lies in 1 KB blocks of 16 rows x 32 k in the order in which the lanes of
// v_mfma_f32_16x16x32_f16 hold them (lane l: row l % 16, k = 8 (l / 16) + j), hi blocks and then lo blocks.
// Blocks go from memory to LDS as they lie, and from LDS to registers without bank conflicts.  X is kept as X^T
// (rows of q, k over p), as P X takes it; X X^T, which runs over q, reads the same blocks from LDS transposed.
// (Keeping X both ways would write it twice.)
//
// Five steps of 56 x 640 x 640 fp32: X X^T 68 us, A A 63, P X 91 a step = 780, 840 and 960 TFLOP/s of multiplied tiles;
// the whole update 1.22 ms.  24 x 1024 x 4096 bf16: 332, 88, 514 us a step, 1050, 990 and 1200 TFLOP/s, 5.2 ms (a
// large fp16 matrix product of the same card: 1.2 to 1.3 PFLOP/s).  What bounds the former is their operands' way into
// LDS: without those loads X X^T takes 51 us and P X 60.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

namespace yuf {
namespace {

typedef _Float16 f16;
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kXcds = 8;
constexpr int kGroup = 64;      // matrices of a launch: their pointers are kernel arguments
constexpr size_t kSpaceMost = (size_t)2 << 30;  // bytes of a group's operands, if it is more than one matrix
constexpr int kSumParts = 64;   // workgroups of a matrix's norm, at most
constexpr int kSumRun = 4096;   // elements of such a workgroup, at least
constexpr int kPrepTile = 64;
constexpr int kStepsMost = 64;
constexpr double kGrowthMost = 256.0;  // of the singular values' bound
constexpr double kPolyMost = 1e6;      // of P's; no polynomial with the former bound comes near it
constexpr double kBelow = 30000.0;     // scaled values stay below this (fp16 holds 65504)

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ void narrow(float x, float &out) { out = x; }
__device__ __forceinline__ void narrow(float x, uint16_t &out) {
    // Round to nearest even; NaN stays a (quiet) NaN.
    const uint32_t u = __float_as_uint(x);
    out = x != x ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// The matrices of a launch.  update: x are gradients, m momenta, out the weights; else out the results.
template <typename T> struct Matrices {
    const T *x[kGroup];
    float *m[kGroup];
    T *out[kGroup];
    int count, rows, cols;
    bool update, nesterov;
    float beta, rest;    // of the momentum: m <- beta m + rest g
    float keep, rate;    // out <- keep out - rate X
};

// For each step, the scales of X, A and P: powers of two.
struct Scales {
    float x[kStepsMost + 1], gram[kStepsMost], poly[kStepsMost];
};

// The value that is orthogonalised, from its gradient and the updated momentum.
template <typename T>
__device__ __forceinline__ float direction(const Matrices<T> &t, float g, float m) {
    return t.nesterov ? fmaf(t.beta, m, t.rest * g) : m;
}

// Four elements of which `count` exist, with the alignment of one.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { using type = f32x4_u; };
template <> struct Vec4<uint16_t> { using type = u16x4_u; };
template <typename T> __device__ __forceinline__ void load4(const T *from, int count, float (&x)[4]) {
    if (count >= 4) {
        const auto v = *reinterpret_cast<const typename Vec4<T>::type *>(from);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = widen(v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = e < count ? widen(from[e]) : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void store4(T *to, int count, const float (&x)[4]) {
    typename Vec4<T>::type v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        T o;
        narrow(x[e], o);
        v[e] = o;
    }
    if (count >= 4) {
        *reinterpret_cast<typename Vec4<T>::type *>(to) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < count) to[e] = v[e];
    }
}

// ------------------------------------------------------------------- norm and momentum
template <typename T>
__global__ void __launch_bounds__(kThreads) ns_norm_kernel(Matrices<T> t, int parts, double *sums) {
    constexpr int kBatch = 4;  // vectors of a lane in flight
    __shared__ double waves[kThreads / kWave];
    const int matrix = blockIdx.y;
    const int64_t n = (int64_t)t.rows * t.cols, run = ((n + parts - 1) / parts + 3) / 4 * 4;
    const int64_t first = blockIdx.x * run, last = min(n, first + run);
    const T *x = t.x[matrix];
    float *m = t.update ? t.m[matrix] : nullptr;
    double sum = 0.0;
    for (int64_t i = first + threadIdx.x * 4; i < last; i += kBatch * kThreads * 4) {
        float v[kBatch][4], old[kBatch][4];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t at = i + u * kThreads * 4;
            load4(x + at, (int)min((int64_t)4, last - at), v[u]);
            if (m) load4(m + at, (int)min((int64_t)4, last - at), old[u]);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t at = i + u * kThreads * 4;
            if (m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    old[u][e] = fmaf(t.beta, old[u][e], t.rest * v[u][e]);
                    v[u][e] = direction(t, v[u][e], old[u][e]);
                }
                store4(m + at, (int)min((int64_t)4, last - at), old[u]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at + e < last) sum = fma((double)v[u][e], (double)v[u][e], sum);
        }
    }
    sum = wave_sum_f64(sum);
    if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / kWave; ++w) sum += waves[w];
        sums[(int64_t)matrix * parts + blockIdx.x] = sum;
    }
}

// -------------------------------------------------------------------- operand blocks
// Where element (row, k) of an operand of `kblocks` blocks along k lies.
__device__ __forceinline__ int64_t block_at(int row, int k, int kblocks) {
    return ((int64_t)(row >> 4) * kblocks + (k >> 5)) * 512 + ((((k & 31) >> 3) * 16 + (row & 15)) << 3) + (k & 7);
}

template <int N, typename V> __device__ __forceinline__ void split(const float (&x)[N], V &hi, V &lo) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        hi[e] = (f16)x[e];
        lo[e] = (f16)(x[e] - (float)hi[e]);
    }
}

// Transposing reads of the fragments of 16 N rows of each of two operands, 32 k.  A lane gives the address (in LDS) of
// four elements along the rows; lane t of a group of 16 gets element t of each run of four lanes' sixteen.  Blocks of
// 16 rows are 512 bytes apart, the second four k 64.  The wait is part of the block: the compiler, which knows
// of no loads in it, would let such reads by its builtin wait for every load into LDS that is on its way.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int N> __device__ __forceinline__ void read_transposed(uint32_t left, uint32_t right, f16x8 (&l)[N], f16x8 (&r)[N]) {
    static_assert(N == 2 || N == 4, "fragments of a wave");
    u32x2 x[4 * N];
    if constexpr (N == 2) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\t"
            "ds_read_b64_tr_b16 %1, %8 offset:64\n\t"
            "ds_read_b64_tr_b16 %2, %8 offset:512\n\t"
            "ds_read_b64_tr_b16 %3, %8 offset:576\n\t"
            "ds_read_b64_tr_b16 %4, %9\n\t"
            "ds_read_b64_tr_b16 %5, %9 offset:64\n\t"
            "ds_read_b64_tr_b16 %6, %9 offset:512\n\t"
            "ds_read_b64_tr_b16 %7, %9 offset:576\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
            : "v"(left), "v"(right)
            : "memory");
    } else {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %16\n\t"
            "ds_read_b64_tr_b16 %1, %16 offset:64\n\t"
            "ds_read_b64_tr_b16 %2, %16 offset:512\n\t"
            "ds_read_b64_tr_b16 %3, %16 offset:576\n\t"
            "ds_read_b64_tr_b16 %4, %16 offset:1024\n\t"
            "ds_read_b64_tr_b16 %5, %16 offset:1088\n\t"
            "ds_read_b64_tr_b16 %6, %16 offset:1536\n\t"
            "ds_read_b64_tr_b16 %7, %16 offset:1600\n\t"
            "ds_read_b64_tr_b16 %8, %17\n\t"
            "ds_read_b64_tr_b16 %9, %17 offset:64\n\t"
            "ds_read_b64_tr_b16 %10, %17 offset:512\n\t"
            "ds_read_b64_tr_b16 %11, %17 offset:576\n\t"
            "ds_read_b64_tr_b16 %12, %17 offset:1024\n\t"
            "ds_read_b64_tr_b16 %13, %17 offset:1088\n\t"
            "ds_read_b64_tr_b16 %14, %17 offset:1536\n\t"
            "ds_read_b64_tr_b16 %15, %17 offset:1600\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]),
              "=&v"(x[8]), "=&v"(x[9]), "=&v"(x[10]), "=&v"(x[11]), "=&v"(x[12]), "=&v"(x[13]), "=&v"(x[14]), "=&v"(x[15])
            : "v"(left), "v"(right)
            : "memory");
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        l[i] = __builtin_shufflevector(__builtin_bit_cast(f16x4, x[2 * i]), __builtin_bit_cast(f16x4, x[2 * i + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
        r[i] = __builtin_shufflevector(__builtin_bit_cast(f16x4, x[2 * N + 2 * i]), __builtin_bit_cast(f16x4, x[2 * N + 2 * i + 1]), 0, 1, 2, 3,
                                       4, 5, 6, 7);
    }
}

struct Buffers {        // of one matrix, in f16 elements from its base
    int64_t xt[2], gram, poly, stride;
    int64_t long_plane, short_plane;  // lo blocks lie that far behind the hi blocks: of X^T, and of A and P
};

template <typename T>
__global__ void __launch_bounds__(kThreads) ns_prepare_kernel(Matrices<T> t, int parts, const double *sums, double eps,
                                                               float scale, f16 *space, Buffers b, int pp) {
    __shared__ float tile[kPrepTile][kPrepTile + 1];
    const int matrix = blockIdx.z, tid = threadIdx.x;
    const bool wide = t.rows <= t.cols;
    double sum = 0.0;
    for (int i = 0; i < parts; ++i) sum += sums[(int64_t)matrix * parts + i];
    const double factor = 1.0 / (sqrt(sum) + eps);
    const int r0 = (wide ? blockIdx.y : blockIdx.x) * kPrepTile, c0 = (wide ? blockIdx.x : blockIdx.y) * kPrepTile;
    const T *x = t.x[matrix];
    const float *m = t.update ? t.m[matrix] : nullptr;
    constexpr int kRows = kPrepTile * kPrepTile / kThreads / 4;
    float v[kRows][4], u[kRows][4];
    const int c = tid % (kPrepTile / 4) * 4;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = (tid / (kPrepTile / 4)) * kRows + i, count = r0 + r < t.rows ? t.cols - c0 - c : 0;
        const int64_t at = (int64_t)(r0 + r) * t.cols + c0 + c;
        load4(x + at, count, v[i]);
        if (m) load4(m + at, count, u[i]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (m) v[i][e] = direction(t, v[i][e], u[i][e]);
            tile[(tid / (kPrepTile / 4)) * kRows + i][c + e] = (float)(v[i][e] * factor) * scale;
        }
    __syncthreads();
    f16 *base = space + matrix * b.stride;
    const int i0 = blockIdx.y * kPrepTile, j0 = blockIdx.x * kPrepTile;  // of X
#pragma unroll
    for (int w = 0; w < kPrepTile * kPrepTile / 8 / kThreads; ++w) {
        const int chunk = w * kThreads + tid, lane = chunk % kWave, block = chunk / kWave;
        const int j = (block >> 1) * 16 + lane % 16, i = (block & 1) * 32 + lane / 16 * 8;
        float x8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x8[e] = wide ? tile[i + e][j] : tile[j][i + e];
        f16x8 hi, lo;
        split(x8, hi, lo);
        f16 *to = base + b.xt[0] + block_at(j0 + j, i0 + i, pp / 32);
        *reinterpret_cast<f16x8 *>(to) = hi;
        *reinterpret_cast<f16x8 *>(to + b.long_plane) = lo;
    }
}

// ---------------------------------------------------------------------------- products
enum { NS_GRAM, NS_POLY, NS_APPLY, NS_LAST };

template <typename T> struct Product {
    f16 *space;
    Buffers b;
    int pp, qp, xt;         // xt: which of the two X^T is read
    int tiles_m, tiles_n, total, per_xcd;
    float factor, linear, diagonal;  // value = factor sum, of P + linear A + diagonal on the diagonal
    Matrices<T> t;          // NS_LAST
};

// C = L R^T of one tile of TILE x TILE; L and R rows of K in blocks.  Four waves have a quarter of the tile each.  A
// stage holds one k block, ST stages lie in LDS; the loads of the stage that is ST - 1 ahead are issued between the
// products of the present one, a few at a time.
template <typename T, int MODE, int TILE, int ST>
__global__ void __launch_bounds__(kThreads, 2) ns_product_kernel(Product<T> p) {
    constexpr int NW = kThreads / kWave;
    constexpr int RB = TILE / 16;             // row blocks of an operand
    constexpr int HB = RB * 2;                // blocks of a stage, hi and lo: L's, then R's
    constexpr int PER = 2 * HB / NW;          // of a wave
    constexpr int MI = RB / 2;                // 16 x 16 blocks of a wave along each side
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    static_assert(HB % NW == 0 && MI % 2 == 0, "shares of a wave");
    constexpr int kStages = ST * 2 * HB * 512;
    __shared__ __attribute__((aligned(1024))) f16 lds[kStages];

    const int flat = (blockIdx.x % kXcds) * p.per_xcd + blockIdx.x / kXcds;  // a matrix's tiles on one XCD
    if (flat >= p.total) return;
    int matrix, bm, bn;
    if (SYM) {
        const int tiles = p.tiles_m * (p.tiles_m + 1) / 2;
        matrix = flat / tiles;
        int rest = flat - matrix * tiles;
        for (bm = 0; rest >= p.tiles_m - bm; ++bm) rest -= p.tiles_m - bm;
        bn = bm + rest;
    } else {
        const int tiles = p.tiles_m * p.tiles_n;
        matrix = flat / tiles;
        const int rest = flat - matrix * tiles;
        bn = rest / p.tiles_m;
        bm = rest - bn * p.tiles_m;
    }
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave >> 1, wn = wave & 1, g4 = lane >> 4, li = lane & 15;
    f16 *const base = p.space + (int64_t)matrix * p.b.stride;
    const Buffers &b = p.b;
    const int K = MODE == NS_GRAM ? p.qp : p.pp, KT = K / 32;
    const int64_t left = MODE == NS_GRAM ? b.xt[p.xt] : MODE == NS_POLY ? b.gram : b.poly;
    const int64_t right = SYM ? left : b.xt[p.xt];
    const int64_t plane_l = MODE == NS_GRAM ? b.long_plane : b.short_plane, plane_r = SYM ? plane_l : b.long_plane;
    const auto rl = make_rsrc(base + left, (uint32_t)(plane_l * 4)), rr = make_rsrc(base + right, (uint32_t)(plane_r * 4));

    uint32_t off[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int x = wave + NW * i, of_r = x >= HB, at = x - of_r * HB;
        const int part = at / RB, tile = of_r ? bn : bm;
        int block;
        if (MODE == NS_GRAM) {  // [16 rows of X^T][32 of the tile's rows, which are k there]
            const int kr = at % RB / (RB / 2), ic = at % (RB / 2);
            block = kr * (p.pp / 32) + tile * (RB / 2) + ic;
        } else {  // a row block
            block = (tile * RB + at % RB) * (K / 32);
        }
        off[i] = (uint32_t)(block * 1024 + part * (int)((of_r ? plane_r : plane_l) * 2) + lane * 16);
    }
    const int step = MODE == NS_GRAM ? 2 * (p.pp / 32) * 1024 : 1024;  // of a stage
    auto issue_one = [&](int i, int kt, int buf) {
        lds_void_t *dst = (lds_void_t *)(lds + (buf * 2 * HB + wave + NW * i) * 512);
        const uint32_t o = off[i];
        // NW divides HB: a load is of one operand for every wave.
        if (NW * i < HB) __builtin_amdgcn_raw_ptr_buffer_load_lds(rl, dst, 16, o, kt * step, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(rr, dst, 16, o, kt * step, 0, 0);
    };
    auto issue = [&](int kt, int buf) {
#pragma unroll
        for (int i = 0; i < PER; ++i) issue_one(i, kt, buf);
    };
    auto arrive = [&](bool all, auto stages) {
        constexpr int n = decltype(stages)::value;
        if (all) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(n * PER) : "memory");
    };

    // Where a lane's transposing reads begin in a k block of 32 rows of X^T: for group g4 at k = 8 g4 + li / 4, four
    // of its 16 rows' elements from 4 (li % 4) on.
    const auto turned = [&](int part, int m) {
        const int block = (part * 2 + (g4 >> 1)) * (RB / 2) + m / 2;
        return block * 512 + li % 4 / 2 * 128 + ((g4 & 1) * 8 + li / 4) * 8 + li % 2 * 4;
    };
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_void_t *)lds;

    // The products with a low part are summed apart: a third of the roundings in the large sum.
    floatx4 acc[MI][MI], low[MI][MI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] = low[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
        if (s < KT) issue(s, s);
    int buf = 0;
    const auto multiply = [&](int kt, auto loads) {
        constexpr bool kLoads = decltype(loads)::value;
        // Stage kt is in LDS for every wave, and every wave has read stage kt - 1.
        arrive(kt + ST - 1 > KT, std::integral_constant<int, ST - 2>{});
        const f16 *const l = lds + buf * 2 * HB * 512, *const r = l + HB * 512;
        f16x8 fl[2][MI], fr[2][MI];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if constexpr (MODE == NS_GRAM) {
                const uint32_t at = lds_at + buf * 2 * HB * 1024;
                read_transposed<MI>(at + turned(q, wm * MI) * 2, at + HB * 1024 + turned(q, wn * MI) * 2, fl[q], fr[q]);
            } else {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    fl[q][i] = *reinterpret_cast<const f16x8 *>(l + (q * RB + wm * MI + i) * 512 + lane * 8);
                    fr[q][i] = *reinterpret_cast<const f16x8 *>(r + (q * RB + wn * MI + i) * 512 + lane * 8);
                }
            }
        }
        // The next loads go between the products: a wave that issues its loads one after the other waits for about 80
        // cycles each, in which it multiplies nothing.
        const int target = buf == 0 ? ST - 1 : buf - 1;
        constexpr int kProducts = 3 * MI * MI, kEvery = kProducts / PER;
        static_assert(kProducts % PER == 0, "products between loads");
#pragma unroll
        for (int n = 0; n < kProducts; ++n) {
            if (kLoads && n % kEvery == 0) {
                __builtin_amdgcn_sched_barrier(0);
                issue_one(n / kEvery, kt + ST - 1, target);
                __builtin_amdgcn_sched_barrier(0);
            }
            const int q = n / (MI * MI), i = n / MI % MI, j = n % MI;  // hi hi, lo hi, hi lo
            floatx4 &sum = q == 0 ? acc[i][j] : low[i][j];
            sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl[q == 1][i], fr[q == 2][j], sum, 0, 0, 0);
        }
        buf = buf == ST - 1 ? 0 : buf + 1;
    };
    int kt = 0;
    for (; kt < KT - (ST - 1); ++kt) multiply(kt, std::true_type{});
    for (; kt < KT; ++kt) multiply(kt, std::false_type{});
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) acc[i][j] += low[i][j];
    // Lane (g4, li) holds rows 4 g4 + r and column li of block (i, j).  As rows of an operand the tile's columns' four
    // elements are neighbours: at a wave's block of 16 columns x 32 rows and at `mine` in it.
    const int row0 = (bm * RB + wm * MI) * 16, col0 = (bn * RB + wn * MI) * 16;
    const int kblocks = p.pp / 32;
    const int mine = (g4 >> 1) * 128 + li * 8 + (g4 & 1) * 4;
    const auto turned_block = [&](int i, int j) { return ((col0 / 16 + j) * kblocks + row0 / 32 + i / 2) * 512 + i % 2 * 256; };
    const int64_t plane = SYM ? b.short_plane : b.long_plane;
    const float factor = p.factor, linear = p.linear, diagonal = p.diagonal;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            acc[i][j] *= factor;
            if (MODE == NS_POLY) {
                const f16 *at = base + b.gram + turned_block(i, j) + mine;  // A, which is symmetric
                const f16x4 hi = *reinterpret_cast<const f16x4 *>(at), lo = *reinterpret_cast<const f16x4 *>(at + plane);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    acc[i][j][r] = fmaf(linear, (float)hi[r] + (float)lo[r], acc[i][j][r]);
                    if (row0 + i * 16 + 4 * g4 + r == col0 + j * 16 + li) acc[i][j][r] += diagonal;
                }
            }
        }
    }
    if constexpr (MODE == NS_LAST) {
        // Through wave-private LDS, 16 lines of the output at a time, so that they are read and written in long runs.
        const Matrices<T> &t = p.t;
        T *const out = t.out[matrix];
        const int lines = t.rows, cols = t.cols;
        const bool wide = t.rows <= t.cols, update = t.update;
        const float keep = t.keep, rate = t.rate;
        // Lane `lane` has four columns of every kLines-th line, of the 16 lines of each of kParts parts.
        const auto finish = [&](auto run, auto parts, int line0, int at0, auto &&fill) {
            constexpr int kRun = decltype(run)::value, kParts = decltype(parts)::value, kPitch = kRun + 4;
            constexpr int kLanes = kRun / 4, kLines = kWave / kLanes, kEach = 16 / kLines;
            static_assert(NW * 16 * kPitch * 2 <= kStages, "the lines fit the stages' LDS");
            float *const stage = reinterpret_cast<float *>(lds) + wave * 16 * kPitch;
            const int line = lane / kLanes, at = lane % kLanes * 4;
            float old[kParts][kEach][4];  // loaded before the first is waited for
            if (update) {
#pragma unroll
                for (int part = 0; part < kParts; ++part)
#pragma unroll
                    for (int u = 0; u < kEach; ++u) {
                        const int row = line0 + part * 16 + u * kLines + line;
                        load4(out + (int64_t)row * cols + at0 + at, row < lines ? cols - at0 - at : 0, old[part][u]);
                    }
            }
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                fill(part, stage, kPitch);
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
#pragma unroll
                for (int u = 0; u < kEach; ++u) {
                    const int row = line0 + part * 16 + u * kLines + line;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = stage[(u * kLines + line) * kPitch + at + e];
                        if (update) v[e] = fmaf(keep, old[part][u][e], -rate * v[e]);
                    }
                    store4(out + (int64_t)row * cols + at0 + at, row < lines ? cols - at0 - at : 0, v);
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            }
        };
        lds_barrier();  // every wave has read its last stage, and what it was given
        if (wide) {
            finish(std::integral_constant<int, MI * 16>{}, std::integral_constant<int, MI>{}, row0, col0, [&](int i, float *stage, int pitch) {
#pragma unroll
                for (int j = 0; j < MI; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) stage[(4 * g4 + r) * pitch + j * 16 + li] = acc[i][j][r];
            });
        } else {  // lines of the output are columns here
            finish(std::integral_constant<int, MI * 16>{}, std::integral_constant<int, MI>{}, col0, row0, [&](int j, float *stage, int pitch) {
#pragma unroll
                for (int i = 0; i < MI; ++i) *reinterpret_cast<floatx4 *>(stage + li * pitch + i * 16 + 4 * g4) = acc[i][j];
            });
        }
        return;
    }
    // Blocks of rows that are the tile's columns, straight from the registers.
    f16 *const to = base + (MODE == NS_GRAM ? b.gram : MODE == NS_POLY ? b.poly : b.xt[p.xt ^ 1]);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r];
            f16x4 hi, lo;
            split(v, hi, lo);
            f16 *at = to + turned_block(i, j);
            *reinterpret_cast<f16x4 *>(at + mine) = hi;
            *reinterpret_cast<f16x4 *>(at + plane + mine) = lo;
        }
    if (!SYM || bm == bn) return;
    // The mirrored tile's blocks, through wave-private LDS.
    lds_barrier();  // every wave has read its last stage
    constexpr int kPitch = 36;
    float *const stage = reinterpret_cast<float *>(lds) + wave * 16 * kPitch;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < MI; j += 2) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) stage[(4 * g4 + r) * kPitch + x * 16 + li] = acc[i][j + x][r];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = stage[li * kPitch + g4 * 8 + e];
            f16x8 hi, lo;
            split(v, hi, lo);
            f16 *at = to + ((row0 / 16 + i) * kblocks + col0 / 32 + j / 2) * 512;
            *reinterpret_cast<f16x8 *>(at + lane * 8) = hi;
            *reinterpret_cast<f16x8 *>(at + plane + lane * 8) = lo;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        }
}

// ------------------------------------------------------------------------- small matrices
// Matrices of up to 64 rows (the smaller side) and 768 columns as one workgroup each, from the norm to the result: a
// step's three products depend on each other, and as launches of their own each is mostly waiting (640 x 64 fp32: 78 us as
// launches, 62 here; 91 with X in memory).  A wave owns every kSmallWaves-th block of 32 columns of X and keeps it in
// registers, in fp32 and in the accumulators' order; it turns a block into operands through its own part of LDS.  X X^T
// is summed over the waves in order; A and P lie in LDS.
constexpr int kSmallWaves = 8, kSmallRows = 64, kSmallBlocks = 3;  // blocks of a wave
constexpr int kSmallThreads = kSmallWaves * kWave, kSmallColumns = kSmallBlocks * kSmallWaves * 32;
constexpr int kUpper = 10;  // 16 x 16 blocks of A on and above the diagonal: (i, j) is block j (j + 1) / 2 + i

template <typename T, int BLOCKS>
__global__ void __launch_bounds__(kSmallThreads, 2) ns_small_kernel(Matrices<T> t, Scales scales, int steps, float a, float b, float c,
                                                                     double eps) {
    constexpr int KB = kSmallRows / 32, MI = kSmallRows / 16;  // k blocks and row blocks of A and P
    constexpr int kPlane = kSmallRows * kSmallRows;            // f16 of a part of A or P
    constexpr int kPitch = 36;                                 // floats of a row of a block in LDS
    __shared__ __attribute__((aligned(1024))) f16 gram[2 * kPlane], poly[2 * kPlane];
    __shared__ __attribute__((aligned(16))) floatx4 sums[kSmallWaves][kUpper][kWave];
    __shared__ double norms[kSmallWaves];
    static_assert(sizeof(sums[0]) >= kSmallRows * kPitch * sizeof(float), "a wave's sums' place holds a block");
    const int matrix = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int g4 = lane >> 4, li = lane & 15;
    const bool wide = t.rows <= t.cols, update = t.update;
    const int P = min(t.rows, t.cols), Q = max(t.rows, t.cols), cols = t.cols;
    const T *const x = t.x[matrix];
    float *const m = update ? t.m[matrix] : nullptr;
    // Elements (row + r, col), r < 4, of X: a lane's are rows 16 i + 4 g4 + r and columns 32 block + 16 j + li.  In a
    // matrix of more rows than columns they are neighbours.
    const auto fetch = [&](const auto *from, int row, int col, float (&v)[4]) {
        if (!wide) return load4(from + (int64_t)col * cols + row, col < Q ? P - row : 0, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = row + r < P && col < Q ? widen(from[(int64_t)(row + r) * cols + col]) : 0.0f;
    };
    const auto keep = [&](auto *to, int row, int col, const float (&v)[4]) {
        using E = std::remove_reference_t<decltype(*to)>;
        if (!wide) return store4<E>(to + (int64_t)col * cols + row, col < Q ? P - row : 0, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            E o;
            narrow(v[r], o);
            if (row + r < P && col < Q) to[(int64_t)(row + r) * cols + col] = o;
        }
    };
    floatx4 X[BLOCKS][MI][2];
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < BLOCKS; ++w)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = i * 16 + 4 * g4, col = (wave + w * kSmallWaves) * 32 + j * 16 + li;
                float v[4];
                fetch(x, row, col, v);
                if (update) {
                    float moved[4];
                    fetch(m, row, col, moved);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        moved[r] = fmaf(t.beta, moved[r], t.rest * v[r]);
                        v[r] = direction(t, v[r], moved[r]);
                    }
                    keep(m, row, col, moved);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    sum = fma((double)v[r], (double)v[r], sum);
                    X[w][i][j][r] = v[r];
                }
            }
    sum = wave_sum_f64(sum);
    if (lane == 0) norms[wave] = sum;
    __syncthreads();
    sum = norms[0];
    for (int w = 1; w < kSmallWaves; ++w) sum += norms[w];
    const double factor = 1.0 / (sqrt(sum) + eps);
#pragma unroll
    for (int w = 0; w < BLOCKS; ++w)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {  // beyond the matrix 0, also where the factor is infinite
                    const bool in = i * 16 + 4 * g4 + r < P && (wave + w * kSmallWaves) * 32 + j * 16 + li < Q;
                    X[w][i][j][r] = in ? (float)(X[w][i][j][r] * factor) * scales.x[0] : 0.0f;
                }
    float *const stage = reinterpret_cast<float *>(sums[wave]);
    const auto fence = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };
    const auto lay = [&](const floatx4 (&block)[MI][2]) {
        fence();
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) stage[(i * 16 + 4 * g4 + r) * kPitch + j * 16 + li] = block[i][j][r];
        fence();
    };
    // Writes block (i, j) of a symmetric matrix into both its places in LDS.
    const auto put = [&](f16 *to, int i, int j, const floatx4 &value) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = value[r];
        f16x4 hi, lo;
        split(v, hi, lo);
        const int row = i * 16 + 4 * g4, col = j * 16 + li;
        f16 *at = to + block_at(col, row, KB);
        *reinterpret_cast<f16x4 *>(at) = hi;
        *reinterpret_cast<f16x4 *>(at + kPlane) = lo;
        if (i == j) return;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            to[block_at(row + r, col, KB)] = hi[r];
            to[block_at(row + r, col, KB) + kPlane] = lo[r];
        }
    };
    const auto of = [&](int block, int &i, int &j) {  // block -> (i, j)
        j = block >= 6 ? 3 : block >= 3 ? 2 : block >= 1 ? 1 : 0;
        i = block - j * (j + 1) / 2;
    };
    const auto mfma3 = [](const f16x8 &lh, const f16x8 &ll, const f16x8 &rh, const f16x8 &rl, floatx4 &high, floatx4 &low) {
        high = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rh, high, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(ll, rh, low, 0, 0, 0);
        low = __builtin_amdgcn_mfma_f32_16x16x32_f16(lh, rl, low, 0, 0, 0);
    };
    for (int step = 0; step < steps; ++step) {
        const float sx = scales.x[step], sa = scales.gram[step], sp = scales.poly[step], next = scales.x[step + 1];
        {
            floatx4 high[kUpper], low[kUpper];
#pragma unroll
            for (int u = 0; u < kUpper; ++u) high[u] = low[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < BLOCKS; ++w) {
                lay(X[w]);
                f16x8 f[2][MI];
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = stage[(i * 16 + li) * kPitch + g4 * 8 + e];
                    split(v, f[0][i], f[1][i]);
                }
#pragma unroll
                for (int j = 0; j < MI; ++j)
#pragma unroll
                    for (int i = 0; i <= j; ++i)
                        mfma3(f[0][i], f[1][i], f[0][j], f[1][j], high[j * (j + 1) / 2 + i], low[j * (j + 1) / 2 + i]);
            }
            fence();
#pragma unroll
            for (int u = 0; u < kUpper; ++u) sums[wave][u][lane] = high[u] + low[u];
        }
        __syncthreads();
        for (int u = wave; u < kUpper; u += kSmallWaves) {
            floatx4 v = sums[0][u][lane];
            for (int w = 1; w < kSmallWaves; ++w) v += sums[w][u][lane];
            int i, j;
            of(u, i, j);
            put(gram, i, j, v * (sa / (sx * sx)));
        }
        __syncthreads();
        for (int u = wave; u < kUpper; u += kSmallWaves) {
            int i, j;
            of(u, i, j);
            floatx4 high{0.f, 0.f, 0.f, 0.f}, low{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                const f16 *l = gram + (i * KB + k) * 512 + lane * 8, *r = gram + (j * KB + k) * 512 + lane * 8;
                mfma3(*reinterpret_cast<const f16x8 *>(l), *reinterpret_cast<const f16x8 *>(l + kPlane), *reinterpret_cast<const f16x8 *>(r),
                      *reinterpret_cast<const f16x8 *>(r + kPlane), high, low);
            }
            const f16 *at = gram + block_at(j * 16 + li, i * 16 + 4 * g4, KB);  // A, which is symmetric
            floatx4 v = (high + low) * (c * (sp / (sa * sa)));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = fmaf(b * (sp / sa), (float)at[r] + (float)at[kPlane + r], v[r]);
                if (i == j && 4 * g4 + r == li) v[r] += a * sp;
            }
            put(poly, i, j, v);
        }
        __syncthreads();
        const float scale = next / (sp * sx);
#pragma unroll
        for (int w = 0; w < BLOCKS; ++w) {
            lay(X[w]);
            f16x8 f[2][2][KB];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = stage[(k * 32 + g4 * 8 + e) * kPitch + j * 16 + li];
                    split(v, f[0][j][k], f[1][j][k]);
                }
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                floatx4 high[2], low[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) high[j] = low[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const f16 *l = poly + (i * KB + k) * 512 + lane * 8;
                    const f16x8 lh = *reinterpret_cast<const f16x8 *>(l), ll = *reinterpret_cast<const f16x8 *>(l + kPlane);
#pragma unroll
                    for (int j = 0; j < 2; ++j) mfma3(lh, ll, f[0][j][k], f[1][j][k], high[j], low[j]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) X[w][i][j] = (high[j] + low[j]) * scale;
            }
        }
    }
    int again = lane;  // its places are computed again: kept from the loads they would take registers all along
    asm volatile("" : "+v"(again));
#pragma unroll
    for (int w = 0; w < BLOCKS; ++w)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = i * 16 + 4 * (again >> 4), col = (wave + w * kSmallWaves) * 32 + j * 16 + (again & 15);
                float v[4], old[4];
                if (update) fetch(t.out[matrix], row, col, old);
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = update ? fmaf(t.keep, old[r], -t.rate * X[w][i][j][r]) : X[w][i][j][r];
                keep(t.out[matrix], row, col, v);
            }
}

// -------------------------------------------------------------------------------- host
struct Plan {
    int p, q, pp, qp, parts, group;
    bool whole;  // a workgroup for each matrix
    bool small_sym, small_apply;
    Buffers b;
    size_t sums, bytes;
};

int round_up(int x, int to) { return (x + to - 1) / to * to; }

// Tiles of 128 x 128 load least for their products; of 64 x 64 four times as many, which counts where 128 x 128 ones
// do not fill the card.  Launches in us, 128 and 64, by tiles of 128 x rows of the sum:
//   X X^T 210 x 640 24 and 21, 288 x 1024 38 and 43; A A 288 x 1024 41 and 37, 420 x 640 33 and 36;
//   P X 100 x 640 18 and 11, 350 x 640 26 and 28.
Plan ns_plan(int count, int rows, int cols) {
    Plan s{};
    s.p = std::min(rows, cols);
    s.q = std::max(rows, cols);
    // Operands in the padding of the larger tiles: two of X, and A and P, of two parts each.
    const size_t most = ((size_t)4 * round_up(s.p, 128) * round_up(s.q, 128) + (size_t)4 * round_up(s.p, 128) * round_up(s.p, 128)) * sizeof(f16);
    s.group = std::min({count, kGroup, (int)std::max<size_t>(1, std::min<size_t>(kGroup, kSpaceMost / most))});
    const int64_t tiles = (s.p + 127) / 128, sym = s.group * (tiles * (tiles + 1) / 2), apply = s.group * tiles * ((s.q + 127) / 128);
    s.whole = s.p <= kSmallRows && s.q <= kSmallColumns;
    s.small_sym = s.p <= 128 || sym <= 256;
    s.small_apply = s.p <= 128 || apply <= 200;
    const int unit = s.small_sym && s.small_apply ? 64 : 128;
    s.pp = round_up(s.p, unit);
    s.qp = round_up(s.q, unit);
    const int64_t n = (int64_t)rows * cols;
    s.parts = (int)std::min<int64_t>(kSumParts, (n + kSumRun - 1) / kSumRun);
    s.b.long_plane = (int64_t)s.pp * s.qp;
    s.b.short_plane = (int64_t)s.pp * s.pp;
    s.b.xt[0] = 0;
    s.b.xt[1] = 2 * s.b.long_plane;
    s.b.gram = 4 * s.b.long_plane;
    s.b.poly = s.b.gram + 2 * s.b.short_plane;
    s.b.stride = s.b.poly + 2 * s.b.short_plane;
    s.sums = (size_t)s.b.stride * sizeof(f16) * s.group;
    s.bytes = s.sums + (size_t)s.group * s.parts * sizeof(double);
    if (s.whole) s.bytes = 256;  // nothing
    return s;
}

const char *ns_refusal(int count, int rows, int cols) {
    if (count < 0 || rows < 0 || cols < 0) return "newton schulz: negative size";
    if (count == 0 || rows == 0 || cols == 0) return nullptr;
    // Offsets inside an operand are 32-bit: two parts of two bytes for each padded element.
    if (rows > 1 << 22 || cols > 1 << 22 || (int64_t)round_up(rows, 128) * round_up(cols, 128) > (int64_t)1 << 28)
        return "newton schulz: a matrix may have 2^28 elements, in sides padded to 128, and sides of 2^22";
    return nullptr;
}

// For each step, the scales of X, A and P, from a bound of X's singular values.
const char *ns_scales(int steps, double a, double b, double c, Scales &s) {
    const auto scale = [](double bound) {
        return (float)std::ldexp(1.0, std::min(40, (int)std::floor(std::log2(kBelow / std::max(bound, 1e-30)))));
    };
    double bound = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double top = bound * bound;  // of X's squared singular values
        // Extremes of a + b u + c u^2 and of t (a + b t^2 + c t^4) over the bound: ends and stationary points.
        double poly = std::max(std::fabs(a), std::fabs(a + b * top + c * top * top)), next = std::fabs(bound * (a + b * top + c * top * top));
        if (c != 0.0) {
            const double u = -b / (2 * c);
            if (u > 0 && u < top) poly = std::max(poly, std::fabs(a + b * u + c * u * u));
        }
        const double disc = 9 * b * b - 20 * a * c;
        if (disc >= 0) {
            // Both roots of 5 c u^2 + 3 b u + a, without cancellation.
            const double h = -0.5 * (3 * b + std::copysign(std::sqrt(disc), b));
            for (const double u : {c != 0 ? h / (5 * c) : -1.0, h != 0 ? a / h : -1.0})
                if (u > 0 && u < top) next = std::max(next, std::fabs(std::sqrt(u) * (a + b * u + c * u * u)));
        }
        if (!(next <= kGrowthMost) || !(poly <= kPolyMost)) return "newton schulz: these coefficients let singular values grow past 256";
        s.x[k] = scale(bound);
        s.gram[k] = scale(top);
        s.poly[k] = scale(poly);
        bound = next * (1.0 + 1e-3);  // rounding
    }
    s.x[steps] = 1.0f;
    return nullptr;
}

template <typename T, int MODE, int TILE, int ST> hipError_t launch_product(Product<T> &p, hipStream_t s) {
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    p.tiles_m = p.pp / TILE; p.tiles_n = SYM ? p.tiles_m : p.qp / TILE;
    p.total = p.t.count * (SYM ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n);
    p.per_xcd = ceil_div(p.total, kXcds);
    hipLaunchKernelGGL((ns_product_kernel<T, MODE, TILE, ST>), dim3(p.per_xcd * kXcds), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

// A product in the tiles that its plan names.  Small tiles take four stages: with few workgroups a CU each has to cover
// its own loads (X X^T of 4 x 640 x 640 fp32 10.3 us, of 1024 x 1024 12.8; two stages 14.2 and 20.3), and of many two
// workgroups a CU do as well as four (14 x 640 x 640 21.4 and 22.8).
template <typename T, int MODE> hipError_t launch_mode(const Plan &plan, Product<T> &p, hipStream_t s) {
    constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
    return (SYM ? plan.small_sym : plan.small_apply) ? launch_product<T, MODE, 64, 4>(p, s) : launch_product<T, MODE, 128, 2>(p, s);
}

template <typename T>
int ns_group(const Plan &plan, const Matrices<T> &t, const Scales &scales, int steps, float a, float b, float c, double eps,
             char *space, hipStream_t s) {
    double *sums = reinterpret_cast<double *>(space + plan.sums);
    f16 *halves = reinterpret_cast<f16 *>(space);
    if (plan.whole) {
        const int blocks = ceil_div(plan.q, 32 * kSmallWaves);  // of a wave
        const auto run = [&](auto n) {
            hipLaunchKernelGGL((ns_small_kernel<T, decltype(n)::value>), dim3(t.count), dim3(kSmallThreads), 0, s, t, scales, steps, a, b, c,
                               eps);
        };
        if (blocks == 1) run(std::integral_constant<int, 1>{});
        else if (blocks == 2) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, kSmallBlocks>{});
        YUF_LAUNCH_CHECK("newton schulz");
        return YUF_OK;
    }
    hipLaunchKernelGGL((ns_norm_kernel<T>), dim3(plan.parts, t.count), dim3(kThreads), 0, s, t, plan.parts, sums);
    hipLaunchKernelGGL((ns_prepare_kernel<T>), dim3(plan.qp / kPrepTile, plan.pp / kPrepTile, t.count), dim3(kThreads), 0, s, t,
                       plan.parts, sums, eps, scales.x[0], halves, plan.b, plan.pp);
    YUF_LAUNCH_CHECK("newton schulz");
    Product<T> p{};
    p.space = halves; p.b = plan.b; p.pp = plan.pp; p.qp = plan.qp; p.t = t;
    for (int k = 0; k < steps; ++k) {
        const float x = scales.x[k], gram = scales.gram[k], poly = scales.poly[k], next = scales.x[k + 1];
        p.xt = k & 1;
        p.factor = gram / (x * x);
        YUF_HIP_TRY((launch_mode<T, NS_GRAM>(plan, p, s)));
        p.factor = c * (poly / (gram * gram)); p.linear = b * (poly / gram); p.diagonal = a * poly;
        YUF_HIP_TRY((launch_mode<T, NS_POLY>(plan, p, s)));
        p.factor = next / (poly * x);
        if (k + 1 < steps) YUF_HIP_TRY((launch_mode<T, NS_APPLY>(plan, p, s)));
        else YUF_HIP_TRY((launch_mode<T, NS_LAST>(plan, p, s)));
    }
    return YUF_OK;
}

// Whether something that is written shares memory with anything else.  A matrix may be replaced by its result.
template <typename T>
const char *ns_overlap(int count, size_t n, const T *const *x, float *const *m, T *const *out, void *workspace, size_t bytes) {
    struct Run {
        uintptr_t begin, end;
        bool written;
    };
    std::vector<Run> runs;
    runs.reserve((size_t)count * 3 + 1);
    const auto add = [&](const void *p, size_t size, bool written) {
        runs.push_back({reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + size, written});
    };
    add(workspace, bytes, true);
    for (int i = 0; i < count; ++i) {
        if (!x[i] || !out[i] || (m && !m[i])) return "newton schulz: null matrix";
        if (m || x[i] != out[i]) add(x[i], n * sizeof(T), false);
        add(out[i], n * sizeof(T), true);
        if (m) add(m[i], n * sizeof(float), true);
    }
    std::sort(runs.begin(), runs.end(), [](const Run &a, const Run &b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;  // where the runs so far end
    for (const Run &r : runs) {
        if (r.begin < written || (r.written && r.begin < any)) return "newton schulz: matrices may not overlap each other or the workspace";
        any = std::max(any, r.end);
        if (r.written) written = std::max(written, r.end);
    }
    return nullptr;
}

template <typename T>
int newton_schulz(int count, int rows, int cols, const T *const *x, float *const *m, T *const *out, Matrices<T> t, int steps,
                  double a, double b, double c, double eps, void *workspace, void *stream) {
    if (const char *why = ns_refusal(count, rows, cols)) return fail(YUF_ERR_INVALID, why);
    if (steps < 1 || steps > kStepsMost) return fail(YUF_ERR_INVALID, "newton schulz: steps must be 1 to 64");
    if (!(eps >= 0.0) || !std::isfinite(eps)) return fail(YUF_ERR_INVALID, "newton schulz: eps must be finite and not negative");
    Scales scales{};
    if (const char *why = ns_scales(steps, a, b, c, scales)) return fail(YUF_ERR_INVALID, why);
    if (count == 0 || rows == 0 || cols == 0) return YUF_OK;
    if (!x || !out || (t.update && !m)) return fail(YUF_ERR_INVALID, "newton schulz: null list of matrices");
    if (!workspace || !scratch_aligned(workspace))
        return fail(YUF_ERR_INVALID, "newton schulz: the workspace must be given and 256-byte aligned");
    const Plan plan = ns_plan(count, rows, cols);
    try {
        if (const char *why = ns_overlap(count, (size_t)rows * cols, x, m, out, workspace, plan.bytes)) return fail(YUF_ERR_INVALID, why);
    } catch (const std::bad_alloc &) {
        return fail(YUF_ERR_OOM, "newton schulz: no host memory for the list of matrices");
    }
    t.rows = rows; t.cols = cols;
    for (int first = 0; first < count; first += plan.group) {
        t.count = std::min(plan.group, count - first);
        for (int i = 0; i < t.count; ++i) {
            t.x[i] = x[first + i];
            t.out[i] = out[first + i];
            t.m[i] = t.update ? m[first + i] : nullptr;
        }
        hipStream_t s = static_cast<hipStream_t>(stream);
        const int rc = ns_group<T>(plan, t, scales, steps, (float)a, (float)b, (float)c, eps, static_cast<char *>(workspace), s);
        if (rc != YUF_OK) return rc;
    }
    return YUF_OK;
}

template <typename T>
int muon_step(int count, int rows, int cols, const T *const *grads, float *const *momenta, T *const *params, double lr,
              double momentum, int nesterov, double weight_decay, int steps, double a, double b, double c, double eps,
              void *workspace, void *stream) {
    if (nesterov != 0 && nesterov != 1) return fail(YUF_ERR_INVALID, "muon step: nesterov must be 0 or 1");
    if (!std::isfinite(lr) || !std::isfinite(momentum) || !std::isfinite(weight_decay))
        return fail(YUF_ERR_INVALID, "muon step: lr, momentum and weight decay must be finite");
    Matrices<T> t{};
    t.update = true;
    t.nesterov = nesterov != 0;
    t.beta = (float)momentum; t.rest = (float)(1.0 - momentum);
    t.keep = (float)(1.0 - lr * weight_decay);
    t.rate = (float)(lr * std::sqrt(std::max(1.0, cols > 0 ? (double)rows / cols : 1.0)));
    return newton_schulz<T>(count, rows, cols, grads, momenta, params, t, steps, a, b, c, eps, workspace, stream);
}

}  // namespace
}  // namespace yuf

extern "C" size_t yuf_newton_schulz_workspace(int count, int rows, int cols) {
    if (yuf::ns_refusal(count, rows, cols) || count == 0 || rows == 0 || cols == 0) return 0;
    return yuf::ns_plan(count, rows, cols).bytes;
}

extern "C" int yuf_newton_schulz_f32(int count, int rows, int cols, const float *const *x, float *const *out, int steps, double a,
                                     double b, double c, double eps, void *workspace, void *stream) {
    return yuf::newton_schulz<float>(count, rows, cols, x, nullptr, out, {}, steps, a, b, c, eps, workspace, stream);
}

extern "C" int yuf_newton_schulz_bf16(int count, int rows, int cols, const uint16_t *const *x, uint16_t *const *out, int steps,
                                      double a, double b, double c, double eps, void *workspace, void *stream) {
    return yuf::newton_schulz<uint16_t>(count, rows, cols, x, nullptr, out, {}, steps, a, b, c, eps, workspace, stream);
}

extern "C" int yuf_muon_step_f32(int count, int rows, int cols, float *const *params, const float *const *grads,
                                 float *const *momenta, double lr, double momentum, int nesterov, double weight_decay, int steps,
                                 double a, double b, double c, double eps, void *workspace, void *stream) {
    return yuf::muon_step<float>(count, rows, cols, grads, momenta, params, lr, momentum, nesterov, weight_decay, steps, a, b, c,
                                 eps, workspace, stream);
}

extern "C" int yuf_muon_step_bf16(int count, int rows, int cols, uint16_t *const *params, const uint16_t *const *grads,
                                  float *const *momenta, double lr, double momentum, int nesterov, double weight_decay, int steps,
                                  double a, double b, double c, double eps, void *workspace, void *stream) {
    return yuf::muon_step<uint16_t>(count, rows, cols, grads, momenta, params, lr, momentum, nesterov, weight_decay, steps, a, b,
                                    c, eps, workspace, stream);
}
