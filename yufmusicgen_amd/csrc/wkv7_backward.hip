// Gradients of the WKV-7 scan, in chunks of 16 tokens on the fp32 matrix cores.
//
// Forward, per (b, h):  S_t = S_{t-1} (diag(d_t) + a_t b_t^T) + v_t k_t^T,  y_t = S_t r_t,
// d = exp(-e^{-0.5} sigmoid(w_raw)).  With the running decay products D_t of a chunk and,
// as rows per token, A = a D_{t-1}, R = r D_t, B = b / D_t, K = k / D_t (d >= 0.545 keeps
// 1 / D below 2^14):
//     Lab = strict(A B^T), Lak = strict(A K^T), Mrb = incl(R B^T), Mrk = incl(R K^T)
//     T = (I - Lab)^{-1},  C = T Lak
//     U = T A S0^T + C V                  (rows S_{t-1} a_t)
//     S1 = (S0 + U^T B + V^T K) diag(D_15)
// With G1, G0 the gradients of S1 and S0, G = G1 diag(D_15), and the same letters with a
// prime for gradients:
//     F = Mrb^T Y' + B G^T,   E = T^T F                    (E = U')
//     V' = Mrk^T Y' + K G^T + C^T F
//     G0 = G + Y'^T R + E^T A
//     Mrb' = incl(Y' U^T), Mrk' = incl(Y' V^T), Lab' = strict(E U^T), Lak' = strict(E V^T)
//     R' = Y' S0 + Mrb' B + Mrk' K        A' = E S0 + Lab' B + Lak' K
//     B' = U G + Mrb'^T R + Lab'^T A      K' = V G + Mrk'^T R + Lak'^T A
//     r' = R' D_t, a' = A' D_{t-1}, b' = B' / D_t, k' = K' / D_t
//     w' = (log d)' (-e^{-0.5}) sigmoid(w) (1 - sigmoid(w))
// (log d_t)' per key column is the sum over what enters the state before d_t -- S0 and, at tokens s < t, b_s and
// k_s -- times what takes from it behind -- G, r_s at tokens s >= t and a_s at tokens s > t.  The pairs with S0 or
// G are, with R'0 = Y' S0, A'0 = E S0, B'0 = U G and K'0 = V G, the first terms above,
//     sum_i (G S0)_i + sum_{s >= t} (R R'0)_s + sum_{s > t} (A A'0)_s + sum_{s < t} (B B'0 + K K'0)_s;
// those inside the chunk, with z = R (R' - R'0) - B (B' - B'0) - K (K' - K'0) + A (A' - A'0), which
// adds up to 0 over the chunk, are
//     - sum_{s < t} z_s - (A (A' - A'0))_t  =  sum_{s >= t} z_s - (A (A' - A'0))_t,
// from its start or from its end, and each token takes the side whose terms are the smaller in sum: terms
// that cancel are not larger than what they leave behind is made of, and nothing before the first
// token or behind the last one with a gradient is left of either.  One sum for all pairs, from the start as the
// difference of sum_i (G0 S0)_i and the earlier tokens' shares, lost up to all digits of a token
// whose state has died out within the chunk.
//
// The sequence is cut into segments of whole chunks that run side by side:
//   wkv7_grad_gram_kernel   what no state enters, for every chunk at once: T, C, Mrb, Mrk.
//   wkv7_grad_local_kernel  per segment: its end state from a zero start, the gradient of its
//                           start from a zero one at its end, and its transition Pi (the end
//                           state of S = I with v = 0), where S1 = S0 Pi + local and G0 =
//                           G1 Pi^T + local.  The first segment starts from the call's state
//                           and the last from its gradient, so that these two are final.
//   wkv7_grad_carry_kernel  both recurrences over the segments, a workgroup per value tile.
//   wkv7_grad_kernel        per segment: S forward over its chunks (kept per chunk, with U),
//                           then G and the gradients backward.
// One segment needs the first and the last alone, two no carry.  Four-chunk segments take the first two
// as one (wkv7_grad_block_kernel, block_form).
//
// 8 x 2048 x 16 x 40 (four segments): 76 + 126 + 6 + 354 us; 3 x 777 x 16 x 64 (ten): 17 + 44 + 17 + 66;
// 1 x 2048 x 16 x 64 (32, the first two as one): 33 + 22 + 56.  The first kernel is bound by memory (306 MB at 4.0
// TB/s, a third of them written), the second and the last by latency and issue together: an fp32 MFMA takes 32
// cycles of a SIMD, a VALU instruction 4 and a 16-byte LDS read about 18, none beside another, and with two waves a
// SIMD at most nothing else fills a wave's waits.
//
// MFMA layouts (16x16x4 f32; lane l, g = l / 16, li = l % 16): A[m = li][k = g],
// B[k = g][n = li], register r of the result D[m = 4 g + r][n = li].  k-step r of a
// product means rows {4 g + r}, so a result is the next product's B operand as it is,
// and an A operand is four consecutive k per lane.  Wave q of NB = ceil(N / 16) owns key
// tile q and value tile q; its stage-0 registers hold (token 4 g + r, column 16 q + li)
// of every input, which is at once the B operand of the products that contract tokens.
#include "common.h"
#include "kernels.h"

#include <algorithm>

namespace yuf {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kC = 16;     // tokens of a chunk
constexpr int kWave = 64;
constexpr int kXcds = 8;
constexpr int kST = 20;    // row stride of the 16 x 16 tiles in LDS
constexpr int kFrag = kWave * 4;  // floats of a 16 x 16 fragment
// Fragments of a chunk.  "Row": lane holds X[li][4 g + r]; "Col": X[4 g + r][li].
enum { kTRow, kCRow, kTCol, kCCol, kMrbCol, kMrkCol, kFrags };

struct GradParams {
    int B, T, H, N;
    int chunks;    // of a sequence
    int segments;  // of a sequence, of seg_chunks chunks each (the last may have fewer)
    int seg_chunks;
    const float *r, *w, *k, *v, *a, *b, *dy;
    const float *state_in, *dstate_out;
    float *dr, *dw, *dk, *dv, *da, *db, *dstate_in;
    float *frags;   // [B H][chunks][kFrags][kFrag]
    float *states;  // [B H][chunks][N][N]: the state before each chunk
    float *u;       // [B H][chunks][NB][kFrag]
    // [B H][segments][N][N]: the state before segment s >= 1, the gradient of the state after
    // segment s <= segments - 2, and Pi and Pi^T of the segments between the first and the last.
    float *starts, *ends, *powers, *powers_t;
};

__device__ __forceinline__ floatx4 mfma(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// c += sum over the 16 values of k of a (lane: 4 consecutive k of row li) and b.
__device__ __forceinline__ floatx4 mul16(floatx4 a, floatx4 b, floatx4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = mfma(a[r], b[r], c);
    return c;
}
// Products side by side: an MFMA waits for the one before it where it adds to the same
// accumulator, so independent sums take turns.
__device__ __forceinline__ void mul16(floatx4 a0, floatx4 b0, floatx4 &c0, floatx4 a1, floatx4 b1, floatx4 &c1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        c0 = mfma(a0[r], b0[r], c0);
        c1 = mfma(a1[r], b1[r], c1);
    }
}
template <int NB> __device__ __forceinline__ void mul16_tiles(const floatx4 (&a)[NB], floatx4 b, floatx4 (&c)[NB]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < NB; ++t) c[t] = mfma(a[t][r], b[r], c[t]);
}
__device__ __forceinline__ floatx4 ld4(const float *p) { return *reinterpret_cast<const floatx4 *>(p); }
__device__ __forceinline__ void st4(float *p, floatx4 v) { *reinterpret_cast<floatx4 *>(p) = v; }
// Four rows of a column, `stride` apart.
__device__ __forceinline__ floatx4 ldcol(const float *p, int stride) {
    return floatx4{p[0], p[stride], p[2 * stride], p[3 * stride]};
}
__device__ __forceinline__ void stcol(float *p, int stride, floatx4 v) {
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r * stride] = v[r];
}
__device__ __forceinline__ floatx4 buf_load4(__amdgpu_buffer_rsrc_t rsrc, uint32_t byte_offset) {
    return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, byte_offset, 0, 0));
}
__device__ __forceinline__ void buf_store4(floatx4 v, __amdgpu_buffer_rsrc_t rsrc, uint32_t byte_offset) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), rsrc, byte_offset, 0, 0);
}

// The 16 tokens x 16 columns of one wave in a chunk of a [B, T, H, N] tensor: lane
// (g, li) holds tokens 4 g + r of its column.  Tokens past T and columns past N read as
// 0 and are not written.
struct Tile {
    uint32_t offset[4];  // bytes from the head's row of the chunk's first token
    uint32_t bytes;      // range of the chunk
    size_t base;         // elements

    __device__ __forceinline__ void at(const GradParams &p, int b, int h, int chunk, int col, int g) {
        const int t0 = chunk * kC, nt = min(kC, p.T - t0), HN = p.H * p.N;
        base = (((size_t)b * p.T + t0) * p.H + h) * p.N;
        bytes = (uint32_t)((nt - 1) * HN + p.N) * 4u;
#pragma unroll
        for (int r = 0; r < 4; ++r) offset[r] = col < p.N ? (uint32_t)((4 * g + r) * HN + col) * 4u : kBufferOob;
    }
    __device__ __forceinline__ floatx4 load(const float *x) const {
        const auto rs = make_rsrc(x + base, bytes);
        floatx4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = buf_load(rs, offset[r]);
        return v;
    }
    __device__ __forceinline__ void store(float *x, floatx4 v) const {
        const auto rs = make_rsrc(x + base, bytes);
#pragma unroll
        for (int r = 0; r < 4; ++r) buf_store(v[r], rs, offset[r]);
    }
};

// Running decay products of a chunk for the lane's column.
struct Decays {
    floatx4 now, before, inv;  // D_t, D_{t-1}, 1 / D_t
    float last;                // D_15
    floatx4 slope;             // d log d / d w = -e^{-0.5} sigmoid(w) (1 - sigmoid(w))

    // valid: tokens of the chunk; the rest keep the state (d = 1).
    __device__ __forceinline__ void set(floatx4 w, int valid, int g) {
        float run[4], acc = 1.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // exp(-w) stays finite, so that 1 - sigmoid(w) = exp(-w) sigmoid(w) keeps its relative precision.
            const float e = __expf(w[r] < -80.0f ? 80.0f : -w[r]);
            const float sig = __builtin_amdgcn_rcpf(1.0f + e);
            const float d = __builtin_amdgcn_exp2f(-0.8750387749f * sig);  // e^{-0.5} log2(e)
            slope[r] = -0.6065306597f * sig * (e * sig);
            acc *= 4 * g + r < valid ? d : 1.0f;
            run[r] = acc;
        }
        // Products of the earlier lane groups' tokens (rows of 16 lanes): pairs, then halves.
        const auto s16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc), __float_as_uint(acc), false, false);
        const float even = __uint_as_float(s16[0]), odd = __uint_as_float(s16[1]);
        const float pair = even * odd;
        const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(pair), __float_as_uint(pair), false, false);
        const float low = __uint_as_float(s32[0]);
        const float base = g == 0 ? 1.0f : g == 1 ? even : g == 2 ? low : low * even;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            before[r] = r == 0 ? base : base * run[r - 1];
            now[r] = base * run[r];
            inv[r] = __builtin_amdgcn_rcpf(now[r]);
        }
        last = __shfl(now[3], 48 + (threadIdx.x & 15));
    }
};

// Sum over the four lanes of a column (one per row of 16 lanes), to all of them.
__device__ __forceinline__ float rows_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Sums over the earlier and over the later lane groups of a column.
struct Around {
    float before, after;
    __device__ __forceinline__ Around(float x, int g) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        const float even = __uint_as_float(a[0]), odd = __uint_as_float(a[1]), pair = even + odd;
        const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(pair), __float_as_uint(pair), false, false);
        const float low = __uint_as_float(b[0]), high = __uint_as_float(b[1]);
        before = g == 0 ? 0.0f : g == 1 ? even : g == 2 ? low : low + even;
        after = g == 0 ? odd + high : g == 1 ? high : g == 2 ? odd : 0.0f;
    }
};
__device__ __forceinline__ float sum4(floatx4 x) { return (x[0] + x[1]) + (x[2] + x[3]); }

// Units dealt so that consecutive ones (the chunks of a head, the heads of a batch row)
// share an XCD's L2.
__device__ __forceinline__ int xcd_unit(int per_xcd) { return (blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds; }

// A wave's LDS writes before its reads of other lanes' words.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The fragments of one chunk by one wave, from its tiles in LDS; sL and sP: 16 x kST floats each.
template <int NB>
__device__ __forceinline__ void chunk_fragments(const float *sA, const float *sR, const float *sB, const float *sK, float *sL, float *sP,
                                                int lane, float *out) {
    constexpr int SA = 16 * NB + 4;
    const int g = lane >> 4, li = lane & 15;
    floatx4 ab = {0.f, 0.f, 0.f, 0.f}, ak = ab, rb = ab, rk = ab;
#pragma unroll
    for (int jb = 0; jb < NB; ++jb) {
        const int at = li * SA + 16 * jb + 4 * g;
        const floatx4 a4 = ld4(sA + at), r4 = ld4(sR + at), b4 = ld4(sB + at), k4 = ld4(sK + at);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            ab = mfma(a4[r], b4[r], ab);
            ak = mfma(a4[r], k4[r], ak);
            rb = mfma(r4[r], b4[r], rb);
            rk = mfma(r4[r], k4[r], rk);
        }
    }
    // Register r: row t = 4 g + r, column s = li.
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = 4 * g + r;
        ab[r] = li < t ? ab[r] : 0.0f;
        ak[r] = li < t ? ak[r] : 0.0f;
        rb[r] = li <= t ? rb[r] : 0.0f;
        rk[r] = li <= t ? rk[r] : 0.0f;
    }
    st4(out + kMrbCol * kFrag, rb);
    st4(out + kMrkCol * kFrag, rk);
    st4(sL + li * kST + 4 * g, ab);  // Lab^T: column s of Lab in row s
    st4(sP + li * kST + 4 * g, ak);  // Lak^T
    wave_lds_fence();
    // Column li of T by forward substitution, right-looking (the four lane groups alike).
    float x[kC];
#pragma unroll
    for (int t = 0; t < kC; ++t) x[t] = li == t ? 1.0f : 0.0f;
#pragma unroll
    for (int s = 0; s < kC - 1; ++s) {
        // Two steps' columns at a time: the compiler would load them all first and add them last, which
        // takes 126 registers, so 70 and more waves at once.
        if (s % 2 == 0)
#pragma unroll
            for (int t = 0; t < kC; ++t) asm volatile("" : "+v"(x[t])::"memory");
#pragma unroll
        for (int m = s / 4; m < 4; ++m) {
            const floatx4 col = ld4(sL + s * kST + 4 * m);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * m + e > s) x[4 * m + e] = fmaf(col[e], x[s], x[4 * m + e]);
        }
    }
    wave_lds_fence();
    // T^T over Lab^T, row s = li: each lane group writes its four tokens.
    const floatx4 own = g == 0 ? floatx4{x[0], x[1], x[2], x[3]}
                      : g == 1 ? floatx4{x[4], x[5], x[6], x[7]}
                      : g == 2 ? floatx4{x[8], x[9], x[10], x[11]}
                               : floatx4{x[12], x[13], x[14], x[15]};
    st4(sL + li * kST + 4 * g, own);
    wave_lds_fence();
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    const floatx4 t_row = ldcol(sL + 4 * g * kST + li, kST);  // T[li][4 g + r]
    st4(out + kTRow * kFrag, t_row);
    st4(out + kTCol * kFrag, ld4(sL + li * kST + 4 * g));     // T[4 g + r][li]
    // C[t][s] = sum T[t][m] Lak[m][s]: B operand Lak[m = 4 g + r][s = li] = the Gram's registers.
    st4(out + kCCol * kFrag, mul16(t_row, ak, zero));
    // C^T[s][t] = sum Lak^T[s][m] T^T[m][t]: its registers, [s = 4 g + r][t = li], are C's row fragment.
    // Its B operand T^T[m = 4 g + r][t = li] is the same four values as T's row fragment.
    st4(out + kCRow * kFrag, mul16(ld4(sP + li * kST + 4 * g), t_row, zero));
}

// One wave per chunk of a head.
template <int NB> __global__ void __launch_bounds__(kWave) wkv7_grad_gram_kernel(GradParams p, int units, int per_xcd) {
    constexpr int SA = 16 * NB + 4;
    __shared__ __attribute__((aligned(16))) float tiles[4 * kC * SA + 2 * kC * kST];
    float *sA = tiles, *sR = sA + kC * SA, *sB = sR + kC * SA, *sK = sB + kC * SA, *scratch = sK + kC * SA;
    const int unit = xcd_unit(per_xcd);
    if (unit >= units) return;
    const int head = unit / p.chunks, chunk = unit - head * p.chunks;
    const int bb = head / p.H, h = head - bb * p.H;
    const int lane = threadIdx.x, g = lane >> 4, li = lane & 15;
    const int valid = min(kC, p.T - chunk * kC);
#pragma unroll
    for (int q = 0; q < NB; ++q) {
        Tile tile;
        tile.at(p, bb, h, chunk, 16 * q + li, g);
        Decays d;
        d.set(tile.load(p.w), valid, g);
        const int at = 4 * g * SA + 16 * q + li;
        stcol(sA + at, SA, tile.load(p.a) * d.before);
        stcol(sR + at, SA, tile.load(p.r) * d.now);
        stcol(sB + at, SA, tile.load(p.b) * d.inv);
        stcol(sK + at, SA, tile.load(p.k) * d.inv);
    }
    wave_lds_fence();
    chunk_fragments<NB>(sA, sR, sB, sK, scratch, scratch + kC * kST, lane,
                        p.frags + ((size_t)head * p.chunks + chunk) * kFrags * kFrag + 4 * lane);
}

// The wave's number, known to be the same for its lanes: descriptors and branches made from it stay scalar.
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// What a wave of the segment kernels is: its head, segment, tile and place in it.
struct Place {
    int head, bb, h, q, g, li, lane, col;
    int c0, c1;  // chunks of the segment
    __device__ __forceinline__ Place(const GradParams &p, int head_, int seg) {
        head = head_;
        bb = head / p.H;
        h = head - bb * p.H;
        q = wave_id();
        lane = threadIdx.x & 63;
        g = lane >> 4;
        li = lane & 15;
        col = 16 * q + li;
        c0 = seg * p.seg_chunks;
        c1 = min(p.chunks, c0 + p.seg_chunks);
    }
};

// State tiles and memory.  "Rows": value 16 q + li, keys 16 jb + 4 g ..; "columns": value
// 16 ib + 4 g + r, key 16 q + li.  A null state reads as zeros.
template <int NB> struct StateIo {
    int N, col, g;
    uint32_t bytes;
    __device__ __forceinline__ StateIo(const GradParams &p, const Place &w) : N(p.N), col(w.col), g(w.g), bytes((uint32_t)(p.N * p.N * 4)) {}
    __device__ __forceinline__ uint32_t row(int jb) const {
        return col < N && 16 * jb + 4 * g < N ? (uint32_t)(col * N + 16 * jb + 4 * g) * 4u : kBufferOob;
    }
    // Column elements share a lane offset; their rows' uniform part goes into the scalar offset, which
    // stays below the range (16 (NB - 1) + 3 < N), while values past N end beyond it.
    __device__ __forceinline__ uint32_t column() const { return col < N ? (uint32_t)(4 * g * N + col) * 4u : kBufferOob; }
    __device__ __forceinline__ uint32_t row_part(int ib, int r) const { return (uint32_t)((16 * ib + r) * N) * 4u; }
    __device__ __forceinline__ void load_rows(const float *s, floatx4 (&x)[NB]) const {
        const auto rs = make_rsrc(s, s ? bytes : 0u);
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) x[jb] = buf_load4(rs, row(jb));
    }
    __device__ __forceinline__ void store_rows(const floatx4 (&x)[NB], float *s) const {
        const auto rs = make_rsrc(s, bytes);
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) buf_store4(x[jb], rs, row(jb));
    }
    __device__ __forceinline__ void load_columns(const float *s, floatx4 (&x)[NB]) const {
        const auto rs = make_rsrc(s, s ? bytes : 0u);
#pragma unroll
        for (int ib = 0; ib < NB; ++ib)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[ib][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, column(), row_part(ib, r), 0));
    }
    __device__ __forceinline__ void store_columns(const floatx4 (&x)[NB], float *s) const {
        const auto rs = make_rsrc(s, bytes);
#pragma unroll
        for (int ib = 0; ib < NB; ++ib)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = x[ib][r];  // a copy: __builtin_bit_cast takes a vector element in place for the first one
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), rs, column(), row_part(ib, r), 0);
            }
    }
};

__device__ __forceinline__ const float *head_state(const float *s, const GradParams &p, int head) {
    return s ? s + (size_t)head * p.N * p.N : nullptr;
}
__device__ __forceinline__ float *seg_state(float *s, const GradParams &p, int head, int seg) {
    return s + ((size_t)head * p.segments + seg) * p.N * p.N;
}

// X S for a row-fragment operand X (tokens, keys) in LDS: its own 16 tokens times the state tiles.
template <int NB> __device__ __forceinline__ floatx4 times_state(const float *x, const floatx4 (&S)[NB]) {
    floatx4 even = {0.f, 0.f, 0.f, 0.f}, odd = even;  // k-steps
#pragma unroll
    for (int jb = 0; jb < NB; ++jb) {
        const floatx4 x4 = ld4(x + 16 * jb);
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            even = mfma(x4[r], S[jb][r], even);
            odd = mfma(x4[r + 1], S[jb][r + 1], odd);
        }
    }
    return even + odd;
}

// S += X^T b for a column-fragment operand X (tokens, keys) in LDS, four tiles at a time.
template <int NB> __device__ __forceinline__ void add_to_state(const float *x, floatx4 b, floatx4 (&S)[NB]) {
    constexpr int SA = 16 * NB + 4, kGroup = NB < 4 ? NB : 4;
#pragma unroll
    for (int j0 = 0; j0 < NB; j0 += kGroup) {
        floatx4 x4[kGroup];
#pragma unroll
        for (int t = 0; t < kGroup; ++t) x4[t] = ldcol(x + 16 * (j0 + t), SA);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int t = 0; t < kGroup; ++t) S[j0 + t] = mfma(x4[t][r], b[r], S[j0 + t]);
    }
}

template <int NB> struct Sweep {
    static constexpr int NP = 16 * NB, SA = NP + 4, kTok = kC * SA;
    static constexpr int kBuf = 3 * kTok + NP;  // three token tiles and D_15
    static constexpr int kFloats = 2 * kBuf;    // two of them: one barrier per chunk
};

// S^T[:, value tile q], as NB tiles of 16 keys, over the segment's chunks; KEEP: the state
// before each chunk and U go to memory; POWER: P likewise, with v = 0.
template <int NB, bool KEEP, bool POWER>
__device__ __forceinline__ void sweep_forward(const GradParams &p, const Place &w, float *lds, floatx4 (&S)[NB], floatx4 (&P)[NB]) {
    using Ly = Sweep<NB>;
    constexpr int SA = Ly::SA, kTok = Ly::kTok;
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    const float *frags = p.frags + (size_t)w.head * p.chunks * kFrags * kFrag + 4 * w.lane;
    float *us = p.u + ((size_t)w.head * p.chunks * NB + w.q) * kFrag + 4 * w.lane;
    const StateIo<NB> io(p, w);
    floatx4 wv, k, v, a, b;
    auto fetch = [&](int c) {
        Tile tile;
        tile.at(p, w.bb, w.h, c, w.col, w.g);
        wv = tile.load(p.w);
        k = tile.load(p.k);
        v = tile.load(p.v);
        a = tile.load(p.a);
        b = tile.load(p.b);
    };
    if (w.c0 < w.c1) fetch(w.c0);
    for (int c = w.c0; c < w.c1; ++c) {
        float *sA = lds + ((c - w.c0) & 1) * Ly::kBuf, *sB = sA + kTok, *sK = sB + kTok, *sD = sK + kTok;
        const floatx4 t_row = ld4(frags + ((size_t)c * kFrags + kTRow) * kFrag);
        const floatx4 c_row = ld4(frags + ((size_t)c * kFrags + kCRow) * kFrag);
        if constexpr (KEEP) io.store_rows(S, p.states + ((size_t)w.head * p.chunks + c) * p.N * p.N);
        Decays d;
        d.set(wv, min(kC, p.T - c * kC), w.g);
        const int at = 4 * w.g * SA + w.col;
        stcol(sA + at, SA, a * d.before);
        stcol(sB + at, SA, b * d.inv);
        stcol(sK + at, SA, k * d.inv);
        if (w.g == 3) sD[w.col] = d.last;
        const floatx4 v4 = v;
        fetch(min(c + 1, w.c1 - 1));
        lds_barrier();
        floatx4 X = zero, Y = zero, U = zero, UP = zero;  // POWER: Y is X of P, else X's odd k-steps
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) {
            const floatx4 a4 = ld4(sA + w.li * SA + 16 * jb + 4 * w.g);
            if constexpr (POWER) {
                mul16(a4, S[jb], X, a4, P[jb], Y);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    X = mfma(a4[r], S[jb][r], X);
                    Y = mfma(a4[r + 1], S[jb][r + 1], Y);
                }
            }
        }
        U = mul16(c_row, v4, U);
        floatx4 k4[NB], b4[NB];
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) k4[jb] = ldcol(sK + 4 * w.g * SA + 16 * jb + w.li, SA);
        mul16_tiles<NB>(k4, v4, S);
        if constexpr (POWER) {
            mul16(t_row, X, U, t_row, Y, UP);
        } else {
            X += Y;
            U = mul16(t_row, X, U);
        }
        if constexpr (KEEP) st4(us + (size_t)c * NB * kFrag, U);
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) b4[jb] = ldcol(sB + 4 * w.g * SA + 16 * jb + w.li, SA);
        mul16_tiles<NB>(b4, U, S);
        if constexpr (POWER) mul16_tiles<NB>(b4, UP, P);
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) {
            const floatx4 d4 = ld4(sD + 16 * jb + 4 * w.g);
            S[jb] *= d4;
            if constexpr (POWER) P[jb] *= d4;
        }
    }
}

// G^T[:, value tile q] backward over the segment's chunks.
template <int NB>
__device__ __forceinline__ void sweep_backward(const GradParams &p, const Place &w, float *lds, floatx4 (&G)[NB]) {
    using Ly = Sweep<NB>;
    constexpr int SA = Ly::SA, kTok = Ly::kTok;
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    const float *frags = p.frags + (size_t)w.head * p.chunks * kFrags * kFrag + 4 * w.lane;
    floatx4 wv, r, y, a, b;
    auto fetch = [&](int c) {
        Tile tile;
        tile.at(p, w.bb, w.h, c, w.col, w.g);
        wv = tile.load(p.w);
        r = tile.load(p.r);
        y = tile.load(p.dy);
        a = tile.load(p.a);
        b = tile.load(p.b);
    };
    if (w.c0 < w.c1) fetch(w.c1 - 1);
    for (int c = w.c1 - 1; c >= w.c0; --c) {
        float *sA = lds + ((c - w.c0) & 1) * Ly::kBuf, *sB = sA + kTok, *sR = sB + kTok, *sD = sR + kTok;
        const floatx4 t_col = ld4(frags + ((size_t)c * kFrags + kTCol) * kFrag);
        const floatx4 rb_col = ld4(frags + ((size_t)c * kFrags + kMrbCol) * kFrag);
        Decays d;
        d.set(wv, min(kC, p.T - c * kC), w.g);
        const int at = 4 * w.g * SA + w.col;
        stcol(sA + at, SA, a * d.before);
        stcol(sB + at, SA, b * d.inv);
        stcol(sR + at, SA, r * d.now);
        if (w.g == 3) sD[w.col] = d.last;
        const floatx4 y4 = y;
        fetch(max(c - 1, w.c0));
        lds_barrier();
        floatx4 F = zero, F1 = zero;  // even and odd k-steps
        F1 = mul16(rb_col, y4, F1);
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) {
            G[jb] *= ld4(sD + 16 * jb + 4 * w.g);
            const floatx4 b4 = ld4(sB + w.li * SA + 16 * jb + 4 * w.g);
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                F = mfma(b4[r], G[jb][r], F);
                F1 = mfma(b4[r + 1], G[jb][r + 1], F1);
            }
        }
        F += F1;
        floatx4 r4[NB], a4[NB];
#pragma unroll
        for (int jb = 0; jb < NB; ++jb) {
            const int o = 4 * w.g * SA + 16 * jb + w.li;
            r4[jb] = ldcol(sR + o, SA);
            a4[jb] = ldcol(sA + o, SA);
        }
        mul16_tiles<NB>(r4, y4, G);
        mul16_tiles<NB>(a4, mul16(t_col, F, zero), G);
    }
}

// Workgroups: the segments 0 .. segments - 2 of every head forward, then 1 .. segments - 1 backward.
template <int NB> __global__ void __launch_bounds__(NB *kWave) wkv7_grad_local_kernel(GradParams p, int units, int per_xcd) {
    __shared__ __attribute__((aligned(16))) float lds[Sweep<NB>::kFloats];
    int unit = xcd_unit(per_xcd);
    if (unit >= units) return;
    const int per_head = p.segments - 1, half = units / 2;
    const bool back = unit >= half;
    if (back) unit -= half;
    const int head = unit / per_head, seg = unit - head * per_head + back;
    const Place w(p, head, seg);
    const StateIo<NB> io(p, w);
    floatx4 S[NB], P[NB];
    if (back) {
        io.load_rows(seg == p.segments - 1 ? head_state(p.dstate_out, p, head) : nullptr, S);
        sweep_backward<NB>(p, w, lds, S);
        io.store_rows(S, seg_state(p.ends, p, head, seg - 1));
        return;
    }
    io.load_rows(seg == 0 ? head_state(p.state_in, p, head) : nullptr, S);
    if (seg == 0) {
        sweep_forward<NB, false, false>(p, w, lds, S, P);
    } else {
#pragma unroll
        for (int jb = 0; jb < NB; ++jb)
#pragma unroll
            for (int r = 0; r < 4; ++r) P[jb][r] = 16 * jb + 4 * w.g + r == w.col ? 1.0f : 0.0f;
        sweep_forward<NB, false, true>(p, w, lds, S, P);
        io.store_rows(P, seg_state(p.powers, p, head, seg));
        io.store_columns(P, seg_state(p.powers_t, p, head, seg));
    }
    io.store_rows(S, seg_state(p.starts, p, head, seg + 1));
}

// The two kernels above as one, for segments of kBlock chunks, a workgroup each.  Its inputs are read
// once, scaled into LDS, and stay there: four waves make the chunks' fragments, then 3 NB
// independent chains run over them without a barrier, NB tiles each of the segment's end state, its Pi, and
// the gradient of its start.  1 x 2048 x 16 x 64: 33 us, so 56 with the two kernels; 2 x 1024 x 16 x 40: 31, so
// 38.  Not for many rounds of workgroups (two of 64 to 81 KB a CU): 8 x 2048 x 16 x 40 in eight: 269, so 213.
constexpr int kBlock = 4;
// Waves of a SIMD that two workgroups of a CU need (their LDS fits up to NB = 4).
template <int NB> constexpr int kBlockPerSimd = NB >= 8 ? 4 : (2 * (3 * NB < 4 ? 4 : 3 * NB) + 3) / 4;
template <int NB> constexpr int kBlockWaves = 3 * NB < 4 ? 4 : 3 * NB > 16 ? 16 : 3 * NB;

template <int NB> __global__ void __launch_bounds__(kBlockWaves<NB> *kWave, kBlockPerSimd<NB>) wkv7_grad_block_kernel(GradParams p, int units, int per_xcd) {
    constexpr int NP = 16 * NB, SA = NP + 4, kTok = kC * SA, kWaves = kBlockWaves<NB>;
    __shared__ __attribute__((aligned(16))) float lds[kBlock * (4 * kTok + NP + 2 * kC * kST)];
    static_assert(sizeof(lds) <= 160 * 1024, "LDS of one CU");
    auto tile_of = [&](int what, int i) { return lds + (4 * i + what) * kTok; };  // 0 A, 1 R, 2 B, 3 K of chunk i
    float *sD = lds + kBlock * 4 * kTok, *scratch = sD + kBlock * NP;
    const int unit = xcd_unit(per_xcd);
    if (unit >= units) return;  // uniform over the workgroup
    const int blocks = (p.chunks + kBlock - 1) / kBlock;
    const int head = unit / blocks, seg = unit - head * blocks;
    const int c0 = seg * kBlock, nc = min(kBlock, p.chunks - c0);
    const int wave = wave_id();
    Place w(p, head, 0);
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};

    for (int i = wave; i < nc * NB; i += kWaves) {
        const int chunk = i / NB, col = 16 * (i - chunk * NB) + w.li;
        Tile tile;
        tile.at(p, w.bb, w.h, c0 + chunk, col, w.g);
        const floatx4 a = tile.load(p.a), r = tile.load(p.r), b = tile.load(p.b), k = tile.load(p.k);
        Decays d;
        d.set(tile.load(p.w), min(kC, p.T - (c0 + chunk) * kC), w.g);
        const int at = 4 * w.g * SA + col;
        stcol(tile_of(0, chunk) + at, SA, a * d.before);
        stcol(tile_of(1, chunk) + at, SA, r * d.now);
        stcol(tile_of(2, chunk) + at, SA, b * d.inv);
        stcol(tile_of(3, chunk) + at, SA, k * d.inv);
        if (w.g == 3) sD[chunk * NP + col] = d.last;
    }
    lds_barrier();
    float *frags = p.frags + ((size_t)head * p.chunks + c0) * kFrags * kFrag + 4 * w.lane;
    if (wave < nc)
        chunk_fragments<NB>(tile_of(0, wave), tile_of(1, wave), tile_of(2, wave), tile_of(3, wave), scratch + 2 * wave * kC * kST,
                            scratch + (2 * wave + 1) * kC * kST, w.lane, frags + (size_t)wave * kFrags * kFrag);
    __syncthreads();  // the fragments are read back from memory

    for (int task = wave; task < 3 * NB; task += kWaves) {
        const int kind = task / NB;  // 0: state, 1: Pi, 2: gradient
        if (kind == 0 && seg == p.segments - 1) continue;
        if (kind == 1 && (seg == 0 || seg == p.segments - 1)) continue;
        if (kind == 2 && seg == 0) continue;
        w.q = task - kind * NB;
        w.col = 16 * w.q + w.li;
        const StateIo<NB> io(p, w);
        const int row = w.li * SA + 4 * w.g, colm = 4 * w.g * SA + w.li;  // operands: rows of tokens, columns of keys
        auto load_token = [&](const float *x, int i) {
            Tile tile;
            tile.at(p, w.bb, w.h, c0 + min(i, nc - 1), w.col, w.g);
            return tile.load(x);
        };
        auto fragment = [&](int i, int which) { return ld4(frags + ((size_t)i * kFrags + which) * kFrag); };
        floatx4 S[NB];
        if (kind == 2) {
            io.load_rows(seg == p.segments - 1 ? head_state(p.dstate_out, p, head) : nullptr, S);
            floatx4 next = load_token(p.dy, nc - 1);
            for (int i = nc - 1; i >= 0; --i) {
                const floatx4 t_col = fragment(i, kTCol), rb_col = fragment(i, kMrbCol), y4 = next;
                next = load_token(p.dy, max(i - 1, 0));
#pragma unroll
                for (int jb = 0; jb < NB; ++jb) S[jb] *= ld4(sD + i * NP + 16 * jb + 4 * w.g);
                floatx4 F = times_state<NB>(tile_of(2, i) + row, S);
                F = mul16(rb_col, y4, F);
                add_to_state<NB>(tile_of(1, i) + colm, y4, S);
                const floatx4 E = mul16(t_col, F, zero);
                add_to_state<NB>(tile_of(0, i) + colm, E, S);
            }
            io.store_rows(S, seg_state(p.ends, p, head, seg - 1));
            continue;
        }
        if (kind == 0) {
            io.load_rows(seg == 0 ? head_state(p.state_in, p, head) : nullptr, S);
        } else {
#pragma unroll
            for (int jb = 0; jb < NB; ++jb)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[jb][r] = 16 * jb + 4 * w.g + r == w.col ? 1.0f : 0.0f;
        }
        floatx4 next = kind == 0 ? load_token(p.v, 0) : zero;
        for (int i = 0; i < nc; ++i) {
            const floatx4 t_row = fragment(i, kTRow), v4 = next;
            floatx4 U = zero;
            const floatx4 X = times_state<NB>(tile_of(0, i) + row, S);
            if (kind == 0) {
                next = load_token(p.v, i + 1);
                U = mul16(fragment(i, kCRow), v4, U);
                add_to_state<NB>(tile_of(3, i) + colm, v4, S);
            }
            U = mul16(t_row, X, U);
            add_to_state<NB>(tile_of(2, i) + colm, U, S);
#pragma unroll
            for (int jb = 0; jb < NB; ++jb) S[jb] *= ld4(sD + i * NP + 16 * jb + 4 * w.g);
        }
        if (kind == 0) {
            io.store_rows(S, seg_state(p.starts, p, head, seg + 1));
        } else {
            io.store_rows(S, seg_state(p.powers, p, head, seg));
            io.store_columns(S, seg_state(p.powers_t, p, head, seg));
        }
    }
}

// A workgroup per (head, value tile, direction): x <- x Pi + local (x Pi^T backward) over the
// segments between the first and the last; wave q computes key tile q, and the tiles of x go round
// through LDS.  Each step waits for memory longer than for its products, so loads run kAhead steps ahead.
template <int NB> __global__ void __launch_bounds__(NB *kWave) wkv7_grad_carry_kernel(GradParams p, int units, int per_xcd) {
    constexpr int kAhead = 3;
    __shared__ __attribute__((aligned(16))) float tiles[2][NB][kFrag];
    int unit = xcd_unit(per_xcd);
    if (unit >= units) return;  // uniform over the workgroup
    const int head = unit / (2 * NB);
    unit -= head * 2 * NB;
    const bool back = unit >= NB;
    const int i = 16 * (back ? unit - NB : unit) + (threadIdx.x & 15);  // value of the lane's column
    const Place w(p, head, 0);
    const int N = p.N, dir = back ? -1 : 1, steps = p.segments - 2;
    const uint32_t bytes = (uint32_t)(N * N * 4);
    float *slots = back ? p.ends : p.starts;
    // Element offsets of (value i, keys 16 q + 4 g ..) of a state and (row 16 q + li, 16 kb + 4 g ..) of Pi.
    const uint32_t own = i < N && 16 * w.q + 4 * w.g < N ? (uint32_t)(i * N + 16 * w.q + 4 * w.g) * 4u : kBufferOob;
    uint32_t at[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
        at[kb] = w.col < N && 16 * kb + 4 * w.g < N ? (uint32_t)(w.col * N + 16 * kb + 4 * w.g) * 4u : kBufferOob;
    // Forward: slot 1 is final, slot s + 1 += slot s Pi_s; backward: slot segments - 2 is, slot
    // s - 1 += slot s Pi_s^T.  x^T[j][i] = sum_k Pi^T[j][k] x^T[k][i] (Pi[j][k] backward).
    const int first = back ? p.segments - 2 : 1;
    const float *powers = seg_state(back ? p.powers : p.powers_t, p, head, 0);
    slots = seg_state(slots, p, head, 0);
    floatx4 pi[kAhead][NB], local[kAhead];
    auto fetch = [&](int n, floatx4 (&m)[NB], floatx4 &l) {
        const int s = first + min(n, steps - 1) * dir;  // past the last step: its values again, unused
        const auto rs = make_rsrc(powers + (size_t)s * N * N, bytes);
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) m[kb] = buf_load4(rs, at[kb]);
        l = buf_load4(make_rsrc(slots + (size_t)(s + dir) * N * N, bytes), own);
    };
    floatx4 x = buf_load4(make_rsrc(slots + (size_t)first * N * N, bytes), own);
    // The waits for loads count exactly where the loop has no branch (steps past the last one store nothing)
    // and the loads before it are issued in its order (the scheduling barriers).
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        fetch(n, pi[n], local[n]);
    }
    __builtin_amdgcn_sched_barrier(0);
    for (int n0 = 0; n0 < steps; n0 += kAhead) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const int n = n0 + e;
            float *tile = &tiles[n & 1][0][4 * w.lane];
            st4(tile + w.q * kFrag, x);
            lds_barrier();
            floatx4 y0 = local[e], y1 = {0.f, 0.f, 0.f, 0.f};  // even and odd k-steps
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                const floatx4 k4 = ld4(tile + kb * kFrag);
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    y0 = mfma(pi[e][kb][r], k4[r], y0);
                    y1 = mfma(pi[e][kb][r + 1], k4[r + 1], y1);
                }
            }
            x = y0 + y1;
            // Loads of a slot that a step writes were issued before its store: each slot is read once, ahead.
            fetch(n + kAhead, pi[e], local[e]);
            const int to = first + (min(n, steps - 1) + 1) * dir;
            buf_store4(x, make_rsrc(slots + (size_t)to * N * N, n < steps ? bytes : 0u), own);
        }
    }
}

// A workgroup of NB waves per segment of a head.  Scheduled for two waves per SIMD instead of three the operands
// come from LDS in time: the call of 8 x 2048 x 16 x 40 600 us, so 562.  By counters a SIMD's time goes, at N = 64 with
// two waves on each (1 x 2048 x 16 x 64), 42 % to MFMAs, 11 to VALU and 12 to LDS instructions; at N = 40 (8 x 2048 x
// 16), whose two three-wave workgroups leave two of a CU's SIMDs with one wave, 36, 10 and 10 on average and 48, 14 and 14
// on the other two, and a wave waits 38 % of its time for memory, LDS and barriers.
template <int NB> __global__ void __launch_bounds__(NB *kWave) __attribute__((amdgpu_waves_per_eu(2, 2))) wkv7_grad_kernel(GradParams p, int units, int per_xcd) {
    constexpr int NP = 16 * NB, SA = NP + 4, kTok = kC * SA;
    // Backward: B, K, V, Y', U, E, G [value][key] and the four 16 x 16 gradients.
    constexpr int kBackward = 6 * kTok + NP * SA + 4 * kC * kST;
    __shared__ __attribute__((aligned(16))) float lds[Sweep<NB>::kFloats > kBackward ? Sweep<NB>::kFloats : kBackward];
    static_assert(sizeof(lds) <= 160 * 1024, "LDS of one CU");
    const int unit = xcd_unit(per_xcd);
    if (unit >= units) return;  // uniform over the workgroup
    const int head = unit / p.segments, seg = unit - head * p.segments;
    const Place w(p, head, seg);
    const StateIo<NB> io(p, w);
    const int q = w.q, g = w.g, li = w.li, col = w.col, N = p.N;
    const floatx4 zero = {0.f, 0.f, 0.f, 0.f};
    const float *frags = p.frags + (size_t)head * p.chunks * kFrags * kFrag + 4 * w.lane;
    const float *states = p.states + (size_t)head * p.chunks * N * N;
    const float *us = p.u + ((size_t)head * p.chunks * NB + q) * kFrag + 4 * w.lane;

    {
        floatx4 S[NB], none[NB];
        io.load_rows(seg == 0 ? head_state(p.state_in, p, head) : seg_state(p.starts, p, head, seg), S);
        sweep_forward<NB, true, false>(p, w, lds, S, none);
    }
    __syncthreads();  // the states are read across waves, and LDS is used anew

    // ----------------------------------------------------------------- backward
    float *sB = lds, *sK = sB + kTok, *sV = sK + kTok, *sY = sV + kTok, *sU = sY + kTok, *sE = sU + kTok;
    float *sG = sE + kTok;  // G, [value][key]
    float *sMrb = sG + NP * SA, *sMrk = sMrb + kC * kST, *sLab = sMrk + kC * kST, *sLak = sLab + kC * kST;
    // G[:, key tile q] as NB tiles of 16 values, and S0 in the same layout.
    floatx4 G[NB], S0[NB];
    io.load_columns(seg == p.segments - 1 ? head_state(p.dstate_out, p, head) : seg_state(p.ends, p, head, seg), G);
    for (int c = w.c1 - 1; c >= w.c0; --c) {
        Tile tile;
        tile.at(p, w.bb, w.h, c, col, g);
        const float *fr = frags + (size_t)c * kFrags * kFrag;
        const floatx4 wv = tile.load(p.w), rr = tile.load(p.r), aa = tile.load(p.a), bv = tile.load(p.b);
        const floatx4 kv = tile.load(p.k), vv = tile.load(p.v), yv = tile.load(p.dy);
        const floatx4 uv = ld4(us + (size_t)c * NB * kFrag);
        io.load_columns(states + (size_t)c * N * N, S0);
        Decays d;
        d.set(wv, min(kC, p.T - c * kC), g);
        const floatx4 A = aa * d.before, R = rr * d.now, B = bv * d.inv, K = kv * d.inv;
        const int at = 4 * g * SA + col;
        stcol(sB + at, SA, B);
        stcol(sK + at, SA, K);
        stcol(sV + at, SA, vv);
        stcol(sY + at, SA, yv);
        stcol(sU + at, SA, uv);
#pragma unroll
        for (int ib = 0; ib < NB; ++ib) {
            G[ib] *= d.last;
            stcol(sG + (16 * ib + 4 * g) * SA + col, SA, G[ib]);
        }
        const floatx4 t_col = ld4(fr + kTCol * kFrag), c_col = ld4(fr + kCCol * kFrag);
        const floatx4 rb_col = ld4(fr + kMrbCol * kFrag), rk_col = ld4(fr + kMrkCol * kFrag);
        lds_barrier();
        // Value tile q: F, V'; key tile q: Y' S0, U G, V G.
        floatx4 F = zero, dV = zero, dR = zero, dA = zero, dB = zero, dK = zero;
        float share = 0.0f;  // sum_i (G S0)_i of the lane's key
        mul16(rb_col, yv, F, rk_col, yv, dV);
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            const int o = li * SA + 16 * t + 4 * g;
            const floatx4 g4 = ld4(sG + col * SA + 16 * t + 4 * g), b4 = ld4(sB + o), k4 = ld4(sK + o);
            const floatx4 y4 = ld4(sY + o), u4 = ld4(sU + o), v4 = ld4(sV + o);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                F = mfma(b4[r], g4[r], F);
                dV = mfma(k4[r], g4[r], dV);
                dR = mfma(y4[r], S0[t][r], dR);
                dB = mfma(u4[r], G[t][r], dB);
                dK = mfma(v4[r], G[t][r], dK);
                share = fmaf(G[t][r], S0[t][r], share);
            }
        }
        floatx4 E = zero;
        mul16(t_col, F, E, c_col, F, dV);
        stcol(sE + at, SA, E);
        tile.store(p.dv, dV);
        // Rows t = 4 g + r, columns s = li of X Z^T, kept where s <= t (s < t).
        auto gram = [&](const float *x, const float *z, float *out, bool strict) {
            floatx4 m = zero, m1 = zero;  // even and odd k-steps
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                const floatx4 x4 = ld4(x + li * SA + 16 * t + 4 * g), z4 = ld4(z + li * SA + 16 * t + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    m = mfma(x4[r], z4[r], m);
                    m1 = mfma(x4[r + 1], z4[r + 1], m1);
                }
            }
            m += m1;
#pragma unroll
            for (int r = 0; r < 4; ++r) out[(4 * g + r) * kST + li] = li < 4 * g + r + !strict ? m[r] : 0.0f;
        };
        const floatx4 pr = R * dR, in = B * dB + K * dK;
        float before = rows_sum(share) + Around(sum4(in), g).before;
        if (q == 0) gram(sY, sU, sMrb, false);
        if (q == (NB > 1 ? 1 : 0)) gram(sY, sV, sMrk, false);
        lds_barrier();
        if (q == (NB > 2 ? 2 : 0)) gram(sE, sU, sLab, true);
        if (q == (NB > 3 ? 3 : NB > 1 ? 1 : 0)) gram(sE, sV, sLak, true);
        {
            // G0 = G + Y'^T R + E^T A
            floatx4 x4[NB];
#pragma unroll
            for (int t = 0; t < NB; ++t) x4[t] = ldcol(sY + 4 * g * SA + 16 * t + li, SA);
            mul16_tiles<NB>(x4, R, G);
#pragma unroll
            for (int t = 0; t < NB; ++t) x4[t] = ldcol(sE + 4 * g * SA + 16 * t + li, SA);
            mul16_tiles<NB>(x4, A, G);
        }
        floatx4 iR = zero, iA = zero, iA1 = zero, iB = zero, iK = zero;  // the chunk's own parts of R', A', B', K'
        mul16(ld4(sMrb + li * kST + 4 * g), B, iR, ldcol(sMrb + 4 * g * kST + li, kST), R, iB);
        mul16(ld4(sMrk + li * kST + 4 * g), K, iR, ldcol(sMrk + 4 * g * kST + li, kST), R, iK);
        floatx4 dA1 = zero;
#pragma unroll
        for (int t = 0; t < NB; ++t) {
            const floatx4 e4 = ld4(sE + li * SA + 16 * t + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                dA = mfma(e4[r], S0[t][r], dA);
                dA1 = mfma(e4[r + 1], S0[t][r + 1], dA1);
            }
        }
        const floatx4 yr = R * iR;
        tile.store(p.dr, (dR + iR) * d.now);
        lds_barrier();
        dA += dA1;
        const floatx4 pa = A * dA;
        float after = Around(sum4(pr + pa), g).after;
        mul16(ld4(sLab + li * kST + 4 * g), B, iA, ldcol(sLab + 4 * g * kST + li, kST), A, iB);
        mul16(ld4(sLak + li * kST + 4 * g), K, iA1, ldcol(sLak + 4 * g * kST + li, kST), A, iK);
        iA += iA1;
        tile.store(p.da, (dA + iA) * d.before);
        tile.store(p.db, (dB + iB) * d.inv);
        tile.store(p.dk, (dK + iK) * d.inv);
        // (log d_t)', in the tokens' order forward for what enters the state and backward for what takes from it.
        const floatx4 ya = A * iA, yb = B * iB + K * iK, rest = yr - yb, z = rest + ya;
        floatx4 m;  // magnitude of a token's terms
#pragma unroll
        for (int r = 0; r < 4; ++r) m[r] = fabsf(yr[r]) + fabsf(yb[r]) + fabsf(ya[r]);
        const Around az(sum4(z), g), am(sum4(m), g);
        float z_before = az.before, m_before = am.before, z_after = az.after, m_after = am.after;
        floatx4 dw, inner, low;  // low: magnitude on the start's side
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            dw[r] = before;
            low[r] = m_before;
            inner[r] = -z_before - ya[r];
            before += in[r];
            m_before += m[r];
            z_before += z[r];
        }
#pragma unroll
        for (int r = 3; r >= 0; --r) {
            m_after += m[r];
            inner[r] = low[r] <= m_after ? inner[r] : z_after + rest[r];
            z_after += z[r];
            dw[r] = (dw[r] + (after + pr[r]) + inner[r]) * d.slope[r];
            after += pr[r] + pa[r];
        }
        tile.store(p.dw, dw);
    }
    if (p.dstate_in && seg == 0) io.store_columns(G, p.dstate_in + (size_t)head * N * N);
}

// Whether the segments' local pass and the chunks' matrices are one kernel: four-chunk segments (at most 1024,
// segment_chunks), and for N > 64, whose LDS leaves room for one a CU, at most 256 of them.  The whole call without
// it and with it, one sequence of 2048 tokens in 256 / 512 / 768 / 1024 segments: N = 16 40 / 44 / 51 / 65 and
// 36 / 40 / 45 / 47 us; N = 40 67 / 93 / 144 / 154 and 59 / 87 / 135 / 154; N = 64 89 / 133 / 199 / 224 and
// 79 / 112 / 175 / 216; N = 128 243 / 374 / 567 / 676 and 212 / 383 / 596 / 769.  (512 tokens, 1024 segments of
// N = 40: 139 and 144.)
bool block_form(int64_t heads, int segments, int seg_chunks, int N) {
    return segments > 1 && seg_chunks == kBlock && (N <= 64 || heads * segments <= 256);
}

// Chunks of a segment.  The last kernel takes as long as its fullest CU, w = ceil(heads segments / 256)
// workgroups of c chunks, a third longer alone on it (5.6 us a chunk at N = 40, 7.4 alone); the local pass
// adds 0.45 of that (a quarter of it for two segments, which have no Pi; 0.25 with the chunks' matrices in
// the block form), the carry 4 us and 0.35 a segment.  Measured so: 8 x 2048 x 16 x 40, 2 / 4 / 8 /
// 16 segments: 644 / 568 / 603 / 626 us; 3 x 777 x 16 x 64, 8 / 10 / 13: 161 / 145 / 156 (13 with the chunks'
// matrices apart: 171); 1 x 2048 x 16 x 64, 8 / 16 / 32: 181 / 131 / 112.
int segment_chunks(int B, int T, int H, int N) {
    const int64_t heads = (int64_t)B * H;
    const int chunks = T / kC + (T % kC != 0);
    int best = std::max(chunks, 1);
    double least = 1e30;
    for (int64_t want = 1; want == 1 || (want <= 1024 / heads && want * kBlock < chunks + kBlock); ++want) {
        const int c = std::max<int>(want == 1 ? 1 : kBlock, (int)((chunks + want - 1) / want)), S = std::max(1, (chunks + c - 1) / c);
        const int64_t w = (heads * S + 255) / 256;
        const double last = (double)w * c * (w == 1 && N <= 64 ? 1.3 : 1.0);
        const double local = S == 1 ? 0.0 : block_form(heads, S, c, N) ? 0.25 : S == 2 ? 0.25 : 0.45 * (S - 1) / S;
        const double cost = last * (1.0 + local) + (S > 2 ? 0.7 + 0.06 * S : 0.0);
        if (cost < least) {
            least = cost;
            best = c;
        }
    }
    return best;
}

struct Scratch {
    size_t frags, states, u, starts, ends, powers, powers_t, bytes;
    int segments, seg_chunks;
};

Scratch scratch_of(int B, int T, int H, int N) {
    const size_t heads = (size_t)B * H, chunks = T / kC + (T % kC != 0), NB = (N + 15) / 16;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Scratch o{};
    o.seg_chunks = segment_chunks(B, T, H, N);
    o.segments = chunks ? (int)(chunks + o.seg_chunks - 1) / o.seg_chunks : 1;
    size_t at = 0;
    auto take = [&](size_t floats) {
        const size_t here = at;
        at += up(floats * sizeof(float));
        return here;
    };
    o.frags = take(heads * chunks * kFrags * kFrag);
    o.states = take(heads * chunks * N * N);
    o.u = take(heads * chunks * NB * kFrag);
    const size_t per_seg = o.segments > 1 ? heads * o.segments * N * N : 0;
    o.starts = take(per_seg);
    o.ends = take(per_seg);
    o.powers = take(per_seg);
    o.powers_t = take(per_seg);
    o.bytes = at + 256;  // some buffer for T = 0 too
    return o;
}

// Why the sizes of a call are not supported, or nothing.
std::string unsupported(int B, int T, int H, int N) {
    if (B < 0 || T < 0 || H < 0) return "wkv7 backward: negative size";
    if (!wkv7_supported(N)) return "wkv7 backward: unsupported head size N=" + std::to_string(N);
    if (B == 0 || H == 0) return "";
    // Offsets inside a chunk of one head are 32-bit.
    if ((int64_t)H * N > (1 << 24)) return "wkv7 backward: H * N above 2^24";
    const int64_t heads = (int64_t)B * H;
    if (heads > (1 << 25) / std::max(1, T / kC + (T % kC != 0))) return "wkv7 backward: too many chunks";
    // A launch has fewer than 2^32 threads: a chunk is one wave, a segment NB.  (Heads of more than one
    // segment have at most 1024 segments together.)
    if ((heads + kXcds - 1) / kXcds * kXcds * ((N + 15) / 16) * kWave >= (int64_t)1 << 32) return "wkv7 backward: too many heads";
    return "";
}

template <int NB> void launch(const GradParams &p, hipStream_t s) {
    const int heads = p.B * p.H, grams = heads * p.chunks, segs = heads * p.segments;
    auto per_xcd = [](int units) { return (units + kXcds - 1) / kXcds; };
    if (block_form(heads, p.segments, p.seg_chunks, p.N)) {
        hipLaunchKernelGGL((wkv7_grad_block_kernel<NB>), dim3(per_xcd(segs) * kXcds), dim3(kBlockWaves<NB> * kWave), 0, s, p, segs, per_xcd(segs));
    } else {
        if (grams > 0)
            hipLaunchKernelGGL((wkv7_grad_gram_kernel<NB>), dim3(per_xcd(grams) * kXcds), dim3(kWave), 0, s, p, grams, per_xcd(grams));
        if (p.segments > 1) {
            const int locals = 2 * heads * (p.segments - 1);
            hipLaunchKernelGGL((wkv7_grad_local_kernel<NB>), dim3(per_xcd(locals) * kXcds), dim3(NB * kWave), 0, s, p, locals, per_xcd(locals));
        }
    }
    if (p.segments > 2) {
        const int carries = heads * 2 * NB;
        hipLaunchKernelGGL((wkv7_grad_carry_kernel<NB>), dim3(per_xcd(carries) * kXcds), dim3(NB * kWave), 0, s, p, carries, per_xcd(carries));
    }
    hipLaunchKernelGGL((wkv7_grad_kernel<NB>), dim3(per_xcd(segs) * kXcds), dim3(NB * kWave), 0, s, p, segs, per_xcd(segs));
}

}  // namespace
}  // namespace yuf

extern "C" size_t yuf_wkv7_scan_backward_workspace(int B, int T, int H, int N) {
    using namespace yuf;
    if (B <= 0 || H <= 0 || !unsupported(B, T, H, N).empty()) return 0;
    return scratch_of(B, T, H, N).bytes;
}

extern "C" int yuf_wkv7_scan_backward_f32(int B, int T, int H, int N, const float *r, const float *w_raw, const float *k,
                                          const float *v, const float *a, const float *b, const float *state_in,
                                          const float *dy, const float *dstate_out, float *dr, float *dw_raw, float *dk,
                                          float *dv, float *da, float *db, float *dstate_in, void *workspace,
                                          void *stream) {
    using namespace yuf;
    if (const std::string why = unsupported(B, T, H, N); !why.empty()) return fail(YUF_ERR_INVALID, why);
    if (B == 0 || H == 0) return YUF_OK;
    if (T > 0 && (!r || !w_raw || !k || !v || !a || !b || !dy || !dr || !dw_raw || !dk || !dv || !da || !db))
        return fail(YUF_ERR_INVALID, "wkv7 backward: null input/output pointer");
    if (!workspace) return fail(YUF_ERR_INVALID, "wkv7 backward: null workspace");
    if (!scratch_aligned(workspace)) return fail(YUF_ERR_INVALID, "wkv7 backward: workspace must be 256-byte aligned");
    // The gradients of one segment are written while another still reads the inputs.
    const Scratch o = scratch_of(B, T, H, N);
    const size_t tok = (size_t)B * T * H * N * sizeof(float), st = (size_t)B * H * N * N * sizeof(float);
    if (outputs_overlap<9, 8>({{r, tok}, {w_raw, tok}, {k, tok}, {v, tok}, {a, tok}, {b, tok}, {state_in, st}, {dy, tok}, {dstate_out, st}},
                              {{dr, tok}, {dw_raw, tok}, {dk, tok}, {dv, tok}, {da, tok}, {db, tok}, {dstate_in, st}, {workspace, o.bytes}}))
        return fail(YUF_ERR_INVALID, "wkv7 backward: an output or the workspace may not be (a part of) an input or another output");
    GradParams p{};
    p.B = B; p.T = T; p.H = H; p.N = N; p.chunks = T / kC + (T % kC != 0);
    p.r = r; p.w = w_raw; p.k = k; p.v = v; p.a = a; p.b = b; p.dy = dy;
    p.state_in = state_in; p.dstate_out = dstate_out;
    p.dr = dr; p.dw = dw_raw; p.dk = dk; p.dv = dv; p.da = da; p.db = db; p.dstate_in = dstate_in;
    char *base = static_cast<char *>(workspace);
    p.frags = reinterpret_cast<float *>(base + o.frags);
    p.states = reinterpret_cast<float *>(base + o.states);
    p.u = reinterpret_cast<float *>(base + o.u);
    p.starts = reinterpret_cast<float *>(base + o.starts);
    p.ends = reinterpret_cast<float *>(base + o.ends);
    p.powers = reinterpret_cast<float *>(base + o.powers);
    p.powers_t = reinterpret_cast<float *>(base + o.powers_t);
    p.segments = o.segments;
    p.seg_chunks = o.seg_chunks;
    hipStream_t s = static_cast<hipStream_t>(stream);
    switch ((N + 15) / 16) {
        case 1: launch<1>(p, s); break;
        case 2: launch<2>(p, s); break;
        case 3: launch<3>(p, s); break;
        case 4: launch<4>(p, s); break;
        default: launch<8>(p, s); break;
    }
    YUF_LAUNCH_CHECK("wkv7 backward");
    return YUF_OK;
}
