// Gradients of the ROSA Householder memory scan.
//
// Forward (rosa.hip): m_t = lambda * H(m_{t-1}) + e_t, e = sigmoid(write) tanh(cand),
// H(x) = x - 2 (x.u) u, q_t = H(m_t), read_t = q_t [* sigmoid(read_raw_t)], t = 1 .. T.
// With dq_t the gradient of q_t and n_t that of m_t (H is symmetric):
//     p_t = dq_t + lambda * n_{t+1},   n_t = H(p_t),   n_T also takes dmemory;
//     p_0 = lambda * n_1,              n_0 = H(p_0) = gradient of the initial memory;
//     dcand = n g (1 - c^2), dwrite = n c g (1 - g), dread_raw = dread q s (1 - s);
//     dlambda = sum_t n_t * q_{t-1},   du = -2 sum_{t >= 0} ((p_t.u) m_t + (m_t.u) p_t).
//
// Both recurrences are chains with one dot product over D per token, independent of each other:
// latency, not bandwidth, bounds them.  A chain is a wave, with D / 64 elements per lane and the
// dot by row permutations, fed from LDS.  The sequence is cut into blocks of kTok tokens, whose
// elementwise parts all waves of a workgroup share, and into ranges of R blocks:
//   1  local   each range's end state from a zero start, in both directions, and the D columns of
//              A^(R kTok) and of its transpose (A = diag(lambda) H), each a chain of its own;
//   2  carry   over the ranges, x <- A^(R kTok) x + local, one workgroup per sequence and
//              direction, the matrix in its registers;
//   3  walk    each range again from its true start, for the states at its blocks' borders;
//   4  blocks  a workgroup per block: e and dq by all waves, the two chains on two of them side by
//              side, then the gradients by all waves again, dlambda and du summed per block;
//   5  those sums over the blocks, in fp64 and one order.
// With R = 1 the carry's states are the blocks' and 3 is left out; with one range (D > 256, whose
// power does not fit a workgroup's registers) 1 and 2 are, and a sequence of one block is 4 and 5.
// 8 x 2048 x 128 with the gate (64 blocks a sequence): 12.6 + 22.2 + 16.4 + 4.0 us, 59 MB at 1.08 TB/s;
// 3 x 777 x 256: 11.9 + 21.6 + 16.6 + 3.8.  Whole segments of 64 tokens by one wave, elementwise parts
// included, took 39 + 12.6 + 93 + 6.4 us of the former.  D > 256 goes token by token along the whole sequence, twice:
// 1 x 2048 x 512 1.22 ms, x 1024 2.37 ms (eight sequences 1.35 and 3.23).
#include "common.h"
#include "kernels.h"

#include <algorithm>

namespace yuf {
namespace {

constexpr int kWave = 64;
constexpr int kMaxDim = 1024;
constexpr int kMaxCarryDim = 256;

// Tokens of a block and waves of a workgroup, by D / 64 rounded up to a power of two: two rows of
// D floats per token in LDS.
constexpr int block_tokens(int epl) { return epl <= 4 ? 32 : 128 / epl; }
constexpr int block_waves(int epl) { return epl <= 4 ? 4 : 8; }

struct RosaGradParams {
    int B, T, D;
    int S;      // blocks of a sequence
    int R, NR;  // blocks of a range, ranges of a sequence
    const float *cand, *write, *read_raw, *decay, *direction, *memory_in, *dread, *dmemory;
    float *dcand, *dwrite, *dread_raw, *dmemory_in;
    // Scratch.
    float *fwd;           // [B, S, D]: m before each block
    float *bwd;           // [B, S, D]: n of the token after each block (not the last)
    float *rfwd, *rbwd;   // [B, NR, D]: the same of ranges (fwd and bwd where R = 1)
    float *power;         // [2][D][D]: row j = A^(R kTok) e_j, then (A^T)^(R kTok) e_j
    double *sums;         // [B * S][2][D]: dlambda and du of a block
};

// Each of these keeps its relative precision, up to its exponential's |x| 2^-24 (2 |x| for tanh): the
// gradients are products of them, and 1 - sigmoid of an open gate, as a difference, would be of its rounding.
// e stays finite, so that no 0 meets an infinity.
struct Gate {
    float value, rest;  // sigmoid(x) = 1 / (1 + e) and 1 - sigmoid(x) = e / (1 + e), e = exp(-x)
    __device__ __forceinline__ explicit Gate(float x) {
        const float e = __expf(x < -80.0f ? 80.0f : -x);  // the comparison keeps NaN
        value = __builtin_amdgcn_rcpf(1.0f + e);
        rest = e * value;
    }
};
__device__ __forceinline__ float gate(float x) { return Gate(x).value; }
// With e = exp(2 x): tanh(x) = (e - 1) / (e + 1) and 1 - tanh(x)^2 = 4 e / (e + 1)^2.  e - 1 loses digits near
// 0, where the first terms of tanh's series do (up to 1/4: the next one is 2^-27 of x).
struct Tanh {
    float value, slope;
    __device__ __forceinline__ explicit Tanh(float x) {
        const float e = __expf(2.0f * (x > 40.0f ? 40.0f : x));
        const float r = __builtin_amdgcn_rcpf(e + 1.0f), q = x * x;
        const float series = fmaf(fmaf(fmaf(fmaf(62.0f / 2835.0f, q, -17.0f / 315.0f), q, 2.0f / 15.0f), q, -1.0f / 3.0f), q * x, x);
        value = fabsf(x) < 0.25f ? series : (e - 1.0f) * r;
        slope = 4.0f * e * r * r;
    }
};

template <int EPL> struct Chain {
    float lam[EPL], u[EPL];
    int lane, D;

    __device__ __forceinline__ bool own(int k) const { return lane + kWave * k < D; }
    __device__ __forceinline__ void init(const RosaGradParams &p) {
        lane = threadIdx.x & 63;
        D = p.D;
        load(p.decay, lam);
        load(p.direction, u);
    }
    __device__ __forceinline__ void load(const float *row, float (&x)[EPL]) const {
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = own(k) ? row[lane + kWave * k] : 0.0f;
    }
    __device__ __forceinline__ void store(const float (&x)[EPL], float *row) const {
#pragma unroll
        for (int k = 0; k < EPL; ++k)
            if (own(k)) row[lane + kWave * k] = x[k];
    }
    __device__ __forceinline__ float dot_u(const float (&x)[EPL]) const {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < EPL; ++k) s = fmaf(x[k], u[k], s);
        return wave_sum(s);
    }
};

// A block's rows in LDS: e_t, replaced by m_t as the forward chain passes, and dq_t, replaced by
// p_t, with the dot products of both.
template <int EPL> struct Block {
    static constexpr int kTok = block_tokens(EPL), kDim = EPL * kWave;
    float e[kTok][kDim], dq[kTok][kDim];
    float mu[kTok], s[kTok];  // m_t.u, p_t.u
};

// m <- lambda H(m) + e over a block's n tokens.  KEEP: m_t and its dot go to LDS.
template <int EPL, bool KEEP>
__device__ __forceinline__ void chain_forward(const Chain<EPL> &c, Block<EPL> &b, int n, float (&m)[EPL]) {
    float e[EPL], next[EPL];
    auto read = [&](int t, float (&x)[EPL]) {
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = b.e[t][c.lane + kWave * k];
    };
    read(0, next);
    float mu = c.dot_u(m);
    for (int t = 0; t < n; ++t) {
#pragma unroll
        for (int k = 0; k < EPL; ++k) e[k] = next[k];
        read(min(t + 1, n - 1), next);
#pragma unroll
        for (int k = 0; k < EPL; ++k) m[k] = fmaf(c.lam[k], fmaf(-2.0f * mu, c.u[k], m[k]), e[k]);
        mu = c.dot_u(m);
        if constexpr (KEEP) {
#pragma unroll
            for (int k = 0; k < EPL; ++k) b.e[t][c.lane + kWave * k] = m[k];
            if (c.lane == 0) b.mu[t] = mu;
        }
    }
}

// n <- H(dq + lambda n) over a block's tokens from its last; dmem (or nullptr) is added to n at the
// first of them, the sequence's last token.  KEEP: p_t and its dot go to LDS.
template <int EPL, bool KEEP>
__device__ __forceinline__ void chain_backward(const Chain<EPL> &c, Block<EPL> &b, int n_tok, const float *dmem, float (&n)[EPL]) {
    float dq[EPL], next[EPL], extra[EPL];
    auto read = [&](int t, float (&x)[EPL]) {
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = b.dq[t][c.lane + kWave * k];
    };
#pragma unroll
    for (int k = 0; k < EPL; ++k) extra[k] = 0.0f;
    if (dmem) c.load(dmem, extra);
    read(n_tok - 1, next);
    for (int t = n_tok - 1; t >= 0; --t) {
#pragma unroll
        for (int k = 0; k < EPL; ++k) dq[k] = next[k];
        read(max(t - 1, 0), next);
#pragma unroll
        for (int k = 0; k < EPL; ++k) dq[k] = fmaf(c.lam[k], n[k], dq[k]);
        const float s = c.dot_u(dq);
#pragma unroll
        for (int k = 0; k < EPL; ++k) n[k] = fmaf(-2.0f * s, c.u[k], dq[k]) + extra[k];
#pragma unroll
        for (int k = 0; k < EPL; ++k) extra[k] = 0.0f;
        if constexpr (KEEP) {
#pragma unroll
            for (int k = 0; k < EPL; ++k) b.dq[t][c.lane + kWave * k] = dq[k];
            if (c.lane == 0) b.s[t] = s;
        }
    }
}

// Phases 1 and 3.  Workgroups: B NR forward ranges, B NR backward ones, then (phase 1) the
// powers' columns, a wave each.
template <int EPL, bool WALK>
__global__ void __launch_bounds__(block_waves(EPL) * kWave) rosa_grad_range_kernel(RosaGradParams p) {
    constexpr int kTok = block_tokens(EPL), kWaves = block_waves(EPL), kOwn = kTok / kWaves;
    __shared__ __attribute__((aligned(16))) Block<EPL> block;
    Chain<EPL> c;
    c.init(p);
    const int wave = threadIdx.x >> 6, ranges = p.B * p.NR;
    int id = blockIdx.x;
    float x[EPL];
    if (!WALK && id >= 2 * ranges) {
        id = (id - 2 * ranges) * kWaves + wave;
        if (id >= 2 * p.D) return;  // no barrier below
        const bool back = id >= p.D;
        const int j = back ? id - p.D : id;
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = c.lane + kWave * k == j ? 1.0f : 0.0f;
        for (int i = 0; i < p.R * kTok; ++i) {  // m <- lambda H(m), n <- H(lambda n)
            if (back) {
#pragma unroll
                for (int k = 0; k < EPL; ++k) x[k] *= c.lam[k];
            }
            const float two = 2.0f * c.dot_u(x);
#pragma unroll
            for (int k = 0; k < EPL; ++k) x[k] = fmaf(-two, c.u[k], x[k]) * (back ? 1.0f : c.lam[k]);
        }
        c.store(x, p.power + ((size_t)back * p.D + j) * p.D);
        return;
    }
    const bool back = id >= ranges;
    if (back) id -= ranges;
    const int b = id / p.NR, range = id - b * p.NR;
    const int s0 = range * p.R, s1 = min(p.S, s0 + p.R);
    if (!WALK && (back ? range == 0 : range == p.NR - 1)) return;  // nobody asks for their ends
#pragma unroll
    for (int k = 0; k < EPL; ++k) x[k] = 0.0f;
    if (WALK && wave == 0) {
        if (!back && range > 0) c.load(p.rfwd + ((size_t)b * p.NR + range) * p.D, x);
        if (!back && range == 0 && p.memory_in) c.load(p.memory_in + (size_t)b * p.D, x);
        if (back && range < p.NR - 1) c.load(p.rbwd + ((size_t)b * p.NR + range) * p.D, x);
    }
    const int first = back ? s1 - 1 : s0, last = back ? s0 : s1 - 1, dir = back ? -1 : 1;
    float one[kOwn][EPL], two[kOwn][EPL];  // cand and write, or dread and read_raw, of the wave's tokens
    auto fetch = [&](int s) {
        const int t0 = s * kTok, n = min(kTok, p.T - t0);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const size_t at = ((size_t)b * p.T + t0 + min(wave + i * kWaves, n - 1)) * p.D;
            c.load((back ? p.dread : p.cand) + at, one[i]);
            if (!back) c.load(p.write + at, two[i]);
            else if (p.read_raw) c.load(p.read_raw + at, two[i]);
        }
    };
    fetch(first);
    for (int s = first;; s += dir) {
        const int t0 = s * kTok, n = min(kTok, p.T - t0);
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                const int t = wave + i * kWaves;
                const float g = back && !p.read_raw ? 1.0f : gate(two[i][k]);
                const float v = c.own(k) ? g * (back ? one[i][k] : Tanh(one[i][k]).value) : 0.0f;
                (back ? block.dq : block.e)[t][c.lane + kWave * k] = v;
            }
        if (s != last) fetch(s + dir);
        lds_barrier();
        if (wave == 0) {
            if (!back) {
                if (WALK) c.store(x, p.fwd + ((size_t)b * p.S + s) * p.D);
                chain_forward<EPL, false>(c, block, n, x);
            } else {
                if (WALK && s < p.S - 1) c.store(x, p.bwd + ((size_t)b * p.S + s) * p.D);
                chain_backward<EPL, false>(c, block, n, s == p.S - 1 && p.dmemory ? p.dmemory + (size_t)b * p.D : nullptr, x);
            }
        }
        if (s == last) break;
        lds_barrier();
    }
    if (!WALK && wave == 0) {
        if (!back) c.store(x, p.rfwd + ((size_t)b * p.NR + range + 1) * p.D);
        else c.store(x, p.rbwd + ((size_t)b * p.NR + range - 1) * p.D);
    }
}

// Phase 2.  DP = D padded to 64, 128 or 256.  Wave w holds columns 16 w + li of the power, lane
// row q (16 lanes) the rows [q DP / 4, ..) of them.  A lane reads one x-value per 64 of DP and the
// multiplications take them from their lanes by row broadcast, so that x costs LDS one word per lane and
// not per product; the four lane rows add up by row swaps: one barrier a step, 0.33 us at D = 128 (0.44 with
// every lane reading its 16 values from LDS).
// acc += sum_r (x of lane r of the lane row) w[r], even and odd r apart.  The compiler splits a row
// broadcast and its multiplication into two instructions; the s_nop covers a move of x just before.
__device__ __forceinline__ void mac_rows(float x, const float (&w)[16], float (&acc)[2]) {
    asm("s_nop 1\n"
        "v_fmac_f32_dpp %0, %2, %3 row_newbcast:0 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %4 row_newbcast:1 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %5 row_newbcast:2 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %6 row_newbcast:3 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %7 row_newbcast:4 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %8 row_newbcast:5 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %9 row_newbcast:6 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %10 row_newbcast:7 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %11 row_newbcast:8 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %12 row_newbcast:9 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %13 row_newbcast:10 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %14 row_newbcast:11 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %15 row_newbcast:12 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %16 row_newbcast:13 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %0, %2, %17 row_newbcast:14 row_mask:0xf bank_mask:0xf\n"
        "v_fmac_f32_dpp %1, %2, %18 row_newbcast:15 row_mask:0xf bank_mask:0xf\n"
        : "+v"(acc[0]), "+v"(acc[1])
        : "v"(x), "v"(w[0]), "v"(w[1]), "v"(w[2]), "v"(w[3]), "v"(w[4]), "v"(w[5]), "v"(w[6]), "v"(w[7]), "v"(w[8]),
          "v"(w[9]), "v"(w[10]), "v"(w[11]), "v"(w[12]), "v"(w[13]), "v"(w[14]), "v"(w[15]));
}

__device__ __forceinline__ float lane_rows_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <int DP> __global__ void __launch_bounds__(DP * 4) rosa_grad_carry_kernel(RosaGradParams p) {
    constexpr int kGroups = DP / 64;  // of 16 rows per lane
    __shared__ float x[2][DP];
    const bool back = blockIdx.x >= (uint32_t)p.B;
    const int b = back ? blockIdx.x - p.B : blockIdx.x;
    const int q = (threadIdx.x >> 4) & 3, li = threadIdx.x & 15, i = (threadIdx.x >> 6) * 16 + li;
    const float *M = p.power + (size_t)back * p.D * p.D;
    float *slots = (back ? p.rbwd : p.rfwd) + (size_t)b * p.NR * p.D;
    float w[kGroups][16];
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = (q * kGroups + g) * 16 + r;
            w[g][r] = j < p.D && i < p.D ? M[(size_t)j * p.D + i] : 0.0f;
        }
    const bool first_row = q == 0;
    // Forward: slot 0 is the initial memory, slot s + 1 <- power slot s + (slot s + 1).
    // Backward: slot NR - 2 is the last range's own, slot s - 1 <- power slot s + (slot s - 1).
    const int dir = back ? -1 : 1, steps = back ? p.NR - 2 : p.NR - 1, start = back ? p.NR - 2 : 0;
    // Loads and stores outside the slots, of lanes that have none to do too, go beyond the descriptor's
    // range: no branch, so a wait for a load does not also wait for the stores behind it.
    const auto rs = make_rsrc(slots, (uint32_t)((size_t)p.NR * p.D * 4));
    auto offset = [&](int n) { return first_row && i < p.D && n <= steps ? (uint32_t)((start + n * dir) * p.D + i) * 4u : kBufferOob; };
    float v = back ? buf_load(rs, offset(0)) : first_row && i < p.D && p.memory_in ? p.memory_in[(size_t)b * p.D + i] : 0.0f;
    if (first_row) x[0][i] = v;
    buf_store(v, rs, offset(0));
    constexpr int kAhead = 4;
    float local[kAhead];  // 0 but in the first lane row
#pragma unroll
    for (int n = 0; n < kAhead; ++n) local[n] = buf_load(rs, offset(n + 1));
    lds_barrier();
    for (int n0 = 0; n0 < steps; n0 += kAhead) {
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const int n = n0 + e;  // steps past the last write nothing
            float acc[2] = {local[e], 0.0f};
            local[e] = buf_load(rs, offset(n + 1 + kAhead));
            float now[kGroups];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) now[g] = x[n & 1][(q * kGroups + g) * 16 + li];
#pragma unroll
            for (int g = 0; g < kGroups; ++g) mac_rows(now[g], w[g], acc);
            v = lane_rows_sum(acc[0] + acc[1]);
            if (first_row) x[(n + 1) & 1][i] = v;
            buf_store(v, rs, offset(n + 1));
            lds_barrier();
        }
    }
}

// Phase 4: a workgroup per (sequence, block).  Wave w owns tokens w, w + kWaves, ..
template <int EPL> __global__ void __launch_bounds__(block_waves(EPL) * kWave) rosa_grad_kernel(RosaGradParams p) {
    constexpr int kTok = block_tokens(EPL), kWaves = block_waves(EPL), kOwn = kTok / kWaves, kDim = EPL * kWave;
    union Lds {
        Block<EPL> block;
        float sums[kWaves][2][kDim];
    };
    __shared__ __attribute__((aligned(16))) Lds lds;
    Block<EPL> &block = lds.block;
    __shared__ float start_mu;
    Chain<EPL> c;
    c.init(p);
    const int wave = threadIdx.x >> 6, b = blockIdx.x / p.S, s = blockIdx.x - b * p.S;
    const int t0 = s * kTok, n = min(kTok, p.T - t0);
    const bool gated = p.read_raw != nullptr;
    const size_t base = ((size_t)b * p.T + t0) * p.D;
    const float *dmem = s == p.S - 1 && p.dmemory ? p.dmemory + (size_t)b * p.D : nullptr;
    double *out = p.sums + (size_t)blockIdx.x * 2 * p.D;
    if (n <= 0) {  // no token at all: the memory's gradient passes through
        float x[EPL] = {};
        if (dmem) c.load(dmem, x);
        if (wave == 0 && p.dmemory_in) c.store(x, p.dmemory_in + (size_t)b * p.D);
        for (int i = threadIdx.x; i < 2 * p.D; i += kWaves * kWave) out[i] = 0.0;
        return;
    }
    float dr[kOwn][EPL], gc[kOwn][EPL], gw[kOwn][EPL];
    {
        float cand[kOwn][EPL], write[kOwn][EPL], dread[kOwn][EPL], rr[kOwn][EPL];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const size_t at = base + (size_t)min(wave + i * kWaves, n - 1) * p.D;
            c.load(p.cand + at, cand[i]);
            c.load(p.write + at, write[i]);
            c.load(p.dread + at, dread[i]);
            if (gated) c.load(p.read_raw + at, rr[i]);
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                const int t = wave + i * kWaves, at = c.lane + kWave * k;
                const Gate g(write[i][k]);
                const Tanh th(cand[i][k]);
                block.e[t][at] = c.own(k) ? g.value * th.value : 0.0f;
                gc[i][k] = g.value * th.slope;
                gw[i][k] = th.value * g.value * g.rest;
                float dq = dread[i][k];
                if (gated) {
                    const Gate r(rr[i][k]);
                    dq *= r.value;
                    dr[i][k] = dq * r.rest;
                }
                block.dq[t][at] = c.own(k) ? dq : 0.0f;
            }
    }
    // m before the block, for the first token's q_{t-1} and (block 0) the initial memory's terms.
    float start[EPL];
#pragma unroll
    for (int k = 0; k < EPL; ++k) start[k] = 0.0f;
    if (s > 0) c.load(p.fwd + ((size_t)b * p.S + s) * p.D, start);
    else if (p.memory_in) c.load(p.memory_in + (size_t)b * p.D, start);
    lds_barrier();
    if (wave == 0) {
        float m[EPL];
#pragma unroll
        for (int k = 0; k < EPL; ++k) m[k] = start[k];
        const float mu = c.dot_u(start);
        if (c.lane == 0) start_mu = mu;
        chain_forward<EPL, true>(c, block, n, m);
    } else if (wave == 1) {
        float x[EPL];
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = 0.0f;
        if (s + 1 < p.S) c.load(p.bwd + ((size_t)b * p.S + s) * p.D, x);
        chain_backward<EPL, true>(c, block, n, dmem, x);
    }
    lds_barrier();
    float dlam[EPL], du[EPL];
#pragma unroll
    for (int k = 0; k < EPL; ++k) dlam[k] = du[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        const int t = wave + i * kWaves;
        if (t >= n) break;
        const size_t at = base + (size_t)t * p.D;
        const float mu = block.mu[t], sp = block.s[t], mu_before = t > 0 ? block.mu[t - 1] : start_mu;
        float oc[EPL], ow[EPL], orr[EPL], x[EPL], extra[EPL];
#pragma unroll
        for (int k = 0; k < EPL; ++k) extra[k] = 0.0f;
        if (dmem && t == n - 1) c.load(dmem, extra);
#pragma unroll
        for (int k = 0; k < EPL; ++k) {
            const int d = c.lane + kWave * k;
            const float m = block.e[t][d], pt = block.dq[t][d], before = t > 0 ? block.e[max(t - 1, 0)][d] : start[k];
            x[k] = fmaf(-2.0f * sp, c.u[k], pt) + extra[k];
            oc[k] = x[k] * gc[i][k];
            ow[k] = x[k] * gw[i][k];
            if (gated) orr[k] = dr[i][k] * fmaf(-2.0f * mu, c.u[k], m);
            dlam[k] = fmaf(x[k], fmaf(-2.0f * mu_before, c.u[k], before), dlam[k]);
            du[k] = fmaf(-2.0f * sp, m, fmaf(-2.0f * mu, pt, du[k]));
        }
        c.store(oc, p.dcand + at);
        c.store(ow, p.dwrite + at);
        if (gated) c.store(orr, p.dread_raw + at);
        if (s == 0 && t == 0) {
            // p_0 = lambda n_1, n_0 = H(p_0)
            float p0[EPL];
#pragma unroll
            for (int k = 0; k < EPL; ++k) p0[k] = c.lam[k] * x[k];
            const float s0 = c.dot_u(p0);
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                du[k] = fmaf(-2.0f * s0, start[k], fmaf(-2.0f * mu_before, p0[k], du[k]));
                p0[k] = fmaf(-2.0f * s0, c.u[k], p0[k]);
            }
            if (p.dmemory_in) c.store(p0, p.dmemory_in + (size_t)b * p.D);
        }
    }
    lds_barrier();  // the block's rows are done with
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
        lds.sums[wave][0][c.lane + kWave * k] = dlam[k];
        lds.sums[wave][1][c.lane + kWave * k] = du[k];
    }
    lds_barrier();
    for (int i = threadIdx.x; i < 2 * kDim; i += kWaves * kWave) {
        const int which = i / kDim, d = i % kDim;
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) t += (double)lds.sums[w][which][d];
        if (d < p.D) out[which * p.D + d] = t;
    }
}

// Phase 5: column sums of sums [rows][2 D], 16 columns a workgroup, 64 rows at a time.
__global__ void __launch_bounds__(1024) rosa_grad_sum_kernel(const double *sums, int rows, int D, float *ddecay,
                                                             float *ddirection) {
    __shared__ double partial[kWave][17];
    const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
    double s = 0.0;
    if (col < 2 * D)
        for (int r = r0; r < rows; r += 64) s += sums[(size_t)r * 2 * D + col];
    partial[r0][c] = s;
    __syncthreads();
    if (r0 >= 16) return;
    // Column r0 of the 16, by the lanes of a row of 16: four rows each, then the row's sum.
    double t = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q) t += partial[4 * c + q][r0];
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) t += __shfl_xor(t, d);
    const int out = blockIdx.x * 16 + r0;
    if (c == 0 && out < 2 * D) (out < D ? ddecay[out] : ddirection[out - D]) = (float)t;
}

int epl_of(int D) { return D <= 64 ? 1 : D <= 128 ? 2 : D <= 256 ? 4 : D <= 512 ? 8 : 16; }

// Blocks of a sequence and of a range.  A range costs the carry a step (0.33 us at D = 128) and each of its
// blocks costs the local pass and the walk, which one-block ranges need not, one (12 us together): R grows as
// the root of the sequence.  The whole call, one sequence of D = 128 with the gate, us:
//     blocks    128   160   256   512   768  1024  2048  3072  4096  8192 16384
//     R = 1      65    75   105   188   275   360
//     R = 4      80    84    92   117   145   172   280   440   550
//     R = 8     124   126   131   152   167   183   245   327   403   827
//     R = 16    219   221   224   247   259   271   313   368   411   689  1429
//     R = 32    412   413   417   453   464   474   516   558   588   811  1283
// (R = 2 would gain 4 to 15 us around 160 blocks.)  D = 64 and 256 cross near the same places, and for eight
// sequences, whose blocks fill the GPU, the R picked is within 6 % of the best.
struct Cut {
    int S, R, NR;
};
Cut cut_of(int T, int D) {
    const int tok = block_tokens(epl_of(D));
    Cut c{};
    c.S = std::max(1, T / tok + (T % tok != 0));
    c.R = D > kMaxCarryDim ? c.S : c.S <= 128 ? 1 : c.S <= 768 ? 4 : c.S <= 4096 ? 8 : c.S <= 12288 ? 16 : 32;
    c.NR = (c.S + c.R - 1) / c.R;
    return c;
}

struct Scratch {
    size_t fwd, bwd, rfwd, rbwd, power, sums, bytes;
};

Scratch scratch_of(int B, int T, int D) {
    const Cut c = cut_of(T, D);
    Scratch o{};
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    const size_t states = (size_t)B * c.S * D * sizeof(float), ranges = (size_t)B * c.NR * D * sizeof(float);
    o.sums = take((size_t)B * c.S * 2 * D * sizeof(double));
    o.fwd = take(c.S > 1 ? states : 0);
    o.bwd = take(c.S > 1 ? states : 0);
    o.rfwd = c.R > 1 ? take(ranges) : o.fwd;
    o.rbwd = c.R > 1 ? take(ranges) : o.bwd;
    o.power = take(c.NR > 1 ? (size_t)2 * D * D * sizeof(float) : 0);
    o.bytes = at;
    return o;
}

// Why the sizes of a call are not supported, or null.
const char *unsupported(int B, int T, int D) {
    if (B < 0 || T < 0) return "rosa backward: negative size";
    if (D < 1 || D > kMaxDim) return "rosa backward: D must be in 1..1024";
    if ((int64_t)B * cut_of(T, D).S >= (1 << 22)) return "rosa backward: too many blocks";  // 2^32 threads a launch
    return nullptr;
}

template <int EPL> void launch(const RosaGradParams &p, hipStream_t s) {
    constexpr int kWaves = block_waves(EPL);
    const dim3 wg(kWaves * kWave);
    if constexpr (EPL * kWave <= kMaxCarryDim) {
        if (p.NR > 1) {
            hipLaunchKernelGGL((rosa_grad_range_kernel<EPL, false>), dim3(2 * p.B * p.NR + (2 * p.D + kWaves - 1) / kWaves), wg, 0, s, p);
            hipLaunchKernelGGL((rosa_grad_carry_kernel<EPL * kWave>), dim3(2 * p.B), dim3(EPL * kWave * 4), 0, s, p);
        }
    }
    if (p.R > 1 && p.S > 1) hipLaunchKernelGGL((rosa_grad_range_kernel<EPL, true>), dim3(2 * p.B * p.NR), wg, 0, s, p);
    hipLaunchKernelGGL((rosa_grad_kernel<EPL>), dim3(p.B * p.S), wg, 0, s, p);
}

}  // namespace
}  // namespace yuf

extern "C" size_t yuf_rosa_scan_backward_workspace(int B, int T, int D) {
    using namespace yuf;
    if (B <= 0 || unsupported(B, T, D)) return 0;
    return scratch_of(B, T, D).bytes;
}

extern "C" int yuf_rosa_scan_backward_f32(int B, int T, int D, const float *cand, const float *write,
                                          const float *read_raw, const float *decay, const float *direction,
                                          const float *memory_in, const float *dread, const float *dmemory,
                                          float *dcand, float *dwrite, float *dread_raw, float *ddecay,
                                          float *ddirection, float *dmemory_in, void *workspace, void *stream) {
    using namespace yuf;
    if (const char *why = unsupported(B, T, D)) return fail(YUF_ERR_INVALID, why);
    if (!decay || !direction || !ddecay || !ddirection)
        return fail(YUF_ERR_INVALID, "rosa backward: null decay, direction or their gradients");
    if (B > 0 && T > 0 && (!cand || !write || !dread || !dcand || !dwrite))
        return fail(YUF_ERR_INVALID, "rosa backward: null input/output pointer");
    if ((read_raw != nullptr) != (dread_raw != nullptr) && T > 0)
        return fail(YUF_ERR_INVALID, "rosa backward: read_raw and its gradient go together");
    if (B > 0 && !workspace) return fail(YUF_ERR_INVALID, "rosa backward: null workspace");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Cut cut = cut_of(T, D);
    if (!scratch_aligned(workspace)) return fail(YUF_ERR_INVALID, "rosa backward: workspace must be 256-byte aligned");
    // The gradients of one block are written while another still reads the inputs.
    const Scratch o = scratch_of(B, T, D);
    const size_t tok = (size_t)B * T * D * sizeof(float), mem = (size_t)B * D * sizeof(float), vec = (size_t)D * sizeof(float);
    if (outputs_overlap<8, 7>({{cand, tok}, {write, tok}, {read_raw, tok}, {decay, vec}, {direction, vec}, {memory_in, mem}, {dread, tok}, {dmemory, mem}},
                              {{dcand, tok}, {dwrite, tok}, {dread_raw, tok}, {ddecay, vec}, {ddirection, vec}, {dmemory_in, mem}, {workspace, o.bytes}}))
        return fail(YUF_ERR_INVALID, "rosa backward: an output or the workspace may not be (a part of) an input or another output");
    RosaGradParams p{};
    p.B = B; p.T = T; p.D = D; p.S = cut.S; p.R = cut.R; p.NR = cut.NR;
    p.cand = cand; p.write = write; p.read_raw = read_raw; p.decay = decay; p.direction = direction;
    p.memory_in = memory_in; p.dread = dread; p.dmemory = dmemory;
    p.dcand = dcand; p.dwrite = dwrite; p.dread_raw = dread_raw; p.dmemory_in = dmemory_in;
    char *base = static_cast<char *>(workspace);
    p.sums = reinterpret_cast<double *>(base + o.sums);
    p.fwd = reinterpret_cast<float *>(base + o.fwd);
    p.bwd = reinterpret_cast<float *>(base + o.bwd);
    p.rfwd = reinterpret_cast<float *>(base + o.rfwd);
    p.rbwd = reinterpret_cast<float *>(base + o.rbwd);
    p.power = reinterpret_cast<float *>(base + o.power);
    if (B > 0) {
        switch (epl_of(D)) {
            case 1: launch<1>(p, s); break;
            case 2: launch<2>(p, s); break;
            case 4: launch<4>(p, s); break;
            case 8: launch<8>(p, s); break;
            default: launch<16>(p, s); break;
        }
    }
    hipLaunchKernelGGL(rosa_grad_sum_kernel, dim3((2 * D + 15) / 16), dim3(1024), 0, s, p.sums, B * cut.S, D, ddecay,
                       ddirection);
    YUF_LAUNCH_CHECK("rosa backward");
    return YUF_OK;
}
