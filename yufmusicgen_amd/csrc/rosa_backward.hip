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
// Both recurrences are chains with one dot product over D per token: latency, not
// bandwidth, bounds them.  A wave runs a chain, with its D / 64 elements per lane
// and the dot by row permutations, and the sequence is cut into segments of L
// tokens that run side by side:
//   1  each segment's end state from a zero start, in both directions, and the D
//      columns of A^L and of (A^T)^L (A = diag(lambda) H), each a chain of its own;
//   2  the carry over the segments, x <- A^L x + local, one workgroup per sequence
//      and direction, the matrix in its registers;
//   3  each segment again from its true start: forward, keeping m_t, then backward
//      with the gradients, dlambda and du summed in fp64 per segment;
//   4  those sums over the segments, in one order.
// A sequence of one segment, and D > 256 (whose A^L does not fit a workgroup's
// registers), runs 3 and 4 alone.
#include "common.h"
#include "kernels.h"

#include <algorithm>

namespace yuf {
namespace {

constexpr int kWave = 64;
constexpr int kMaxDim = 1024;
constexpr int kMaxSegDim = 256;
constexpr int kCarryThreads = 1024;

struct RosaGradParams {
    int B, T, D;
    int L, S;  // tokens of a segment, segments of a sequence
    const float *cand, *write, *read_raw, *decay, *direction, *memory_in, *dread, *dmemory;
    float *dcand, *dwrite, *dread_raw, *dmemory_in;
    // Scratch.
    float *m;        // [B, T, D]: m_t
    float *fwd;      // [B, S, D]: m before each segment (its slot s + 1 first holds segment s's local end)
    float *bwd;      // [B, S, D]: n of the token after each segment (slot s - 1 first holds segment s's local one)
    float *power;    // [2][D][D]: row j = A^L e_j, then (A^T)^L e_j
    double *sums;    // [B * S][2][D]: dlambda and du of a segment
};

// Tokens whose loads are in flight ahead of the chain.
template <int EPL> constexpr int kAhead = EPL <= 2 ? 8 : EPL == 4 ? 4 : EPL == 8 ? 2 : 1;

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
    // m <- lambda H(m) + e
    __device__ __forceinline__ void step(float (&m)[EPL], const float (&e)[EPL]) const {
        const float two = 2.0f * dot_u(m);
#pragma unroll
        for (int k = 0; k < EPL; ++k) m[k] = fmaf(lam[k], fmaf(-two, u[k], m[k]), e[k]);
    }
};

// m over tokens [t0, t1), kept in p.m where KEEP.
template <int EPL, bool KEEP>
__device__ __forceinline__ void run_forward(const RosaGradParams &p, const Chain<EPL> &c, int b, int t0, int t1,
                                            float (&m)[EPL]) {
    constexpr int K = kAhead<EPL>;
    const size_t base = (size_t)b * p.T;
    float cand[K][EPL], write[K][EPL];
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const size_t at = (base + min(t + i, t1 - 1)) * p.D;
            c.load(p.cand + at, cand[i]);
            c.load(p.write + at, write[i]);
        }
    };
    fetch(t0);
    for (int t = t0; t < t1; t += K) {
        float e[K][EPL];
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int k = 0; k < EPL; ++k) e[i][k] = c.own(k) ? sigmoidf_(write[i][k]) * tanhf(cand[i][k]) : 0.0f;
        if (t + K < t1) fetch(t + K);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (t + i >= t1) break;
            c.step(m, e[i]);
            if constexpr (KEEP) c.store(m, p.m + (base + t + i) * p.D);
        }
    }
}

// n over tokens t1 - 1 .. t0; n holds n_{t1} on entry (zero behind the last token) and n_{t0} at the end.
template <int EPL, bool GRADS>
__device__ __forceinline__ void run_backward(const RosaGradParams &p, const Chain<EPL> &c, int b, int t0, int t1,
                                             float (&n)[EPL], double (&dlam)[EPL], double (&du)[EPL]) {
    constexpr int K = kAhead<EPL> > 4 ? 4 : kAhead<EPL>;
    const size_t base = (size_t)b * p.T;
    const bool gated = p.read_raw != nullptr;
    float dread[K][EPL], rr[K][EPL], cand[K][EPL], write[K][EPL], m[K][EPL];
    auto fetch = [&](int t) {  // tokens t, t - 1, ...
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const size_t at = (base + max(t - i, t0)) * p.D;
            c.load(p.dread + at, dread[i]);
            if (gated) c.load(p.read_raw + at, rr[i]);
            if constexpr (GRADS) {
                c.load(p.cand + at, cand[i]);
                c.load(p.write + at, write[i]);
                c.load(p.m + at, m[i]);
            }
        }
    };
    fetch(t1 - 1);
    bool first = true;  // of the segment: its n_{t1} q_{t1 - 1} is the next segment's
    for (int t = t1 - 1; t >= t0; t -= K) {
        float dq[K][EPL], dr[K][EPL], gc[K][EPL], gw[K][EPL], mt[K][EPL];
#pragma unroll
        for (int i = 0; i < K; ++i)
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                const float s = gated ? sigmoidf_(rr[i][k]) : 1.0f;
                dq[i][k] = c.own(k) ? dread[i][k] * s : 0.0f;
                if constexpr (GRADS) {
                    dr[i][k] = dread[i][k] * s * (1.0f - s);
                    const float g = sigmoidf_(write[i][k]), th = tanhf(cand[i][k]);
                    gc[i][k] = g * (1.0f - th * th);
                    gw[i][k] = th * g * (1.0f - g);
                    mt[i][k] = m[i][k];
                }
            }
        if (t - K >= t0) fetch(t - K);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (t - i < t0) break;
            const size_t at = (base + t - i) * p.D;
            float pt[EPL], mu = 0.0f;
            if constexpr (GRADS) {
                mu = c.dot_u(mt[i]);
                float out[EPL];
#pragma unroll
                for (int k = 0; k < EPL; ++k) {
                    const float q = fmaf(-2.0f * mu, c.u[k], mt[i][k]);
                    if (!first) dlam[k] = fma((double)n[k], (double)q, dlam[k]);
                    out[k] = dr[i][k] * q;
                }
                if (gated) c.store(out, p.dread_raw + at);
            }
#pragma unroll
            for (int k = 0; k < EPL; ++k) pt[k] = fmaf(c.lam[k], n[k], dq[i][k]);
            const float s = c.dot_u(pt);
#pragma unroll
            for (int k = 0; k < EPL; ++k) n[k] = fmaf(-2.0f * s, c.u[k], pt[k]);
            if (t - i == p.T - 1 && p.dmemory) {
                float dm[EPL];
                c.load(p.dmemory + (size_t)b * p.D, dm);
#pragma unroll
                for (int k = 0; k < EPL; ++k) n[k] += dm[k];
            }
            if constexpr (GRADS) {
                float oc[EPL], ow[EPL];
#pragma unroll
                for (int k = 0; k < EPL; ++k) {
                    oc[k] = n[k] * gc[i][k];
                    ow[k] = n[k] * gw[i][k];
                    du[k] = fma(-2.0 * (double)s, (double)mt[i][k], fma(-2.0 * (double)mu, (double)pt[k], du[k]));
                }
                c.store(oc, p.dcand + at);
                c.store(ow, p.dwrite + at);
            }
            first = false;
        }
    }
}

// Phase 1.  Workgroups (one wave each): B (S - 1) forward chains, B (S - 1) backward
// ones, then D + D unit vectors.
template <int EPL> __global__ void __launch_bounds__(kWave) rosa_grad_local_kernel(RosaGradParams p) {
    Chain<EPL> c;
    c.init(p);
    const int per_dir = p.B * (p.S - 1);
    int id = blockIdx.x;
    float x[EPL];
    if (id < 2 * per_dir) {
#pragma unroll
        for (int k = 0; k < EPL; ++k) x[k] = 0.0f;
        const bool back = id >= per_dir;
        if (back) id -= per_dir;
        const int b = id / (p.S - 1), s = id - b * (p.S - 1);
        if (!back) {
            run_forward<EPL, false>(p, c, b, s * p.L, (s + 1) * p.L, x);
            c.store(x, p.fwd + ((size_t)b * p.S + s + 1) * p.D);
        } else {
            double none[EPL], none2[EPL];  // not read: no gradients here
            run_backward<EPL, false>(p, c, b, (s + 1) * p.L, min(p.T, (s + 2) * p.L), x, none, none2);
            c.store(x, p.bwd + ((size_t)b * p.S + s) * p.D);
        }
        return;
    }
    id -= 2 * per_dir;
    const bool back = id >= p.D;
    const int j = back ? id - p.D : id;
#pragma unroll
    for (int k = 0; k < EPL; ++k) x[k] = c.lane + kWave * k == j ? 1.0f : 0.0f;
    float zero[EPL] = {};
    for (int i = 0; i < p.L; ++i) {
        if (!back) {
            c.step(x, zero);
        } else {
#pragma unroll
            for (int k = 0; k < EPL; ++k) x[k] *= c.lam[k];
            const float two = 2.0f * c.dot_u(x);
#pragma unroll
            for (int k = 0; k < EPL; ++k) x[k] = fmaf(-two, c.u[k], x[k]);
        }
    }
    c.store(x, p.power + ((size_t)back * p.D + j) * p.D);
}

// Phase 2.  DP = D padded to 64, 128 or 256; thread (part, i) holds rows
// [part * kRows, ..) of column i of the power.
template <int DP> __global__ void __launch_bounds__(kCarryThreads) rosa_grad_carry_kernel(RosaGradParams p) {
    constexpr int kParts = kCarryThreads / DP, kRows = DP / kParts;
    __shared__ __attribute__((aligned(16))) float x[DP];
    __shared__ float partial[kParts][DP];
    const bool back = blockIdx.x >= (uint32_t)p.B;
    const int b = back ? blockIdx.x - p.B : blockIdx.x;
    const int part = threadIdx.x / DP, i = threadIdx.x % DP;
    const float *M = p.power + (size_t)back * p.D * p.D;
    float *slots = (back ? p.bwd : p.fwd) + (size_t)b * p.S * p.D;
    float w[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int j = part * kRows + r;
        w[r] = j < p.D && i < p.D ? M[(size_t)j * p.D + i] : 0.0f;
    }
    const bool live = part == 0 && i < p.D;
    // Forward: slot 0 is the initial memory, slot s + 1 <- A^L slot s + (slot s + 1).
    // Backward: slot S - 2 is the last segment's own, slot s - 1 <- (A^T)^L slot s + (slot s - 1).
    const int dir = back ? -1 : 1, steps = back ? p.S - 2 : p.S - 1;
    int s = back ? p.S - 2 : 0;
    if (part == 0) {
        float v = 0.0f;
        if (i < p.D) {
            if (back) v = slots[(size_t)s * p.D + i];
            else {
                v = p.memory_in ? p.memory_in[(size_t)b * p.D + i] : 0.0f;
                slots[i] = v;
            }
        }
        x[i] = v;
    }
    float local = live && steps > 0 ? slots[(size_t)(s + dir) * p.D + i] : 0.0f;
    __syncthreads();
    for (int n = 0; n < steps; ++n) {
        const float next = live && n + 1 < steps ? slots[(size_t)(s + 2 * dir) * p.D + i] : 0.0f;
        float acc = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) acc = fmaf(w[r], x[part * kRows + r], acc);
        partial[part][i] = acc;
        __syncthreads();
        s += dir;
        if (part == 0) {
            float v = local;
#pragma unroll
            for (int q = 0; q < kParts; ++q) v += partial[q][i];
            x[i] = i < p.D ? v : 0.0f;
            if (live) slots[(size_t)s * p.D + i] = v;
        }
        local = next;
        __syncthreads();
    }
}

// Phase 3: a wave per (sequence, segment).
template <int EPL> __global__ void __launch_bounds__(kWave) rosa_grad_kernel(RosaGradParams p) {
    Chain<EPL> c;
    c.init(p);
    const int b = blockIdx.x / p.S, s = blockIdx.x - b * p.S;
    const int t0 = s * p.L, t1 = min(p.T, t0 + p.L);
    float start[EPL], m[EPL], n[EPL];
    double dlam[EPL], du[EPL];
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
        start[k] = n[k] = 0.0f;
        dlam[k] = du[k] = 0.0;
    }
    if (s > 0) c.load(p.fwd + ((size_t)b * p.S + s) * p.D, start);
    else if (p.memory_in) c.load(p.memory_in + (size_t)b * p.D, start);
    if (s + 1 < p.S) c.load(p.bwd + ((size_t)b * p.S + s) * p.D, n);
#pragma unroll
    for (int k = 0; k < EPL; ++k) m[k] = start[k];
    if (t0 < t1) {
        run_forward<EPL, true>(p, c, b, t0, t1, m);
        run_backward<EPL, true>(p, c, b, t0, t1, n, dlam, du);
    } else if (p.dmemory) {  // no token at all: the gradient passes through
        c.load(p.dmemory + (size_t)b * p.D, n);
    }
    if (t0 < t1) {
        const float mu = c.dot_u(start);
#pragma unroll
        for (int k = 0; k < EPL; ++k) dlam[k] = fma((double)n[k], (double)fmaf(-2.0f * mu, c.u[k], start[k]), dlam[k]);
        if (s == 0) {
            float p0[EPL];
#pragma unroll
            for (int k = 0; k < EPL; ++k) p0[k] = c.lam[k] * n[k];
            const float sp = c.dot_u(p0);
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                du[k] += -2.0 * ((double)sp * start[k] + (double)mu * p0[k]);
                n[k] = fmaf(-2.0f * sp, c.u[k], p0[k]);
            }
        }
    }
    if (s == 0 && p.dmemory_in) c.store(n, p.dmemory_in + (size_t)b * p.D);
    double *out = p.sums + (size_t)blockIdx.x * 2 * p.D;
#pragma unroll
    for (int k = 0; k < EPL; ++k)
        if (c.own(k)) {
            out[c.lane + kWave * k] = dlam[k];
            out[p.D + c.lane + kWave * k] = du[k];
        }
}

// Phase 4: column sums of sums [rows][2 D], 64 columns a workgroup, 16 rows at a time.
__global__ void __launch_bounds__(1024) rosa_grad_sum_kernel(const double *sums, int rows, int D, float *ddecay,
                                                             float *ddirection) {
    __shared__ double partial[16][kWave];
    const int col = blockIdx.x * kWave + (threadIdx.x & 63), r0 = threadIdx.x >> 6;
    double s = 0.0;
    if (col < 2 * D)
        for (int r = r0; r < rows; r += 16) s += sums[(size_t)r * 2 * D + col];
    partial[r0][threadIdx.x & 63] = s;
    __syncthreads();
    if (r0 != 0 || col >= 2 * D) return;
#pragma unroll
    for (int r = 1; r < 16; ++r) s += partial[r][threadIdx.x];
    float *out = col < D ? ddecay + col : ddirection + (col - D);
    *out = (float)s;
}

// Segments of 64 tokens (128 for the longest sequences, whose carry would outlast the
// segments), from two of them up.
int segment_len(int T, int D) {
    if (D > kMaxSegDim || T < 128) return std::max(T, 1);
    return T > 8192 ? 128 : 64;
}

struct Scratch {
    size_t m, fwd, bwd, power, sums, bytes;
};

Scratch scratch_of(int B, int T, int D, int S) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Scratch o{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t here = at; at += up(n); return here; };
    o.sums = take((size_t)B * S * 2 * D * sizeof(double));
    o.m = take((size_t)B * T * D * sizeof(float));
    o.fwd = take(S > 1 ? (size_t)B * S * D * sizeof(float) : 0);
    o.bwd = take(S > 1 ? (size_t)B * S * D * sizeof(float) : 0);
    o.power = take(S > 1 ? (size_t)2 * D * D * sizeof(float) : 0);
    o.bytes = at;
    return o;
}

int segments(int T, int D) {
    const int L = segment_len(T, D);
    return std::max(1, (T + L - 1) / L);
}

template <int EPL> void launch(const RosaGradParams &p, hipStream_t s) {
    if constexpr (EPL <= kMaxSegDim / kWave) {
        if (p.S > 1) {
            hipLaunchKernelGGL((rosa_grad_local_kernel<EPL>), dim3(2 * p.B * (p.S - 1) + 2 * p.D), dim3(kWave), 0, s, p);
            hipLaunchKernelGGL((rosa_grad_carry_kernel<EPL * kWave>), dim3(2 * p.B), dim3(kCarryThreads), 0, s, p);
        }
    }
    hipLaunchKernelGGL((rosa_grad_kernel<EPL>), dim3(p.B * p.S), dim3(kWave), 0, s, p);
}

}  // namespace
}  // namespace yuf

extern "C" size_t yuf_rosa_scan_backward_workspace(int B, int T, int D) {
    using namespace yuf;
    if (B <= 0 || T < 0 || D < 1 || D > kMaxDim) return 0;
    return scratch_of(B, T, D, segments(T, D)).bytes;
}

extern "C" int yuf_rosa_scan_backward_f32(int B, int T, int D, const float *cand, const float *write,
                                          const float *read_raw, const float *decay, const float *direction,
                                          const float *memory_in, const float *dread, const float *dmemory,
                                          float *dcand, float *dwrite, float *dread_raw, float *ddecay,
                                          float *ddirection, float *dmemory_in, void *workspace, void *stream) {
    using namespace yuf;
    if (B < 0 || T < 0) return fail(YUF_ERR_INVALID, "rosa backward: negative size");
    if (D < 1 || D > kMaxDim) return fail(YUF_ERR_INVALID, "rosa backward: D must be in 1..1024");
    if (!decay || !direction || !ddecay || !ddirection)
        return fail(YUF_ERR_INVALID, "rosa backward: null decay, direction or their gradients");
    if (B > 0 && T > 0 && (!cand || !write || !dread || !dcand || !dwrite))
        return fail(YUF_ERR_INVALID, "rosa backward: null input/output pointer");
    if ((read_raw != nullptr) != (dread_raw != nullptr) && T > 0)
        return fail(YUF_ERR_INVALID, "rosa backward: read_raw and its gradient go together");
    if (B > 0 && !workspace) return fail(YUF_ERR_INVALID, "rosa backward: null workspace");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int S = segments(T, D);
    if ((int64_t)B * S > (1 << 29)) return fail(YUF_ERR_INVALID, "rosa backward: too many segments");
    RosaGradParams p{};
    p.B = B; p.T = T; p.D = D; p.L = segment_len(T, D); p.S = S;
    p.cand = cand; p.write = write; p.read_raw = read_raw; p.decay = decay; p.direction = direction;
    p.memory_in = memory_in; p.dread = dread; p.dmemory = dmemory;
    p.dcand = dcand; p.dwrite = dwrite; p.dread_raw = dread_raw; p.dmemory_in = dmemory_in;
    const Scratch o = scratch_of(B, T, D, S);
    char *base = static_cast<char *>(workspace);
    p.sums = reinterpret_cast<double *>(base + o.sums);
    p.m = reinterpret_cast<float *>(base + o.m);
    p.fwd = reinterpret_cast<float *>(base + o.fwd);
    p.bwd = reinterpret_cast<float *>(base + o.bwd);
    p.power = reinterpret_cast<float *>(base + o.power);
    if (B > 0) {
        if (D <= 64) launch<1>(p, s);
        else if (D <= 128) launch<2>(p, s);
        else if (D <= 256) launch<4>(p, s);
        else if (D <= 512) launch<8>(p, s);
        else launch<16>(p, s);
    }
    hipLaunchKernelGGL(rosa_grad_sum_kernel, dim3((2 * D + kWave - 1) / kWave), dim3(1024), 0, s, p.sums, B * S, D, ddecay,
                       ddirection);
    YUF_LAUNCH_CHECK("rosa backward");
    return YUF_OK;
}
