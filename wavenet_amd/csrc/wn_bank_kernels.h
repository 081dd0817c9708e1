// Transforms of examples under the filters they were routed to, and their backward pass: one workgroup per example,
// everything in LDS (the building blocks of wn_device.h), one filter after another.
#pragma once

#include "wn_bank.h"

namespace wn {

// The taps of one filter, padded from N to NP as FilterDev pads them, and the high-pass taps that follow from them.
// taps: the same address in every lane.
template <int NP>
__device__ __forceinline__ void bank_taps(const double* taps, int N, double (&a)[NP], double (&b)[NP]) {
    const int d = (NP - N) / 2;
#pragma unroll
    for (int j = 0; j < NP; j++) {
        const int t = j - d;
        a[j] = (t >= 0 && t < N) ? taps[t < 0 ? 0 : (t < N ? t : N - 1)] : 0.0;
    }
    const double sg = (d & 1) ? -1.0 : 1.0;
#pragma unroll
    for (int j = 0; j < NP; j++) b[j] = ((j & 1) ? -sg : sg) * a[NP - 1 - j];
}

// Filter and weight of entry (e, j); false where the index names no filter.
__device__ __forceinline__ bool bank_entry(const BankArgs& A, int e, int j, int& f, double& w) {
    const size_t at = (size_t)e * A.k + j;
    f = __builtin_amdgcn_readfirstlane(A.idx ? A.idx[at] : 0);
    w = A.w ? A.w[at] : 1.0;
    return f >= 0 && f < A.F;
}

// Tap k' = k + d of the gradient from the window sums (reduce_gradient, wn_kernels.h, without a FilterDev): thread k'
// returns the sum over the workgroup, the threads beyond NP return 0.  sign: that of the high-pass window sums.
template <int NP, int T>
__device__ __forceinline__ double bank_gradient(const double (&gL)[NP], const double (&gH)[NP], int N, double* red, int tid, double sign = 1.0) {
    const int d = (NP - N) / 2;
    const double sg = ((N - 1 + d) & 1) ? -sign : sign;      // (-1)^(N-1-k), k = k' - d
    double cp[NP];
#pragma unroll
    for (int kp = 0; kp < NP; kp++) cp[kp] = gL[kp] + ((kp & 1) ? -sg : sg) * gH[NP - 1 - kp];
    const int lane = tid & 63;
    const double mine = wave_scatter_sums<NP>(cp, lane);
    if constexpr (T == 64) {
        return lane < NP ? mine : 0.0;
    } else {
        __syncthreads();
        if (lane < NP) red[(tid >> 6) * NP + lane] = mine;
        __syncthreads();
        double s = 0;
        if (tid < NP) {
#pragma unroll
            for (int wv = 0; wv < T / 64; wv++) s += red[wv * NP + tid];
        }
        return s;
    }
}

// The example in LDS as a checkpoint: 16 threads per block, 4 values each.
template <int T>
__device__ __forceinline__ void bank_keep(const double* x, int n, signed char* q, float* qs, int tid) {
    const int lane = tid & 63;
    for (int base = 0; base < n; base += 4 * T) {          // the same turns in every thread
        const int at = base + 4 * tid;
        double v[4], m = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = at + i < n ? x[at + i] : 0.0;
            m = ckpt_max(m, ckpt_magnitude(v[i]));
        }
        m = ckpt_max(m, xlane<1>(m, lane));
        m = ckpt_max(m, xlane<2>(m, lane));
        m = ckpt_max(m, xlane<4>(m, lane));
        m = ckpt_max(m, xlane<8>(m, lane));
        const float scale = ckpt_scale(m);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (at + i < n) q[at + i] = (signed char)ckpt_quantise(v[i], scale);
        }
        if ((tid & 15) == 0 && at < n) qs[at / CKPT_BLOCK] = scale;
    }
}

// K >= n / T values per thread, Q = log2 K
template <int NP, int T, int Q>
__global__ __launch_bounds__(T) void k_bank_forward(BankArgs A) {
    constexpr int K = 1 << Q;
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int tid = threadIdx.x;
    const int lgR = A.lgR, lgC = A.lgC, R = 1 << lgR, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
    const bool rows = lgC > 0;                             // a signal of one column has no row stage
    double* bufX = smem;
    double* bufY1 = rows ? bufX + n : bufX;
    double* bufP = bufY1 + n;
    double* bufY = bufP + n;
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        const size_t off = (size_t)e * n;
        for (int i = tid; i < n; i += T) bufX[i] = A.X[off + i];
        __syncthreads();
        if (A.q_out) bank_keep<T>(bufX, n, A.q_out + off, A.qs_out + (size_t)e * nb, tid);
        double acc[K];
#pragma unroll
        for (int i = 0; i < K; i++) acc[i] = 0;
        for (int j = 0; j < A.k; j++) {
            int f;
            double w;
            if (!bank_entry(A, e, j, f, w)) {
#pragma unroll
                for (int i = 0; i < K; i++) acc[i] += 0.0 * w;      // nothing, unless the weight says there is no answer
                continue;
            }
            double a[NP], b[NP];
            bank_taps<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
            if (rows) fwd_pass<NP, T>(bufX, bufP, bufY1, R, 1, lgR, lgC, true, a, b, tid);
            fwd_pass<NP, T>(bufY1, bufP, bufY, 1, R, lgC, lgR, false, a, b, tid);
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i * T + tid < n) acc[i] = __builtin_fma(w, bufY[i * T + tid], acc[i]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < K; i++) {
            if (i * T + tid < n) A.Y[off + i * T + tid] = acc[i];
        }
        __syncthreads();
    }
}

template <int NP, int T, int Q>
__global__ __launch_bounds__(T) void k_bank_backward(BankArgs A) {
    constexpr int K = 1 << Q;
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int tid = threadIdx.x;
    const int lgR = A.lgR, lgC = A.lgC, R = 1 << lgR, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
    const bool rows = lgC > 0;
    double* bufX = smem;
    double* bufY1 = rows ? bufX + n : bufX;
    double* bufP = bufY1 + n;
    double* bufD = bufP + n;
    double* red = bufD + n;
    const int d = (NP - A.N) / 2;
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        const size_t off = (size_t)e * n;
        for (int i = tid; i < n; i += T)
            bufX[i] = A.X ? A.X[off + i] : (double)A.q[off + i] * (double)A.qs[(size_t)e * nb + i / CKPT_BLOCK];
        __syncthreads();
        double acc[K];
#pragma unroll
        for (int i = 0; i < K; i++) acc[i] = 0;
        for (int j = 0; j < A.k; j++) {
            const size_t at = (size_t)e * A.k + j;
            int f;
            double w;
            if (!bank_entry(A, e, j, f, w)) {
#pragma unroll
                for (int i = 0; i < K; i++) acc[i] += 0.0 * w;
                if (tid < A.N) A.grad[at * A.N + tid] = 0.0;
                if (A.dw && tid == 0) A.dw[at] = 0.0;
                continue;
            }
            double a[NP], b[NP];
            bank_taps<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
            for (int i = tid; i < n; i += T) bufD[i] = A.D[off + i];
            if (rows) fwd_pass<NP, T>(bufX, bufP, bufY1, R, 1, lgR, lgC, true, a, b, tid);
            fwd_pass_lo<NP, T>(bufY1, bufP, 1, R, lgC, lgR, false, a, tid);
            __syncthreads();
            double gL[NP], gH[NP];
#pragma unroll
            for (int u = 0; u < NP; u++) { gL[u] = 0; gH[u] = 0; }
            bwd_pass<NP, T, K, true>(bufD, bufY1, bufP, 1, R, lgC, lgR, false, true, a, b, gL, gH, tid);
            if (rows) {
                fwd_pass_lo<NP, T>(bufX, bufP, R, 1, lgR, lgC, true, a, tid);
                bwd_pass<NP, T, K, true>(bufD, bufX, bufP, R, 1, lgR, lgC, true, true, a, b, gL, gH, tid);
            }
            double dot = 0;
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i * T + tid < n) {
                    const double v = bufD[i * T + tid];
                    dot = __builtin_fma(v, bufX[i * T + tid], dot);
                    acc[i] = __builtin_fma(w, v, acc[i]);
                }
            }
            __syncthreads();
            dot = block_sum<T>(dot, red, tid);             // <D, F X> = <F^T D, X>
            if (A.dw && tid == 0) A.dw[at] = dot;
            const double g = bank_gradient<NP, T>(gL, gH, A.N, red, tid);
            if (tid >= d && tid < d + A.N) A.grad[at * A.N + tid - d] = w * g;
            __syncthreads();
        }
        if (A.dX) {
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i * T + tid < n) A.dX[off + i * T + tid] = acc[i];
            }
        }
        __syncthreads();
    }
}

}  // namespace wn
