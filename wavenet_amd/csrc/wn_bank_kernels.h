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
__device__ __forceinline__ bool bank_entry(const BankArgs& A, unsigned e, int j, int& f, double& w) {
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
        int b[4];
        ckpt_quantise4(b, v, scale);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (at + i < n) q[at + i] = (signed char)b[i];
        }
        if ((tid & 15) == 0 && at < n) qs[at / CKPT_BLOCK] = scale;
    }
}

// out = sum over the waves of weight times the wave's n values in LDS, on top of what an earlier round of filters left there
__device__ __forceinline__ void bank_join(const double* results, int stride, const double* weights, int n, double* out, bool more, int waves) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        double s = more ? out[i] : 0.0;
        for (int t = 0; t < waves; t++) s = __builtin_fma(weights[t], results[t * stride + i], s);
        out[i] = s;
    }
}

// The example is shared by the workgroup's teams of T threads, one filter each; teams of more than a wave are alone.  A
// team without a filter goes through the motions with filter 0, since the passes hold barriers, and leaves zeros.
template <int T>
struct BankTeam {
    int tid, team, teams;
    __device__ BankTeam() : tid(threadIdx.x), team(0), teams(1) {
        if constexpr (T == 64) {
            tid = threadIdx.x & 63;
            team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            teams = blockDim.x >> 6;
        }
    }
};
// doubles of LDS per team beside the shared example: stages of the transform, scratch of the sums
__host__ __device__ constexpr int bank_team_doubles(int n, bool rows, int scratch) { return (rows ? 3 : 2) * n + scratch; }

template <int NP, int T, int Q>
__global__ __launch_bounds__(T == 64 ? 256 : T) void k_bank_forward(BankArgs A) {
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const BankTeam<T> G;
    const int lgR = A.lgR, lgC = A.lgC, R = 1 << lgR, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
    const bool rows = lgC > 0;                             // a signal of one column has no row stage
    const int stride = bank_team_doubles(n, rows, 0);
    double* bufX = smem;
    double* weights = smem + n;                            // [teams]
    double* bufY = weights + G.teams + G.team * stride;
    double* bufP = bufY + n;
    double* bufY1 = rows ? bufP + n : bufX;
    for (unsigned e = blockIdx.x; e < (unsigned)A.B; e += gridDim.x) {
        const size_t off = (size_t)e * n;
        for (int i = threadIdx.x; i < n; i += blockDim.x) bufX[i] = A.X[off + i];
        __syncthreads();
        if (A.q_out && G.team == 0) bank_keep<T>(bufX, n, A.q_out + off, A.qs_out + (size_t)e * nb, G.tid);
        for (int j0 = 0; j0 < A.k; j0 += G.teams) {
            int f = 0;
            double w = 0;
            const bool named = j0 + G.team < A.k && bank_entry(A, e, j0 + G.team, f, w);
            double a[NP], b[NP];
            bank_taps<NP>(A.filters + (size_t)(named ? f : 0) * A.N, A.N, a, b);
            if (rows) fwd_pass<NP, T>(bufX, bufP, bufY1, R, 1, lgR, lgC, true, a, b, G.tid);
            fwd_pass<NP, T>(bufY1, bufP, bufY, 1, R, lgC, lgR, false, a, b, G.tid);
            if (!named) {
                for (int i = G.tid; i < n; i += T) bufY[i] = 0.0;   // times the weight: a NaN where that says there is no answer
            }
            if (G.tid == 0) weights[G.team] = w;
            __syncthreads();
            bank_join(weights + G.teams, stride, weights, n, A.Y + off, j0 > 0, G.teams);
            __syncthreads();
        }
    }
}

// 2^Q >= n / T: values per thread
template <int NP, int T, int Q>
__global__ __launch_bounds__(T == 64 ? 256 : T) void k_bank_backward(BankArgs A) {
    constexpr int K = 1 << Q;
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const BankTeam<T> G;
    const int lgR = A.lgR, lgC = A.lgC, R = 1 << lgR, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
    const bool rows = lgC > 0;
    const int stride = bank_team_doubles(n, rows, T / 64 * NP + 2);
    double* bufX = smem;
    double* weights = smem + n;
    double* bufD = weights + G.teams + G.team * stride;
    double* bufP = bufD + n;
    double* bufY1 = rows ? bufP + n : bufX;
    double* red = bufD + (rows ? 3 : 2) * n;
    const int d = (NP - A.N) / 2;
    for (unsigned e = blockIdx.x; e < (unsigned)A.B; e += gridDim.x) {
        const size_t off = (size_t)e * n;
        for (int i = threadIdx.x; i < n; i += blockDim.x)
            bufX[i] = A.X ? A.X[off + i] : (double)A.q[off + i] * (double)A.qs[(size_t)e * nb + i / CKPT_BLOCK];
        __syncthreads();
        for (int j0 = 0; j0 < A.k; j0 += G.teams) {
            const int j = j0 + G.team;
            const size_t at = (size_t)e * A.k + j;
            int f = 0;
            double w = 0;
            const bool named = j < A.k && bank_entry(A, e, j, f, w);
            double a[NP], b[NP];
            bank_taps<NP>(A.filters + (size_t)(named ? f : 0) * A.N, A.N, a, b);
            for (int i = G.tid; i < n; i += T) bufD[i] = named ? A.D[off + i] : 0.0;
            if (rows) fwd_pass<NP, T>(bufX, bufP, bufY1, R, 1, lgR, lgC, true, a, b, G.tid);
            fwd_pass_lo<NP, T>(bufY1, bufP, 1, R, lgC, lgR, false, a, G.tid);
            __syncthreads();
            double gL[NP], gH[NP];
#pragma unroll
            for (int u = 0; u < NP; u++) { gL[u] = 0; gH[u] = 0; }
            bwd_pass<NP, T, K, true>(bufD, bufY1, bufP, 1, R, lgC, lgR, false, true, a, b, gL, gH, G.tid);
            if (rows) {
                fwd_pass_lo<NP, T>(bufX, bufP, R, 1, lgR, lgC, true, a, G.tid);
                bwd_pass<NP, T, K, true>(bufD, bufX, bufP, R, 1, lgR, lgC, true, true, a, b, gL, gH, G.tid);
            }
            double dot = 0;
            for (int i = G.tid; i < n; i += T) dot = __builtin_fma(bufD[i], bufX[i], dot);
            if constexpr (T > 64) __syncthreads();
            dot = block_sum<T>(dot, red, G.tid);           // <D, F X> = <F^T D, X>
            const double g = bank_gradient<NP, T>(gL, gH, A.N, red, G.tid);
            if (j < A.k) {
                if (A.dw && G.tid == 0) A.dw[at] = named ? dot : 0.0;
                if (G.tid >= d && G.tid < d + A.N) A.grad[at * A.N + G.tid - d] = named ? w * g : 0.0;
            }
            if (!named) {
                for (int i = G.tid; i < n; i += T) bufD[i] = 0.0;   // (0 * inf in a filter would be a NaN)
            }
            if (G.tid == 0) weights[G.team] = w;
            __syncthreads();
            if (A.dX) bank_join(weights + G.teams, stride, weights, n, A.dX + off, j0 > 0, G.teams);
            __syncthreads();
        }
    }
}

}  // namespace wn
