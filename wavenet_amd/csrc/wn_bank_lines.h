// Routed transforms of 1D signals of 128 ... 1024 samples: one wave runs one filter of one signal with the cascade in
// registers, from the line pieces of wn_lines.h.  As in wn_bank64.h the waves of a workgroup share an example, one filter
// each, and their results meet in LDS.
#pragma once

#include "wn_bank64.h"
#include "wn_lines.h"

namespace wn {

// taps the same in every lane: scalar registers, as far as they go
template <int NP>
__device__ __forceinline__ double bank_taps_line(const double* taps, int N, double (&a)[NP], double (&b)[NP]) {
    const double sg = bank_taps64<NP>(taps, N, a, b);
    if constexpr (NP <= 16) {
#pragma unroll
        for (int j = 0; j < NP; j++) { a[j] = w1d_uniform(a[j]); b[j] = w1d_uniform(b[j]); }
    }
    return sg;
}

// M = n / 64 consecutive samples per lane
template <int M>
__device__ __forceinline__ void bank_load_line(double (&x)[M], const BankArgs& A, size_t off, size_t block, int lane, bool from_q) {
    if (from_q) {
        signed char q[M];
        __builtin_memcpy(q, A.q + off + M * lane, M);
        const double scale = (double)A.qs[block + (M * lane) / CKPT_BLOCK];
#pragma unroll
        for (int i = 0; i < M; i++) x[i] = (double)q[i] * scale;
    } else {
        ln_load_samples<M>(A.X + off, x, lane);
    }
}
// 64 / M lanes hold a block of the checkpoint
template <int M>
__device__ __forceinline__ void bank_keep_line(const double (&x)[M], signed char* q, float* qs, int lane) {
    double m = 0;
#pragma unroll
    for (int i = 0; i < M; i++) m = ckpt_max(m, ckpt_magnitude(x[i]));
    if constexpr (M <= 32) m = ckpt_max(m, xlane<1>(m, lane));
    if constexpr (M <= 16) m = ckpt_max(m, xlane<2>(m, lane));
    if constexpr (M <= 8) m = ckpt_max(m, xlane<4>(m, lane));
    if constexpr (M <= 4) m = ckpt_max(m, xlane<8>(m, lane));
    if constexpr (M <= 2) m = ckpt_max(m, xlane<16>(m, lane));
    const float scale = ckpt_scale(m);
    const double inv = ckpt_inverse(scale);
    signed char b[M];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < M; i++) b[i] = (signed char)ckpt_quantise_fast(x[i], inv, odd);
    if (__any(odd)) {
#pragma unroll
        for (int i = 0; i < M; i++) b[i] = (signed char)ckpt_quantise(x[i], scale);
    }
    __builtin_memcpy(q + M * lane, b, M);
    if (M * lane % CKPT_BLOCK == 0) qs[M * lane / CKPT_BLOCK] = scale;
}
// out = sum over the waves of weight times the wave's n values in LDS (on top of what is there)
__device__ __forceinline__ void bank_join_line(const double* smem, int n, double* out, bool more, int waves) {
    const double* weights = smem + waves * n;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        double s = more ? out[i] : 0.0;
        for (int t = 0; t < waves; t++) s = __builtin_fma(weights[t], smem[t * n + i], s);
        out[i] = s;
    }
}

template <int NP, int M>
__global__ __launch_bounds__(256, (NP > 16 ? 1 : 2)) void k_bank_forward_line(BankArgs A) {
    constexpr int n = 64 * M;
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int lane0 = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    double* buf = smem + (size_t)wave * n;
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        int lane = lane0;
        asm volatile("" : "+v"(lane));                     // LDS and cross-lane addresses are made where they are used
        const size_t off = (size_t)e * n, block = (size_t)e * M;
        for (int j0 = 0; j0 < A.k; j0 += waves) {
            const int j = j0 + wave;
            int f = 0;
            double wgt = 0;
            const bool named = j < A.k && bank_entry(A, e, j, f, wgt);
            const bool keep = A.q_out && j0 == 0 && wave == 0;
            LinePyramid<M> p;
            if (named || keep) ln_load_samples<M>(A.X + off, p.x, lane);
            if (keep) bank_keep_line<M>(p.x, A.q_out + off, A.qs_out + block, lane);
            if (named) {
                double a[NP], b[NP], unused;
                const double sg = bank_taps_line<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
                LineLane<M> y;
                ln_forward<NP, M>(p, a, b, lane, y, unused);
                if (BANK_B_FROM_A<NP> && sg < 0) {         // every coefficient but the first
#pragma unroll
                    for (int i = 1; i < M; i++) y.v[i] = -y.v[i];
                    if (lane) y.v[0] = -y.v[0];
                }
                ln_store<M>(buf, y.v, y.v[0], lane);
            } else {
#pragma unroll
                for (int i = 0; i < M; i++) buf[64 * i + lane] = 0.0;   // times the weight: a NaN where that says there is no answer
            }
            if (lane == 0) smem[waves * n + wave] = wgt;
            __syncthreads();
            bank_join_line(smem, n, A.Y + off, j0 > 0, waves);
            __syncthreads();
        }
    }
}

// (16 taps, 777 signals of 1024 samples, two filters each: one wave per SIMD 28 us; two, with 158 registers spilled, 39 us)
template <int NP, int M, bool FROM_Q>
__global__ __launch_bounds__(256, (NP >= 16 ? 1 : 2)) void k_bank_backward_line(BankArgs A) {
    constexpr int n = 64 * M;
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int lane0 = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    double* buf = smem + (size_t)wave * n;
    const int dpad = (NP - A.N) / 2;
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        int lane = lane0;
        asm volatile("" : "+v"(lane));
        const size_t off = (size_t)e * n, block = (size_t)e * M;
        for (int j0 = 0; j0 < A.k; j0 += waves) {
            const int j = j0 + wave;
            const size_t at = (size_t)e * A.k + j;
            int f = 0;
            double wgt = 0;
            if (j < A.k && bank_entry(A, e, j, f, wgt)) {
                double a[NP], b[NP], unused, gL[NP], gH[NP], dtop[M];
                const double sg = bank_taps_line<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
                LinePyramid<M> p;
                bank_load_line<M>(p.x, A, off, block, lane, FROM_Q);
                LineLane<M> d;
                ln_load<M>(A.D + off, d, lane);
                if (BANK_B_FROM_A<NP> && sg < 0) {
#pragma unroll
                    for (int i = 1; i < M; i++) d.v[i] = -d.v[i];
                    if (lane) d.v[0] = -d.v[0];
                }
                {
                    LineLane<M> y;                         // (the coefficients themselves are not wanted)
                    ln_forward<NP, M>(p, a, b, lane, y, unused);
                }
#pragma unroll
                for (int u = 0; u < NP; u++) { gL[u] = 0; gH[u] = 0; }
                ln_backward<NP, M, true>(p, d, dtop, a, b, gL, gH, lane);
                bank_pin<NP>(gL, gH);
                double dot = 0;
#pragma unroll
                for (int i = 0; i < M; i++) dot = __builtin_fma(dtop[i], p.x[i], dot);
                ln_store_samples<M>(buf, dtop, lane);
                dot = wave_allsum(dot, lane);              // <D, F X> = <F^T D, X>
                if (A.dw && lane == 0) A.dw[at] = dot;
                const double g = bank_gradient<NP, 64>(gL, gH, A.N, nullptr, lane, sg);
                if (lane >= dpad && lane < dpad + A.N) A.grad[at * A.N + lane - dpad] = wgt * g;
            } else {
                if (j < A.k) {
                    if (lane < A.N) A.grad[at * A.N + lane] = 0.0;
                    if (A.dw && lane == 0) A.dw[at] = 0.0;
                }
#pragma unroll
                for (int i = 0; i < M; i++) buf[64 * i + lane] = 0.0;
            }
            if (lane == 0) smem[waves * n + wave] = wgt;
            __syncthreads();
            if (A.dX) bank_join_line(smem, n, A.dX + off, j0 > 0, waves);
            __syncthreads();
        }
    }
}

}  // namespace wn
