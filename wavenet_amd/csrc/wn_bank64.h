// Routed transforms of 64x64 examples: one wave runs one filter of one example, lane = row or column, from the register
// pieces of wn_wave64.h.  The waves of a workgroup share an example, one filter each; their results meet in the LDS tiles
// that they transpose through anyway, and every wave adds up and stores a share of the columns.
#pragma once

#include "wn_bank_kernels.h"
#include "wn_wave64.h"

namespace wn {

// From 16 taps on the high-pass taps are signed low-pass taps, as in k_train64 (wn_wave64.h): coefficient (r, c) is then off by
// s_r s_c, s = sg on the high-pass indices and 1 on index 0.
template <int NP>
constexpr bool BANK_B_FROM_A = (NP >= 16);
template <int NP>
__device__ __forceinline__ double bank_taps64(const double* taps, int N, double (&a)[NP], double (&b)[NP]) {
    bank_taps<NP>(taps, N, a, b);
    if constexpr (BANK_B_FROM_A<NP>) {
#pragma unroll
        for (int j = 0; j < NP; j++) b[j] = (j & 1) ? -a[NP - 1 - j] : a[NP - 1 - j];
        return (((NP - N) / 2) & 1) ? -1.0 : 1.0;
    }
    return 1.0;
}
// v[i] (other index: the lane) times s_i s_lane
__device__ __forceinline__ void bank_signs64(double (&v)[64], double sg, int lane) {
    const double sl = lane ? sg : 1.0;
    v[0] *= sl;
#pragma unroll
    for (int i = 1; i < 64; i++) v[i] *= sl * sg;
}

// ---- checkpoints ------------------------------------------------------------------------------------------
// Register c of lane l is the value at column c, row l, and a block of the checkpoint is a column.  Bytes travel as
// dwords of four rows: lane 4 g + i moves rows 4 g ... 4 g + 3 of columns 4 m + i, and the four lanes of a quad exchange.

template <int I>
__device__ __forceinline__ int quad_lane(int v) {   // of the quad's lane I
    return __builtin_amdgcn_update_dpp(0, v, I * 0x55, 0xF, 0xF, true);
}

struct Bank64Q {
    int d[16];
    float scale;           // of column `lane`
};
__device__ __forceinline__ void bank_fetch64_q(Bank64Q& c, const signed char* q, const float* qs, int lane) {
    const int* p = reinterpret_cast<const int*>(q);
    asm volatile("" : "+s"(p), "+s"(qs));
    c.scale = qs[lane];
    p += 16 * (lane & 3) + (lane >> 2);
#pragma unroll
    for (int m = 0; m < 16; m++) c.d[m] = p[64 * m];
}
__device__ __forceinline__ void bank_values64_q(double (&v)[64], const Bank64Q& c, int lane) {
    const int shift = 24 - 8 * (lane & 3);
#pragma unroll
    for (int m = 0; m < 16; m++) {
        const int b[4] = {quad_lane<0>(c.d[m]), quad_lane<1>(c.d[m]), quad_lane<2>(c.d[m]), quad_lane<3>(c.d[m])};
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float sc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, c.scale), 4 * m + t));
            // a byte times a float scale is exact in a double
            v[4 * m + t] = (double)((b[t] << shift) >> 24) * (double)sc;
        }
    }
}

// Largest magnitude of every column: lane c returns that of column c.  On lane bit t a lane keeps the half of its columns
// whose number has that bit equal to its own.  EXACT: NaN wins; else it may be lost.  The two wide exchanges are the
// hardware's swaps of half waves and half of their halves, which leave both operands where the maximum wants them.
template <bool EXACT>
__device__ __forceinline__ double bank_larger(double a, double b) {
    if constexpr (EXACT) return ckpt_max(ckpt_magnitude(a), ckpt_magnitude(b));
    else return ckpt_max_quick(a, b);
}
template <int H, bool EXACT>
__device__ __forceinline__ void bank_column_max(double (&m)[32], int lane) {
    const bool up = (lane & H) != 0;
#pragma unroll
    for (int i = 0; i < H; i++) {
        const double keep = up ? m[i + H] : m[i], send = up ? m[i] : m[i + H];
        m[i] = bank_larger<EXACT>(keep, xlane<H>(send, lane));
    }
    if constexpr (H > 1) bank_column_max<H / 2, EXACT>(m, lane);
}
template <int W, bool EXACT>
__device__ __forceinline__ double bank_swap_max(double a, double b) {
    auto swap = [](unsigned x, unsigned y) {
        if constexpr (W == 32) return __builtin_amdgcn_permlane32_swap(x, y, false, false);
        else return __builtin_amdgcn_permlane16_swap(x, y, false, false);
    };
    const auto lo = swap((unsigned)__double2loint(a), (unsigned)__double2loint(b));
    const auto hi = swap((unsigned)__double2hiint(a), (unsigned)__double2hiint(b));
    return bank_larger<EXACT>(__hiloint2double((int)hi[0], (int)lo[0]), __hiloint2double((int)hi[1], (int)lo[1]));
}
template <bool EXACT>
__device__ __forceinline__ double bank_max64(const double (&v)[64], int lane) {
    double m[32];
#pragma unroll
    for (int i = 0; i < 32; i++) m[i] = bank_swap_max<32, EXACT>(v[i], v[i + 32]);
#pragma unroll
    for (int i = 0; i < 16; i++) m[i] = bank_swap_max<16, EXACT>(m[i], m[i + 16]);
    bank_column_max<8, EXACT>(m, lane);
    return m[0];
}

// Columns 4 m ... 4 m + 3 for the groups m = first, first + step, ... (the registers are indexed at compile time), their scales
// included: a maximum that lost a NaN is odd to the wave that quantises the NaN's column, and to no other.
template <bool EXACT>
__device__ __forceinline__ bool bank_keep64(const double (&v)[64], signed char* q, float* qs, int first, int step, int lane) {
    const float scale = ckpt_scale(bank_max64<EXACT>(v, lane));
    const double inv = ckpt_inverse(scale);
    bool odd = false;
    if ((lane >> 2) % step == first) qs[lane] = scale;
    int* out = reinterpret_cast<int*>(q) + 16 * (lane & 3) + (lane >> 2);
    const int shift = 8 * (lane & 3);
    int turn = first;
#pragma unroll
    for (int m = 0; m < 16; m++) {
        if (m != turn) continue;                           // the same in every lane
        turn += step;
        unsigned own = 0;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            int b;
            if constexpr (EXACT) {
                b = ckpt_quantise(v[4 * m + t], __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), 4 * m + t)));
            } else {
                b = ckpt_quantise_fast(v[4 * m + t],
                                       __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(inv), 4 * m + t),
                                                        __builtin_amdgcn_readlane(__double2loint(inv), 4 * m + t)), odd);
            }
            own |= (unsigned)(b & 0xFF) << (8 * t);
        }
        const int s0 = quad_lane<0>((int)own), s1 = quad_lane<1>((int)own), s2 = quad_lane<2>((int)own), s3 = quad_lane<3>((int)own);
        out[64 * m] = ((s0 >> shift) & 0xFF) | (((s1 >> shift) & 0xFF) << 8) | (((s2 >> shift) & 0xFF) << 16) | (((s3 >> shift) & 0xFF) << 24);
    }
    return odd;
}

// Columns wave, wave + waves, ... of the sum of the waves' tiles times their weights: to memory, or on top of what an
// earlier round of filters left there.  BY_ROW: tile[row * 65 + c], else tile[c * 65 + row].
template <bool BY_ROW>
__device__ __forceinline__ void bank_join64(const double* smem, double* out, bool more, int wave, int waves, int lane) {
    const double* weights = smem + waves * W64_TILE;
    for (int c0 = wave; c0 < 64; c0 += 8 * waves) {
        double s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = c0 + i * waves;
            s[i] = (more && c < 64) ? out[64 * c + lane] : 0.0;
        }
        for (int t = 0; t < waves; t++) {
            const double wgt = weights[t];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int c = c0 + i * waves;
                if (c < 64) s[i] = __builtin_fma(wgt, smem[t * W64_TILE + (BY_ROW ? lane * 65 + c : c * 65 + lane)], s[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = c0 + i * waves;
            if (c < 64) out[64 * c + lane] = s[i];
        }
    }
}

// The window sums as values that the compiler has to have here: it would otherwise put off the whole correlation to where
// the sums are used, and hold every line's values until then (4 taps: 560 registers in scratch memory).
template <int NP>
__device__ __forceinline__ void bank_pin(double (&gL)[NP], double (&gH)[NP]) {
#pragma unroll
    for (int u = 0; u < NP; u++) asm volatile("" : "+v"(gL[u]), "+v"(gH[u]));
}

// ---- kernels ----------------------------------------------------------------------------------------------
// (An example is 32 KiB: e + gridDim.x stays far below 2^31.)

// The next example's rows are on their way while this one's columns are transformed (the registers are there, at one wave per
// SIMD); the store of the weight and the join wait for them.
template <int NP>
__global__ __launch_bounds__(256, 1) void k_bank_forward64(BankArgs A) {
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    double x[64];
    if (blockIdx.x < A.B) w64_load_rows(x, A.X + (size_t)blockIdx.x * 4096, lane);
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        const size_t off = (size_t)e * 4096;
        unsigned tile_off = (unsigned)wave * W64_TILE;
        asm volatile("" : "+s"(tile_off));
        double* tile = smem + tile_off;
        double* trow = tile + lane * 65;
        for (int j0 = 0; j0 < A.k; j0 += waves) {
            const int j = j0 + wave;
            double v[64], w[64], p[64];
            int f = 0;
            double wgt = 0;
            const bool named = j < A.k && bank_entry(A, e, j, f, wgt);
            if (j0 == 0 && A.q_out) {
                float* qs = A.qs_out + (size_t)e * 64;
                const bool odd = bank_keep64<false>(x, A.q_out + off, qs, wave, waves, lane);
                if (__any(odd)) bank_keep64<true>(x, A.q_out + off, qs, wave, waves, lane);
            }
            if (named) {
                double a[NP], b[NP];
                const double sg = bank_taps64<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
                w64_fwd_levels<NP, 5, true>(x, p, w, trow, a, b);
                if (j0 + waves >= A.k && e + gridDim.x < A.B) w64_load_rows(x, A.X + off + (size_t)gridDim.x * 4096, lane);
                w64_read_transposed(w, tile, lane);
                w64_fwd_levels<NP, 5, false>(w, p, v, trow, a, b);   // v = Y(:, lane)
                if (BANK_B_FROM_A<NP> && sg < 0) bank_signs64(v, sg, lane);
#pragma unroll
                for (int r = 0; r < 64; r++) trow[r] = v[r];
            } else {
                if (j0 + waves >= A.k && e + gridDim.x < A.B) w64_load_rows(x, A.X + off + (size_t)gridDim.x * 4096, lane);
#pragma unroll
                for (int r = 0; r < 64; r++) trow[r] = 0.0;           // times the weight: a NaN where that says there is no answer
            }
            if (lane == 0) smem[waves * W64_TILE + wave] = wgt;
            __syncthreads();
            bank_join64<false>(smem, A.Y + off, j0 > 0, wave, waves, lane);
            __syncthreads();
        }
    }
}

template <int NP, bool FROM_Q>
__global__ __launch_bounds__(256, 1) void k_bank_backward64(BankArgs A) {
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int dpad = (NP - A.N) / 2;
    double d[64];
    Bank64Q c;
    const auto fetch = [&](int e) {
        w64_load_rows(d, A.D + (size_t)e * 4096, lane);
        if constexpr (FROM_Q) bank_fetch64_q(c, A.q + (size_t)e * 4096, A.qs + (size_t)e * 64, lane);
    };
    if (blockIdx.x < A.B) fetch(blockIdx.x);
    for (int e = blockIdx.x; e < A.B; e += gridDim.x) {
        const size_t off = (size_t)e * 4096;
        unsigned tile_off = (unsigned)wave * W64_TILE;
        asm volatile("" : "+s"(tile_off));
        double* tile = smem + tile_off;
        double* trow = tile + lane * 65;
        for (int j0 = 0; j0 < A.k; j0 += waves) {
            const int j = j0 + wave;
            const size_t at = (size_t)e * A.k + j;
            int f = 0;
            double wgt = 0;
            if (j < A.k && bank_entry(A, e, j, f, wgt)) {
                double a[NP], b[NP], w[64];
                const double sg = bank_taps64<NP>(A.filters + (size_t)f * A.N, A.N, a, b);
                w64_transpose(d, tile, lane);                          // d[r] = errors on Y(r, lane)
                if (BANK_B_FROM_A<NP> && sg < 0) bank_signs64(d, sg, lane);
                {
                    double v[64], p[64];
                    if constexpr (FROM_Q) bank_values64_q(v, c, lane);
                    else w64_load_rows(v, A.X + off, lane);
                    w64_fwd_levels<NP, 5, true>(v, p, w, trow, a, b);
                    w64_read_transposed(w, tile, lane);                // w[r] = Y1(r, lane)
                    w64_pyramid_to_tile<NP, 5>(w, p, trow, a);
                }
                double gL[NP], gH[NP];
#pragma unroll
                for (int u = 0; u < NP; u++) { gL[u] = 0; gH[u] = 0; }
                w64_bwd_levels<NP, 0, W64_TOP_TILE, true>(d, w, trow, a, b, gL, gH);   // columns
                bank_pin<NP>(gL, gH);
                w64_read_transposed(d, tile, lane);                    // d[c] = errors on Y1(lane, c)
                if constexpr (FROM_Q) {
                    bank_fetch64_q(c, A.q + off, A.qs + (size_t)e * 64, lane);      // again, and not held in registers until here
                    bank_values64_q(w, c, lane);
                } else {
                    w64_load_rows(w, A.X + off, lane);
                }
                {
                    double p[64];
                    w64_pyramid_to_tile<NP, 5>(w, p, trow, a);
                }
                w64_bwd_levels<NP, 0, W64_TOP_TILE, true>(d, w, trow, a, b, gL, gH);   // rows: trow[c] = errors on X(lane, c)
                bank_pin<NP>(gL, gH);
                double dot = 0;
#pragma unroll
                for (int i = 0; i < 64; i++) dot = __builtin_fma(trow[i], w[i], dot);
                dot = wave_allsum(dot, lane);                          // <D, F X> = <F^T D, X>
                if (A.dw && lane == 0) A.dw[at] = dot;
                const double g = bank_gradient<NP, 64>(gL, gH, A.N, nullptr, lane, sg);
                if (lane >= dpad && lane < dpad + A.N) A.grad[at * A.N + lane - dpad] = wgt * g;
            } else {
                if (j < A.k) {
                    if (lane < A.N) A.grad[at * A.N + lane] = 0.0;
                    if (A.dw && lane == 0) A.dw[at] = 0.0;
                }
#pragma unroll
                for (int i = 0; i < 64; i++) trow[i] = 0.0;
            }
            if (lane == 0) smem[waves * W64_TILE + wave] = wgt;
            {   // The errors that come next are asked for before the results are put together, which waits for them (forward and
                // backward pass of 4096 examples from the checkpoint all the same 315 -> 305 us).
                const int next = j0 + waves < A.k ? e : e + (int)gridDim.x;
                if (next < A.B) fetch(next);
            }
            __syncthreads();
            if (A.dX) bank_join64<true>(smem, A.dX + off, j0 > 0, wave, waves, lane);
            __syncthreads();
        }
    }
}

}  // namespace wn
