// Transforms of examples under the filters they were routed to, and their backward pass: one workgroup per example,
// everything in LDS (the building blocks of wn_device.h); up to 1024 samples a wave per filter, beyond one filter after another.
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

// ---- passes of one wave over lines in LDS -----------------------------------------------------------------------
// As fwd_pass and bwd_pass (wn_device.h), term by term: a lane has two neighbouring outputs (or errors) of a line, whose
// windows share all but two values, and strides are shifts, so that a value costs a subtraction, a mask and an addition of
// address instead of a multiplication more.  Latency bounds it, at two waves per SIMD that the registers leave to the backward
// pass: 3.0 k vector instructions per example and filter of 16x32 and 8 taps are 20 us of that kernel's 44 for 4000 such pairs.
struct BankLines {
    int lgEs, lgLs;          // log2 of the strides between a line's values and between lines
    int lgNL, lgLen;         // log2 of the number of lines and of their length
    bool lanes_on_lines;     // neighbouring lanes on neighbouring lines
    __device__ unsigned line_offset(int line) const { return (unsigned)line << (lgLs + 3); }
    // item w of 2^lgNL lines times 2^lgM items
    __device__ void split(int w, int lgM, int& line, int& m) const {
        if (lanes_on_lines) { line = w & ((1 << lgNL) - 1); m = w >> lgNL; }
        else                { m = w & ((1 << lgM) - 1);     line = w >> lgM; }
    }
};
__device__ __forceinline__ double& bank_value(double* base, unsigned bytes) { return *reinterpret_cast<double*>(reinterpret_cast<char*>(base) + bytes); }
__device__ __forceinline__ const double& bank_value(const double* base, unsigned bytes) {
    return *reinterpret_cast<const double*>(reinterpret_cast<const char*>(base) + bytes);
}

// lo[k] = sum_j a[j] in[(N/2 + 2k - j) mod 2 half] and with HI hi[k] likewise with b, half = 2^lgHalf
template <int NP, bool HI>
__device__ __forceinline__ void bank_fwd_level(const double* in, double* lo, double* hi, const BankLines& L, int lgHalf, const double (&a)[NP],
                                               const double (&b)[NP], int lane) {
    const int s = L.lgEs + 3;
    const unsigned mask = ((2u << lgHalf) - 1) << s;
    if (lgHalf == 0) {
        for (int line = lane; line < (1 << L.lgNL); line += 64) {
            const unsigned at = L.line_offset(line);
            double sl = 0, sh = 0;
#pragma unroll
            for (int j = 0; j < NP; j++) {
                const double v = bank_value(in, at + (((unsigned)(NP / 2 - j) << s) & mask));
                sl = __builtin_fma(a[j], v, sl);
                if constexpr (HI) sh = __builtin_fma(b[j], v, sh);
            }
            bank_value(lo, at) = sl;
            if constexpr (HI) bank_value(hi, at) = sh;
        }
        return;
    }
    const int lgM = lgHalf - 1;
    for (int w = lane; w < (1 << (L.lgNL + lgM)); w += 64) {
        int line, m;
        L.split(w, lgM, line, m);
        const unsigned at = L.line_offset(line), top = (unsigned)(4 * m + NP / 2 + 2) << s, to = at + ((unsigned)(2 * m) << s);
        double v[NP + 2];    // v[t] = in[4 m + N/2 + 2 - t]: output 2 m + 1 starts at t = 0, output 2 m at t = 2
#pragma unroll
        for (int t = 0; t < NP + 2; t++) v[t] = bank_value(in, at + ((top - ((unsigned)t << s)) & mask));
        double l0 = 0, l1 = 0, h0 = 0, h1 = 0;
#pragma unroll
        for (int j = 0; j < NP; j++) {
            l0 = __builtin_fma(a[j], v[j + 2], l0);
            l1 = __builtin_fma(a[j], v[j], l1);
            if constexpr (HI) {
                h0 = __builtin_fma(b[j], v[j + 2], h0);
                h1 = __builtin_fma(b[j], v[j], h1);
            }
        }
        bank_value(lo, to) = l0;
        bank_value(lo, to + (1u << s)) = l1;
        if constexpr (HI) {
            bank_value(hi, to) = h0;
            bank_value(hi, to + (1u << s)) = h1;
        }
    }
}
// Coefficients of the lines (out) and their low-pass pyramid P, P[2^i + k] = level i; without HI the pyramid down to level 1
// alone, which is what the backward pass reads.  Every lane sees them.
template <int NP, bool HI>
__device__ __forceinline__ void bank_fwd_pass(const double* in, double* P, double* out, const BankLines& L, const double (&a)[NP],
                                              const double (&b)[NP], int lane) {
    for (int i = L.lgLen - 1; i >= (HI ? 0 : 1); i--) {
        const double* src = (i == L.lgLen - 1) ? in : P + ((size_t)2 << (i + L.lgEs));
        bank_fwd_level<NP, HI>(src, P + ((size_t)1 << (i + L.lgEs)), HI ? out + ((size_t)1 << (i + L.lgEs)) : nullptr, L, i, a, b, lane);
        team_sync<64>();
    }
    if constexpr (HI) {
        const double* first = L.lgLen ? P + ((size_t)1 << L.lgEs) : in;
        for (int line = lane; line < (1 << L.lgNL); line += 64) out[(size_t)line << L.lgLs] = first[(size_t)line << L.lgLs];
        team_sync<64>();
    }
}

// One level of the backward cascade: errors D[0 .. len) on the low-pass, D[len .. 2 len) on the high-pass values, in place to
// the errors D[0 .. 2 len) on the level's input; act: that input.  Window sums as in bwd_level (wn_device.h).  K >= n / 64.
template <int NP, int K>
__device__ __forceinline__ void bank_bwd_level(double* D, const double* act, const BankLines& L, int lgLen, const double (&a)[NP],
                                               const double (&b)[NP], double (&gL)[NP], double (&gH)[NP], int lane) {
    constexpr int S = NP / 2;
    constexpr int JE = S & 1, JO = (S + 1) & 1;
    constexpr int CE = (JE - S) / 2, CO = (1 + JO - S) / 2;      // exact; CO is CE or CE + 1
    const int s = L.lgEs + 3;
    const unsigned amask = ((2u << lgLen) - 1) << s, rmask = ((1u << lgLen) - 1) << s, high = 1u << (lgLen + s), one = 1u << s;
    if (lgLen == 0) {                                            // one error of either kind, of this lane's line alone
        for (int line = lane; line < (1 << L.lgNL); line += 64) {
            const unsigned at = L.line_offset(line);
            const double dl = bank_value(D, at), dh = bank_value(D, at + high);
            double se = 0, so = 0;
#pragma unroll
            for (int u = 0; u < NP; u++) {
                const double v = bank_value(act, at + (((unsigned)(NP / 2 - u) << s) & amask));
                gL[u] = __builtin_fma(dl, v, gL[u]);
                gH[u] = __builtin_fma(dh, v, gH[u]);
            }
#pragma unroll
            for (int i = 0; i < NP / 2; i++) {
                se = __builtin_fma(a[JE + 2 * i], dl, se);
                se = __builtin_fma(b[JE + 2 * i], dh, se);
                so = __builtin_fma(a[JO + 2 * i], dl, so);
                so = __builtin_fma(b[JO + 2 * i], dh, so);
            }
            bank_value(D, at) = se;
            bank_value(D, at + one) = so;
        }
        team_sync<64>();
        return;
    }
    constexpr int NIT = (K + 3) / 4;                             // pairs of errors per lane
    const int lgM = lgLen - 1, W = 1 << (L.lgNL + lgM);
    double nw[NIT][4];
#pragma unroll
    for (int it = 0; it < NIT; it++) {
        const int w = lane + it * 64;
        if (w < W) {
            int line, m;
            L.split(w, lgM, line, m);
            const unsigned at = L.line_offset(line), first = (unsigned)(2 * m + CE) << s, top = (unsigned)(4 * m + NP / 2 + 2) << s;
            double dl[S + 2], dh[S + 2];                         // errors 2 m + CE + t
#pragma unroll
            for (int t = 0; t < S + 2; t++) {
                const unsigned o = at + ((first + ((unsigned)t << s)) & rmask);
                dl[t] = bank_value(D, o);
                dh[t] = bank_value(D, o + high);
            }
            double e0 = 0, o0 = 0, e1 = 0, o1 = 0;
#pragma unroll
            for (int i = 0; i < S; i++) {
                e0 = __builtin_fma(a[JE + 2 * i], dl[i], e0);
                e0 = __builtin_fma(b[JE + 2 * i], dh[i], e0);
                o0 = __builtin_fma(a[JO + 2 * i], dl[i + CO - CE], o0);
                o0 = __builtin_fma(b[JO + 2 * i], dh[i + CO - CE], o0);
                e1 = __builtin_fma(a[JE + 2 * i], dl[i + 1], e1);
                e1 = __builtin_fma(b[JE + 2 * i], dh[i + 1], e1);
                o1 = __builtin_fma(a[JO + 2 * i], dl[i + 1 + CO - CE], o1);
                o1 = __builtin_fma(b[JO + 2 * i], dh[i + 1 + CO - CE], o1);
            }
            nw[it][0] = e0; nw[it][1] = o0; nw[it][2] = e1; nw[it][3] = o1;
            double v[NP + 2];                                    // as in bank_fwd_level; errors 2 m and 2 m + 1 are t = -CE and 1 - CE
#pragma unroll
            for (int t = 0; t < NP + 2; t++) v[t] = bank_value(act, at + ((top - ((unsigned)t << s)) & amask));
#pragma unroll
            for (int u = 0; u < NP; u++) {
                gL[u] = __builtin_fma(dl[-CE], v[u + 2], gL[u]);
                gH[u] = __builtin_fma(dh[-CE], v[u + 2], gH[u]);
                gL[u] = __builtin_fma(dl[1 - CE], v[u], gL[u]);
                gH[u] = __builtin_fma(dh[1 - CE], v[u], gH[u]);
            }
        }
    }
    team_sync<64>();
#pragma unroll
    for (int it = 0; it < NIT; it++) {
        const int w = lane + it * 64;
        if (w < W) {
            int line, m;
            L.split(w, lgM, line, m);
            const unsigned to = L.line_offset(line) + ((unsigned)(4 * m) << s);
#pragma unroll
            for (int i = 0; i < 4; i++) bank_value(D, to + ((unsigned)i << s)) = nw[it][i];
        }
    }
    team_sync<64>();
}
template <int NP, int K>
__device__ __forceinline__ void bank_bwd_pass(double* D, const double* in, const double* P, const BankLines& L, const double (&a)[NP],
                                              const double (&b)[NP], double (&gL)[NP], double (&gH)[NP], int lane) {
    for (int i = 0; i < L.lgLen; i++)
        bank_bwd_level<NP, K>(D, i == L.lgLen - 1 ? in : P + ((size_t)2 << (i + L.lgEs)), L, i, a, b, gL, gH, lane);
}

// Whether a team of T threads with 2^Q samples each takes the passes above.  With fewer samples pairs leave lanes idle; a
// workgroup of several waves has too few registers for the wider windows at 16 taps and more (128x32, 32 taps: 680 us
// against 1294); at up to 512 samples they cost the second wave per SIMD with 16 taps and gain nothing with 2 or 4.
// 1000 examples, four filters of 2, 4, 8, 16, 32 taps, forward and backward, without pairs and with them:
//   32x32: 122, 145, 205, 306, 755 us     110, 129, 158, 227, 467
//   16x32:  45,  53,  74, 113, 365         45,  53,  67, 122, 265
//   16x16:  26,  32,  47,  70, 234         28,  36,  47,  91, 198
constexpr bool bank_in_pairs(int NP, int T, int Q) { return T == 64 && (Q == 4 || (Q == 3 && (NP == 8 || NP == 32))); }
// Forward and backward pass along the rows (ROWS) or columns of an example in LDS
template <int NP, int T, int Q, bool ROWS, bool HI>
__device__ __forceinline__ void bank_fwd(const double* in, double* P, double* out, int lgR, int lgC, const double (&a)[NP], const double (&b)[NP], int tid) {
    const int lgLs = ROWS ? 0 : lgR, lgEs = ROWS ? lgR : 0, lgNL = ROWS ? lgR : lgC, lgLen = ROWS ? lgC : lgR;
    if constexpr (bank_in_pairs(NP, T, Q)) bank_fwd_pass<NP, HI>(in, P, out, {lgEs, lgLs, lgNL, lgLen, ROWS}, a, b, tid);
    else if constexpr (HI)             fwd_pass<NP, T>(in, P, out, 1 << lgEs, 1 << lgLs, lgNL, lgLen, ROWS, a, b, tid);
    else                               fwd_pass_lo<NP, T>(in, P, 1 << lgEs, 1 << lgLs, lgNL, lgLen, ROWS, a, tid);
}
template <int NP, int T, int Q, bool ROWS>
__device__ __forceinline__ void bank_bwd(double* D, const double* in, const double* P, int lgR, int lgC, const double (&a)[NP], const double (&b)[NP],
                                         double (&gL)[NP], double (&gH)[NP], int tid) {
    const int lgLs = ROWS ? 0 : lgR, lgEs = ROWS ? lgR : 0, lgNL = ROWS ? lgR : lgC, lgLen = ROWS ? lgC : lgR;
    if constexpr (bank_in_pairs(NP, T, Q)) bank_bwd_pass<NP, (1 << Q)>(D, in, P, {lgEs, lgLs, lgNL, lgLen, ROWS}, a, b, gL, gH, tid);
    else bwd_pass<NP, T, (1 << Q), true>(D, in, P, 1 << lgEs, 1 << lgLs, lgNL, lgLen, ROWS, true, a, b, gL, gH, tid);
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
    const int lgR = A.lgR, lgC = A.lgC, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
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
            if (rows) bank_fwd<NP, T, Q, true, true>(bufX, bufP, bufY1, lgR, lgC, a, b, G.tid);
            bank_fwd<NP, T, Q, false, true>(bufY1, bufP, bufY, lgR, lgC, a, b, G.tid);
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
    extern __shared__ __attribute__((aligned(16))) double smem[];
    const BankTeam<T> G;
    const int lgR = A.lgR, lgC = A.lgC, n = 1 << (lgR + lgC), nb = (n + CKPT_BLOCK - 1) / CKPT_BLOCK;
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
            if (rows) bank_fwd<NP, T, Q, true, true>(bufX, bufP, bufY1, lgR, lgC, a, b, G.tid);
            bank_fwd<NP, T, Q, false, false>(bufY1, bufP, nullptr, lgR, lgC, a, b, G.tid);
            __syncthreads();
            double gL[NP], gH[NP];
#pragma unroll
            for (int u = 0; u < NP; u++) { gL[u] = 0; gH[u] = 0; }
            bank_bwd<NP, T, Q, false>(bufD, bufY1, bufP, lgR, lgC, a, b, gL, gH, G.tid);
            if (rows) {
                bank_fwd<NP, T, Q, true, false>(bufX, bufP, nullptr, lgR, lgC, a, b, G.tid);
                bank_bwd<NP, T, Q, true>(bufD, bufX, bufP, lgR, lgC, a, b, gL, gH, G.tid);
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
