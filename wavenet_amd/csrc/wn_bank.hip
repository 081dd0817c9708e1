// Routed filter bank: wn_forward_routed, wn_backprop_routed.
#include <algorithm>

#include "wn_bank_kernels.h"

extern "C" const void* wn_kernel_bank_np2(int kind, int sc);
extern "C" const void* wn_kernel_bank_np4(int kind, int sc);
extern "C" const void* wn_kernel_bank_np8(int kind, int sc);
extern "C" const void* wn_kernel_bank_np16(int kind, int sc);
extern "C" const void* wn_kernel_bank_np32(int kind, int sc);
extern "C" const void* wn_kernel_bank64_np2(int kind);
extern "C" const void* wn_kernel_bank64_np4(int kind);
extern "C" const void* wn_kernel_bank64_np8(int kind);
extern "C" const void* wn_kernel_bank64_np16(int kind);
extern "C" const void* wn_kernel_bank64_np32(int kind);
extern "C" const void* wn_kernel_bank_line_np2(int kind, int M);
extern "C" const void* wn_kernel_bank_line_np4(int kind, int M);
extern "C" const void* wn_kernel_bank_line_np8(int kind, int M);
extern "C" const void* wn_kernel_bank_line_np16(int kind, int M);
extern "C" const void* wn_kernel_bank_line_np32(int kind, int M);

namespace wn {

constexpr size_t BANK_TILE = (64 * 65 + 1) * sizeof(double);   // LDS per wave of the 64x64 kernels: a tile and a weight

struct BankReduceArgs {
    const int* idx;
    const double* grad;
    double* out;
    long long entries;
    int N;
};

// dfilters[f] = sum of the gradients of the entries that name f.  A workgroup per filter looks through all indices, eight a
// thread at a time so that their loads are in flight together (one at a time, 256 threads: 22 us for 8192 entries, 16
// filters); thread t adds entries t, t + T, ... in order, then the threads are added in a fixed tree: the same bits from
// run to run.
// 32 sums a thread do not fit the registers of 1024 (500 8x8 images, two of 16 filters of 32 taps, forward and backward: 56 us
// with 1024, 49 with 512).
constexpr int reduce_threads(int NP) { return NP > 16 ? 512 : 1024; }
template <int NP>
__global__ __launch_bounds__(reduce_threads(NP)) void k_bank_reduce(BankReduceArgs A) {
    constexpr int REDUCE_T = reduce_threads(NP);
    __shared__ double red[REDUCE_T / 64 * NP];
    const int f = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    double s[NP];
#pragma unroll
    for (int t = 0; t < NP; t++) s[t] = 0;
    for (long long base = tid; base < A.entries; base += 8 * REDUCE_T) {
        int at[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long e = base + i * REDUCE_T;
            at[i] = e < A.entries ? (A.idx ? A.idx[e] : 0) : -1;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (at[i] == f) {
                const double* g = A.grad + (base + i * REDUCE_T) * A.N;
#pragma unroll
                for (int t = 0; t < NP; t++) s[t] += t < A.N ? g[t] : 0.0;
            }
        }
    }
    const double mine = wave_scatter_sums<NP>(s, lane);
    if (lane < NP) red[(tid >> 6) * NP + lane] = mine;
    __syncthreads();
    if (tid < A.N) {
        double sum = 0;
#pragma unroll
        for (int w = 0; w < REDUCE_T / 64; w++) sum += red[w * NP + tid];
        A.out[(size_t)f * A.N + tid] = sum;
    }
}

}  // namespace wn

namespace {

using wn::fail;

struct SizeClass { int T, Q; };
const SizeClass kSizeClasses[5] = {{64, 1}, {64, 3}, {64, 4}, {256, 3}, {512, 3}};

int size_class(long long n) { return n <= 128 ? 0 : n <= 512 ? 1 : n <= 1024 ? 2 : n <= 2048 ? 3 : n <= 4096 ? 4 : -1; }

int ilog2_exact(int v) { return (v < 1 || (v & (v - 1))) ? -1 : __builtin_ctz((unsigned)v); }

const void* kernel_for(int NP, int kind, int sc) {
    switch (NP) {
        case 2: return wn_kernel_bank_np2(kind, sc);
        case 4: return wn_kernel_bank_np4(kind, sc);
        case 8: return wn_kernel_bank_np8(kind, sc);
        case 16: return wn_kernel_bank_np16(kind, sc);
        case 32: return wn_kernel_bank_np32(kind, sc);
    }
    return nullptr;
}
const void* kernel64_for(int NP, int kind) {
    switch (NP) {
        case 2: return wn_kernel_bank64_np2(kind);
        case 4: return wn_kernel_bank64_np4(kind);
        case 8: return wn_kernel_bank64_np8(kind);
        case 16: return wn_kernel_bank64_np16(kind);
        case 32: return wn_kernel_bank64_np32(kind);
    }
    return nullptr;
}
const void* line_kernel_for(int NP, int kind, int M) {
    switch (NP) {
        case 2: return wn_kernel_bank_line_np2(kind, M);
        case 4: return wn_kernel_bank_line_np4(kind, M);
        case 8: return wn_kernel_bank_line_np8(kind, M);
        case 16: return wn_kernel_bank_line_np16(kind, M);
        case 32: return wn_kernel_bank_line_np32(kind, M);
    }
    return nullptr;
}
const void* reduce_for(int NP) {
    switch (NP) {
        case 2: return (const void*)&wn::k_bank_reduce<2>;
        case 4: return (const void*)&wn::k_bank_reduce<4>;
        case 8: return (const void*)&wn::k_bank_reduce<8>;
        case 16: return (const void*)&wn::k_bank_reduce<16>;
    }
    return (const void*)&wn::k_bank_reduce<32>;
}

// What both directions check: shape, bank, routing.  Fills A and the compiled tap count.
int check_bank(wn_context* ctx, int B, int R, int C, const double* filters, int F, int N, const int* idx, const double* w, int k,
               wn::BankArgs& A, int& NP, int& sc) {
    if (B < 0) return fail(ctx, WN_ERR_ARG, "negative batch size");
    A.lgR = ilog2_exact(R);
    A.lgC = ilog2_exact(C);
    if (A.lgR < 0 || A.lgC < 0)
        return fail(ctx, WN_ERR_BAD_SHAPE, "shape {" + std::to_string(R) + ", " + std::to_string(C) + "} is not radix 2");
    if (filters) {
        if (F < 1) return fail(ctx, WN_ERR_ARG, "no filters");
        if (N <= 0) return fail(ctx, WN_ERR_BAD_FILTER, "Input filter is empty.");
        if (N % 2) return fail(ctx, WN_ERR_BAD_FILTER, "Input filter length is not a multiple of 2.");
        A.filters = filters;
    } else {
        if (!ctx->has_filter) return fail(ctx, WN_ERR_STATE, "no filter set");
        if (F != 1 || N != ctx->N) return fail(ctx, WN_ERR_ARG, "the context holds one filter of " + std::to_string(ctx->N) + " taps");
        A.filters = ctx->dfilt->a_true;
    }
    if (N > WN_MAX_TAPS) return fail(ctx, WN_ERR_UNSUPPORTED, "filter length " + std::to_string(N) + " exceeds " + std::to_string(WN_MAX_TAPS));
    NP = 2;
    while (NP < N) NP *= 2;
    if (k < 1 || k > WN_MAX_TOPK) return fail(ctx, WN_ERR_ARG, "k is " + std::to_string(k) + ", not 1 ... " + std::to_string(WN_MAX_TOPK));
    if (!idx && k != 1 && B > 0) return fail(ctx, WN_ERR_ARG, "without indices every example has one filter, k is " + std::to_string(k));
    const long long n = 1LL << (A.lgR + A.lgC);
    sc = size_class(n);
    if (sc < 0)
        return fail(ctx, WN_ERR_UNSUPPORTED, "routed transforms: examples of " + std::to_string(n) + " samples exceed the " + std::to_string(WN_MAX_FUSED));
    if (!wn::aligned_to(filters, 8) || !wn::aligned_to(idx, 4) || !wn::aligned_to(w, 8)) return fail(ctx, WN_ERR_ARG, "misaligned pointer");
    A.B = B; A.k = k; A.F = F; A.N = N; A.idx = idx; A.w = w;
    return WN_OK;
}

// sizes of a call's arguments, in elements
struct BankMemory {
    unsigned long long values, entries, bank;   // of X and the like, of idx and w, of the filters
    unsigned long long blocks;                  // of a checkpoint
    BankMemory(const wn::BankArgs& A)
        : values((unsigned long long)A.B << (A.lgR + A.lgC)), entries((unsigned long long)A.B * A.k), bank((unsigned long long)A.F * A.N),
          blocks((unsigned long long)A.B * (((1ull << (A.lgR + A.lgC)) + wn::CKPT_BLOCK - 1) / wn::CKPT_BLOCK)) {}
};

unsigned grid_for(wn_context* ctx, int B) { return (unsigned)std::min<long long>(B, (long long)ctx->numCU * 32); }

// kind 0 forward, 1 backward from the examples, 2 backward from a checkpoint.
int launch_bank(wn_context* ctx, int NP, int sc, int kind, wn::BankArgs& A) {
    const size_t n = (size_t)1 << (A.lgR + A.lgC);
    if (ctx->wave64 && A.lgR == 6 && A.lgC == 6) {
        // a workgroup per example, a wave per filter, up to the four whose tiles fit a CU (2048 examples, 2 and 4 filters:
        // forward 54 and 86 us; one wave for all of them in turn 66 and 114)
        const int waves = std::min(A.k, 4);
        // as many workgroups as are on the chip at a time, each fetching its next example early
        const unsigned grid = (unsigned)std::min(A.B, ctx->numCU * (4 / waves));
        return wn::launch_kernel(ctx, kernel64_for(NP, kind), grid, 64 * waves, waves * wn::BANK_TILE, A);
    }
    if (ctx->wave64 && A.lgC == 0 && A.lgR >= 7 && A.lgR <= 10) {
        const int waves = std::min(A.k, 4);
        return wn::launch_kernel(ctx, line_kernel_for(NP, kind, 1 << (A.lgR - 6)), grid_for(ctx, A.B), 64 * waves, waves * (n + 1) * sizeof(double), A);
    }
    // a team of threads per filter: a wave each, up to four, while a wave is enough for an example
    const int T = kSizeClasses[sc].T, teams = T == 64 ? std::min(A.k, 4) : 1;
    const size_t team = (size_t)wn::bank_team_doubles((int)n, A.lgC > 0, kind ? T / 64 * NP + 2 : 0);
    return wn::launch_kernel(ctx, kernel_for(NP, kind != 0, sc), grid_for(ctx, A.B), T * teams, (n + teams * (1 + team)) * sizeof(double), A);
}

}  // namespace

extern "C" {

int wn_forward_routed(wn_context* ctx, const double* X_dev, int B, int R, int C, const double* filters_dev, int F, int N,
                      const int* idx_dev, const double* w_dev, int k, double* Y_dev, signed char* q_dev, float* scale_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::BankArgs A = {};
        int NP, sc;
        int rc = check_bank(ctx, B, R, C, filters_dev, F, N, idx_dev, w_dev, k, A, NP, sc);
        if (rc || B == 0) return rc;
        if (!X_dev || !Y_dev) return fail(ctx, WN_ERR_ARG, "null pointer");
        if (!q_dev != !scale_dev) return fail(ctx, WN_ERR_ARG, "a checkpoint is values and scales");
        if (!wn::aligned_to(X_dev, 8) || !wn::aligned_to(Y_dev, 8) || !wn::aligned_to(scale_dev, 4)) return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        const BankMemory M(A);
        rc = wn::refuse_overlaps(ctx, {{"Y", Y_dev, M.values * 8}, {"q", q_dev, M.values}, {"scale", scale_dev, M.blocks * 4}},
                                 {{"X", X_dev, M.values * 8}, {"filters", filters_dev, M.bank * 8}, {"idx", idx_dev, M.entries * 4}, {"w", w_dev, M.entries * 8}});
        if (rc) return rc;
        A.X = X_dev; A.Y = Y_dev; A.q_out = q_dev; A.qs_out = scale_dev;
        return launch_bank(ctx, NP, sc, 0, A);
    });
}

int wn_backprop_routed(wn_context* ctx, const double* Delta_dev, const double* X_dev, const signed char* q_dev, const float* scale_dev,
                       int B, int R, int C, const double* filters_dev, int F, int N, const int* idx_dev, const double* w_dev, int k,
                       double* grad_dev, double* dfilters_dev, double* dw_dev, double* dX_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::BankArgs A = {};
        int NP, sc;
        int rc = check_bank(ctx, B, R, C, filters_dev, F, N, idx_dev, w_dev, k, A, NP, sc);
        if (rc) return rc;
        if (!wn::aligned_to(dfilters_dev, 8)) return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        if (B > 0) {
            if (!Delta_dev || !grad_dev) return fail(ctx, WN_ERR_ARG, "null pointer");
            if (!q_dev != !scale_dev) return fail(ctx, WN_ERR_ARG, "a checkpoint is values and scales");
            if (!X_dev == !q_dev) return fail(ctx, WN_ERR_ARG, "either the examples or their checkpoint");
            if (!wn::aligned_to(Delta_dev, 8) || !wn::aligned_to(X_dev, 8) || !wn::aligned_to(scale_dev, 4) || !wn::aligned_to(grad_dev, 8) ||
                !wn::aligned_to(dw_dev, 8) || !wn::aligned_to(dX_dev, 8))
                return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        }
        const BankMemory M(A);
        rc = wn::refuse_overlaps(ctx, {{"grad", grad_dev, M.entries * N * 8}, {"dfilters", dfilters_dev, M.bank * 8}, {"dw", dw_dev, M.entries * 8},
                                       {"dX", dX_dev, M.values * 8}},
                                 {{"Delta", Delta_dev, M.values * 8}, {"X", X_dev, M.values * 8}, {"q", q_dev, M.values}, {"scale", scale_dev, M.blocks * 4},
                                  {"filters", filters_dev, M.bank * 8}, {"idx", idx_dev, M.entries * 4}, {"w", w_dev, M.entries * 8}});
        if (rc) return rc;
        if (B > 0) {
            A.D = Delta_dev; A.X = X_dev; A.q = q_dev; A.qs = scale_dev; A.grad = grad_dev; A.dw = dw_dev; A.dX = dX_dev;
            rc = launch_bank(ctx, NP, sc, q_dev ? 2 : 1, A);
            if (rc) return rc;
        }
        if (!dfilters_dev) return WN_OK;
        wn::BankReduceArgs S = {idx_dev, grad_dev, dfilters_dev, (long long)B * k, N};
        return wn::launch_kernel(ctx, reduce_for(NP), (unsigned)F, wn::reduce_threads(NP), 0, S);
    });
}

}  // extern "C"
