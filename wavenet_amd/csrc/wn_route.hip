// Router of the filter bank: wn_route, wn_route_backward.
//
// A row of F scores belongs to LPR lanes of a wave, VPL scores each (filter i * LPR + lane).  Scores, exponentials and
// what is compared are doubles: the choice of a filter hangs on differences of any size.
#include <algorithm>

#include "wn_bank.h"

namespace wn {

struct RouteArgs {
    const void* scores;
    long long rs, cs;        // elements between rows, between filters
    int T, F, k, groups, kept, per;   // per: filters in a group
    unsigned per_magic;      // f / per = f * per_magic >> 20, f < 1024
    int sigmoid, renorm;
    double scale, score_scale;
    const double* bias;
    int* idx;
    double* w;
    int* counts;
    // backward
    const int* idx_in;
    const double* dw;
    void* dscores;
};

constexpr int ROUTE_T = 256;

template <int LPR>
__device__ __forceinline__ double row_max(double v) {
#pragma unroll
    for (int m = 1; m < LPR; m *= 2) v = __builtin_fmax(v, __shfl_xor(v, m, 64));
    return v;
}
template <int LPR>
__device__ __forceinline__ double row_sum(double v) {
#pragma unroll
    for (int m = 1; m < LPR; m *= 2) v += __shfl_xor(v, m, 64);
    return v;
}
template <int LPR>
__device__ __forceinline__ bool row_any(bool v) {
    int x = v;
#pragma unroll
    for (int m = 1; m < LPR; m *= 2) x |= __shfl_xor(x, m, 64);
    return x != 0;
}
__device__ __forceinline__ void route_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ double minus_inf() { return -__builtin_huge_val(); }

// log of the sigmoid, up to a constant the log of a softmax
__device__ __forceinline__ double log_share(double s, bool sigmoid) {
    return sigmoid ? __builtin_fmin(s, 0.0) - log1p(exp(-__builtin_fabs(s))) : s;
}

// The scores of a row, score_scale applied; absent filters are closed (-inf).
template <class S, int LPR, int VPL>
__device__ __forceinline__ void load_scores(double (&s)[VPL], const RouteArgs& A, long long row, int l) {
    const S* p = (const S*)A.scores + row * A.rs;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int f = i * LPR + l;
        s[i] = f < A.F ? A.score_scale * widen(p[f * A.cs]) : minus_inf();
    }
}

template <class S, int LPR, int VPL>
__global__ __launch_bounds__(ROUTE_T) void k_route(RouteArgs A) {
    extern __shared__ __attribute__((aligned(16))) double route_lds[];
    constexpr int ROWS = ROUTE_T / LPR;
    const int sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const int lane0 = (threadIdx.x & 63) - l;              // first lane of the row within its wave
    double* crow = route_lds + sub * (A.F + A.groups + 1); // group choice only: the row's values, then its groups' scores
    double* grow = crow + A.F;
    if (A.counts && blockIdx.x == 0) {                     // added up by the next kernel
        for (int f = threadIdx.x; f < A.F; f += ROUTE_T) A.counts[f] = 0;
    }
    for (long long base = (long long)blockIdx.x * ROWS; base < A.T; base += (long long)gridDim.x * ROWS) {
        const bool live = base + sub < A.T;
        const long long row = live ? base + sub : A.T - 1;
        double s[VPL], c[VPL];
        load_scores<S, LPR, VPL>(s, A, row, l);
        bool bad = false;
        double m = minus_inf();
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            bad |= !(s[i] <= 1.7976931348623157e308);      // NaN or +inf
            m = __builtin_fmax(m, s[i]);
        }
        m = row_max<LPR>(m);
        bad = row_any<LPR>(bad);
        const bool shares = A.bias || A.kept < A.groups || (!A.renorm && !A.sigmoid);   // p of every filter is wanted
        double Z = 1;
        if (shares && !A.sigmoid) {
            Z = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                c[i] = s[i] > minus_inf() ? exp(s[i] - m) : 0.0;
                Z += c[i];
            }
            Z = row_sum<LPR>(Z);
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int f = i * LPR + l;
            double v = s[i];
            if (A.bias || A.kept < A.groups) {
                v = A.sigmoid ? 1.0 / (1.0 + exp(-s[i])) : c[i] / Z;
                if (A.bias && f < A.F) v += A.bias[f];
                if (!(s[i] > minus_inf()) || !(v > minus_inf())) v = minus_inf();
            }
            c[i] = v;
        }
        if (A.kept < A.groups) {
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                if (i * LPR + l < A.F) crow[i * LPR + l] = c[i];
            }
            route_lds_order();
            for (int g = l; g < A.groups; g += LPR) {
                double first = minus_inf(), second = minus_inf();
                for (int i = 0; i < A.per; i++) {
                    const double v = crow[g * A.per + i];
                    second = __builtin_fmax(second, __builtin_fmin(first, v));
                    first = __builtin_fmax(first, v);
                }
                grow[g] = second > minus_inf() ? first + second : first;
            }
            route_lds_order();
            unsigned long long keep = 0;
            for (int g = l; g < A.groups; g += LPR) {
                const double mine = grow[g];
                int ahead = 0;
                for (int h = 0; h < A.groups; h++) ahead += grow[h] > mine || (grow[h] == mine && h < g);
                if (ahead < A.kept) keep |= 1ull << g;
            }
#pragma unroll
            for (int x = 1; x < LPR; x *= 2) keep |= __shfl_xor(keep, x, 64);
            route_lds_order();                             // before the next row's values
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const unsigned f = i * LPR + l;
                if (!((keep >> ((f * A.per_magic) >> 20)) & 1)) c[i] = minus_inf();
                else if (!A.bias) c[i] = s[i];             // the order of the scores is the order of the shares
            }
        }
        // k rounds: the largest value left, the lowest filter among equal ones
        int mine_f = -1;
        double mine_s = minus_inf();
        for (int j = 0; j < A.k; j++) {
            double best = minus_inf(), bs = minus_inf();
            int bf = 1 << 30;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                if (c[i] > best) { best = c[i]; bf = i * LPR + l; bs = s[i]; }
            }
#pragma unroll
            for (int x = 1; x < LPR; x *= 2) {
                const double ov = __shfl_xor(best, x, 64), os = __shfl_xor(bs, x, 64);
                const int of = __shfl_xor(bf, x, 64);
                if (ov > best || (ov == best && of < bf)) { best = ov; bf = of; bs = os; }
            }
            if (best == minus_inf()) bf = -1;
            if (l == j) { mine_f = bf; mine_s = bs; }
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                if (i * LPR + l == bf) c[i] = minus_inf();
            }
        }
        // weights, one chosen filter per lane
        const bool have = l < A.k && mine_f >= 0;
        double w = 0;
        if (A.renorm) {
            const double lp = have ? log_share(mine_s, A.sigmoid) : minus_inf();
            const double top = row_max<LPR>(lp);
            const double u = have ? exp(lp - top) : 0.0;
            const double sum = row_sum<LPR>(u);
            if (have) w = A.scale * (u / sum);
        } else if (have) {
            w = A.scale * (A.sigmoid ? 1.0 / (1.0 + exp(-mine_s)) : exp(mine_s - m) / Z);
        }
        if (bad) { mine_f = -1; w = __builtin_nan(""); }
        if (live && l < A.k) {
            A.idx[row * A.k + l] = mine_f;
            A.w[row * A.k + l] = w;
        }
        (void)lane0;
    }
}

// counts[f] += entries of idx that name f: a histogram per workgroup in LDS, then one addition per filter (whole
// numbers, so that their order does not matter).
__global__ __launch_bounds__(1024) void k_route_counts(RouteArgs A) {
    __shared__ int hist[WN_MAX_EXPERTS];
    for (int f = threadIdx.x; f < A.F; f += 1024) hist[f] = 0;
    __syncthreads();
    const long long total = (long long)A.T * A.k;
    for (long long i = (long long)blockIdx.x * 1024 + threadIdx.x; i < total; i += (long long)gridDim.x * 1024) {
        const int f = A.idx_in[i];
        if (f >= 0) atomicAdd(&hist[f], 1);
    }
    __syncthreads();
    for (int f = threadIdx.x; f < A.F; f += 1024) {
        if (hist[f]) atomicAdd(&A.counts[f], hist[f]);
    }
}

template <class S, int LPR, int VPL>
__global__ __launch_bounds__(ROUTE_T) void k_route_backward(RouteArgs A) {
    constexpr int ROWS = ROUTE_T / LPR;
    const int sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    const int lane0 = (threadIdx.x & 63) - l;
    for (long long base = (long long)blockIdx.x * ROWS; base < A.T; base += (long long)gridDim.x * ROWS) {
        const bool live = base + sub < A.T;
        const long long row = live ? base + sub : A.T - 1;
        const S* p = (const S*)A.scores + row * A.rs;
        const int f_mine = l < A.k ? A.idx_in[row * A.k + l] : -1;
        const bool have = f_mine >= 0 && f_mine < A.F;
        const double g = have ? A.scale * A.dw[row * A.k + l] : 0.0;
        const double s_mine = have ? A.score_scale * widen(p[f_mine * A.cs]) : minus_inf();
        double ds[VPL], d = 0, all = 0;        // d: what the chosen filter of this lane gets on its own
#pragma unroll
        for (int i = 0; i < VPL; i++) ds[i] = 0;
        if (A.renorm) {
            const double lp = have ? log_share(s_mine, A.sigmoid) : minus_inf();
            const double top = row_max<LPR>(lp);
            const double u = (have && lp > minus_inf()) ? exp(lp - top) : 0.0;
            const double sum = row_sum<LPR>(u);
            const double share = u > 0 ? u / sum : 0.0;
            const double mean = row_sum<LPR>(have ? share * g : 0.0);
            d = have ? share * (g - mean) : 0.0;
            if (have && A.sigmoid) d *= 1.0 / (1.0 + exp(s_mine));
        } else if (A.sigmoid) {
            const double e = exp(-__builtin_fabs(s_mine)), t = 1.0 / (1.0 + e);
            d = have ? g * (e * t * t) : 0.0;              // p (1 - p)
        } else if (row_any<LPR>(have)) {
            double s[VPL], m = minus_inf(), Z = 0;
            load_scores<S, LPR, VPL>(s, A, row, l);
#pragma unroll
            for (int i = 0; i < VPL; i++) m = __builtin_fmax(m, s[i]);
            m = row_max<LPR>(m);
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                s[i] = s[i] == minus_inf() ? 0.0 : exp(s[i] - m);
                Z += s[i];
            }
            Z = row_sum<LPR>(Z);
            const double pm = (have && s_mine != minus_inf()) ? exp(s_mine - m) / Z : 0.0;
            all = row_sum<LPR>(have ? g * pm : 0.0);
#pragma unroll
            for (int i = 0; i < VPL; i++) ds[i] = s[i] == 0.0 ? 0.0 : -(s[i] / Z) * all;
            d = have ? g * pm : 0.0;
        }
        for (int j = 0; j < A.k; j++) {
            const int f = __shfl(f_mine, lane0 + j, 64);
            const double v = __shfl(d, lane0 + j, 64);
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                if (i * LPR + l == f) ds[i] += v;
            }
        }
        if (live) {
            S* out = (S*)A.dscores + row * A.rs;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                const int f = i * LPR + l;
                if (f < A.F) out[f * A.cs] = narrow<S>(A.score_scale * ds[i]);
            }
        }
    }
}

}  // namespace wn

namespace {

using wn::fail;

struct RouteClass { const void* forward; const void* backward; int lpr; };

template <class S>
RouteClass route_class(int F) {
#define WN_ROUTE(L, V) return {(const void*)&wn::k_route<S, L, V>, (const void*)&wn::k_route_backward<S, L, V>, L}
    if (F <= 16) WN_ROUTE(16, 1);
    if (F <= 32) WN_ROUTE(16, 2);
    if (F <= 64) WN_ROUTE(16, 4);
    if (F <= 128) WN_ROUTE(16, 8);
    if (F <= 256) WN_ROUTE(16, 16);
    if (F <= 512) WN_ROUTE(64, 8);
    WN_ROUTE(64, 16);
#undef WN_ROUTE
}
RouteClass route_class(int dtype, int F) {
    switch (dtype) {
        case WN_F64: return route_class<double>(F);
        case WN_F32: return route_class<float>(F);
        case WN_F16: return route_class<wn::f16_bits>(F);
    }
    return route_class<wn::bf16_bits>(F);
}

// Checks what both directions take and fills the common part of the arguments.
int check_routing(wn_context* ctx, const void* scores, int dtype, int T, int F, long long rs, long long cs, const wn_routing* r,
                  wn::RouteArgs& A) {
    const size_t es = wn::element_bytes(dtype);
    if (!es) return fail(ctx, WN_ERR_ARG, "unknown element type " + std::to_string(dtype));
    if (!r) return fail(ctx, WN_ERR_ARG, "null pointer");
    if (T < 0 || F < 1) return fail(ctx, WN_ERR_ARG, "bad counts");
    if (F > WN_MAX_EXPERTS) return fail(ctx, WN_ERR_UNSUPPORTED, std::to_string(F) + " filters exceed " + std::to_string(WN_MAX_EXPERTS));
    if (r->score != WN_SCORE_SOFTMAX && r->score != WN_SCORE_SIGMOID) return fail(ctx, WN_ERR_ARG, "unknown score function " + std::to_string(r->score));
    if (r->k < 1 || r->k > F) return fail(ctx, WN_ERR_ARG, "k is " + std::to_string(r->k) + " of " + std::to_string(F) + " filters");
    if (r->k > WN_MAX_TOPK) return fail(ctx, WN_ERR_UNSUPPORTED, "k is " + std::to_string(r->k) + ", beyond " + std::to_string(WN_MAX_TOPK));
    if (r->groups < 1 || F % r->groups) return fail(ctx, WN_ERR_ARG, std::to_string(F) + " filters do not make " + std::to_string(r->groups) + " equal groups");
    if (r->groups > WN_MAX_GROUPS && r->groups_kept < r->groups) return fail(ctx, WN_ERR_UNSUPPORTED, std::to_string(r->groups) + " groups exceed " + std::to_string(WN_MAX_GROUPS));
    if (r->groups_kept < 1 || r->groups_kept > r->groups) return fail(ctx, WN_ERR_ARG, "groups kept: " + std::to_string(r->groups_kept) + " of " + std::to_string(r->groups));
    if (!(__builtin_fabs(r->scale) <= 1e300)) return fail(ctx, WN_ERR_ARG, "scale is not a finite number");
    if (!(__builtin_fabs(r->score_scale) <= 1e300) || r->score_scale == 0) return fail(ctx, WN_ERR_ARG, "score_scale is not a finite number other than zero");
    if (T == 0) return WN_OK;
    const long long far = 1LL << 40;
    if (rs < 0 || cs < 0 || rs > far || cs > far) return fail(ctx, WN_ERR_ARG, "bad strides");
    // no two scores in one place: filters inside rows, or rows inside filters
    const bool rows_outside = (F == 1 || cs >= 1) && (T == 1 || rs > (F - 1) * cs);
    const bool rows_inside = (T == 1 || rs >= 1) && (F == 1 || (__int128)cs > (__int128)(T - 1) * rs);
    if (!rows_outside && !rows_inside) return fail(ctx, WN_ERR_ARG, "strides make scores overlap");
    if (!scores) return fail(ctx, WN_ERR_ARG, "null pointer");
    if (!wn::aligned_to(scores, es)) return fail(ctx, WN_ERR_ARG, "misaligned pointer");
    A.scores = scores; A.rs = rs; A.cs = cs;
    A.T = T; A.F = F; A.k = r->k;
    A.groups = r->groups; A.kept = r->groups_kept; A.per = F / r->groups;
    A.per_magic = ((1u << 20) + A.per - 1) / A.per;
    A.sigmoid = r->score == WN_SCORE_SIGMOID; A.renorm = r->renormalise != 0;
    A.scale = r->scale; A.score_scale = r->score_scale;
    return WN_OK;
}

}  // namespace

extern "C" {

int wn_route(wn_context* ctx, const void* scores_dev, int dtype, int T, int F, long long row_stride, long long col_stride,
             const wn_routing* routing, const double* bias_dev, int* idx_dev, double* w_dev, int* counts_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::RouteArgs A = {};
        int rc = check_routing(ctx, scores_dev, dtype, T, F, row_stride, col_stride, routing, A);
        if (rc) return rc;
        A.T = T; A.F = F;
        A.bias = bias_dev; A.idx = idx_dev; A.w = w_dev; A.counts = counts_dev; A.idx_in = idx_dev;
        if (T > 0) {
            if (!idx_dev || !w_dev) return fail(ctx, WN_ERR_ARG, "null pointer");
            if (!wn::aligned_to(bias_dev, 8) || !wn::aligned_to(idx_dev, 4) || !wn::aligned_to(w_dev, 8) || !wn::aligned_to(counts_dev, 4))
                return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        } else if (!counts_dev) {
            return WN_OK;
        }
        const RouteClass K = route_class(dtype, F);
        const int rows = wn::ROUTE_T / K.lpr;
        const long long grid = std::max(1LL, std::min<long long>(((long long)T + rows - 1) / rows, (long long)ctx->numCU * 16));
        const size_t shmem = A.kept < A.groups ? (size_t)rows * (F + A.groups + 1) * sizeof(double) : 0;
        rc = wn::launch_kernel(ctx, K.forward, (unsigned)grid, wn::ROUTE_T, shmem, A);
        if (rc || !counts_dev || T == 0) return rc;
        const long long entries = (long long)T * A.k;
        const long long cgrid = std::max(1LL, std::min<long long>((entries + 16383) / 16384, 64));
        return wn::launch_kernel(ctx, (const void*)&wn::k_route_counts, (unsigned)cgrid, 1024, 0, A);
    });
}

int wn_route_backward(wn_context* ctx, const void* scores_dev, int dtype, int T, int F, long long row_stride, long long col_stride,
                      const wn_routing* routing, const int* idx_dev, const double* dw_dev, void* dscores_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::RouteArgs A = {};
        int rc = check_routing(ctx, scores_dev, dtype, T, F, row_stride, col_stride, routing, A);
        if (rc || T == 0) return rc;
        if (!idx_dev || !dw_dev || !dscores_dev) return fail(ctx, WN_ERR_ARG, "null pointer");
        if (!wn::aligned_to(idx_dev, 4) || !wn::aligned_to(dw_dev, 8) || !wn::aligned_to(dscores_dev, wn::element_bytes(dtype)))
            return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        A.idx_in = idx_dev; A.dw = dw_dev; A.dscores = dscores_dev;
        const RouteClass K = route_class(dtype, F);
        const int rows = wn::ROUTE_T / K.lpr;
        const long long grid = std::min<long long>(((long long)T + rows - 1) / rows, (long long)ctx->numCU * 16);
        return wn::launch_kernel(ctx, K.backward, (unsigned)grid, wn::ROUTE_T, 0, A);
    });
}

}  // extern "C"
