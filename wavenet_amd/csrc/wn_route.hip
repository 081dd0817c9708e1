// Router of the filter bank: wn_route, wn_route_backward.
//
// A row of F scores belongs to LPR lanes of a wave, VPL consecutive ones each, in registers from the first read to the last
// write.  Scores, exponentials and what is compared are doubles: the choice of a filter hangs on differences of any size.
//
// The k largest are found by merging sorted lists.  The filter's number replaces the low bits of the value, so that one
// double carries both, v_max_f64 / v_min_f64 compare them, equal values come out in order of the filter, and there are no
// rounds: every lane sorts its own values, then log2(LPR) exchanges each merge two lists of K >= k.  (One row of 256 scores,
// k = 8: about 300 of these instructions; k rounds of a largest value with its number took some 1400.)  Where the bits
// given up could have mattered, which is checked on the result, the row is chosen again by rounds on the full values.
#include <algorithm>
#include <cstdlib>

#include "wn_bank.h"

namespace wn {

struct RouteArgs {
    const void* scores;
    int dtype;
    long long rs, cs;        // elements between rows, between filters
    int T, F, k, groups, kept, per;   // per: filters in a group
    unsigned per_magic;      // f / per = f * per_magic >> 20, f < 1024
    int sigmoid, renorm;
    int settle_rows;         // rows of a workgroup of the second kernel at a time, at most SETTLE_T
    int count_here;          // the first kernel counts, there is no second one
    int doubts;              // values may lie closer than what the first kernel compares
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
constexpr unsigned long long ROUTE_LOW = WN_MAX_EXPERTS - 1;   // bits that hold a filter's number

__device__ __forceinline__ double minus_inf() { return -__builtin_huge_val(); }
__device__ __forceinline__ unsigned long long bits_of(double v) { return __builtin_bit_cast(unsigned long long, v); }
__device__ __forceinline__ double of_bits(unsigned long long u) { return __builtin_bit_cast(double, u); }

// v_max_f64 / v_min_f64 as they are: the compiler's fmax first makes every operand that came through a cross-lane move a
// quiet NaN, one instruction more each.
__device__ __forceinline__ double key_max(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double key_min(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// e^x for x <= 0 within about one unit in the last place: x = n ln 2 + r with |r| <= ln 2 / 2 (ln 2 in two parts), the Taylor
// series of e^r to r^13 (what is left out is below 2^-57), times 2^n.  Without the cases that do not come up here: x is
// clamped to where the result is 0 anyway, and rows with a NaN are void.
__device__ __forceinline__ double route_exp(double x) {
    x = key_max(x, -800.0);
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0x1.62e42fefp-1, x);   // ln 2 to 33 bits: n times that is exact
    r = __builtin_fma(n, -0x1.473de6af278edp-34, r);
    double t = 1.0 / 6227020800.0;
    t = __builtin_fma(t, r, 1.0 / 479001600.0);
    t = __builtin_fma(t, r, 1.0 / 39916800.0);
    t = __builtin_fma(t, r, 1.0 / 3628800.0);
    t = __builtin_fma(t, r, 1.0 / 362880.0);
    t = __builtin_fma(t, r, 1.0 / 40320.0);
    t = __builtin_fma(t, r, 1.0 / 5040.0);
    t = __builtin_fma(t, r, 1.0 / 720.0);
    t = __builtin_fma(t, r, 1.0 / 120.0);
    t = __builtin_fma(t, r, 1.0 / 24.0);
    t = __builtin_fma(t, r, 1.0 / 6.0);
    t = __builtin_fma(t, r, 0.5);
    t = __builtin_fma(t, r, 1.0);
    t = __builtin_fma(t, r, 1.0);
    return __builtin_ldexp(t, (int)n);
}
// 1 / d for 1 <= d <= 2: the hardware's estimate and two Newton steps
__device__ __forceinline__ double route_reciprocal(double d) {
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}
__device__ __forceinline__ double route_sigmoid(double s) {
    const double e = route_exp(-__builtin_fabs(s)), t = route_reciprocal(1.0 + e);
    return s < 0 ? e * t : t;
}
// reductions over the LPR lanes of a row, the same result in each
template <int LPR, class Op>
__device__ __forceinline__ double row_reduce(double v, int lane, Op op) {
    v = op(v, xlane<1>(v, lane));
    v = op(v, xlane<2>(v, lane));
    v = op(v, xlane<4>(v, lane));
    v = op(v, xlane<8>(v, lane));
    if constexpr (LPR > 16) v = op(v, xlane<16>(v, lane));
    if constexpr (LPR > 32) v = op(v, xlane<32>(v, lane));
    return v;
}
template <int LPR>
__device__ __forceinline__ double row_max(double v, int lane) {
    return row_reduce<LPR>(v, lane, [](double a, double b) { return key_max(a, b); });
}
template <int LPR>
__device__ __forceinline__ double row_sum(double v, int lane) {
    return row_reduce<LPR>(v, lane, [](double a, double b) { return a + b; });
}
// the lanes of a row in a mask of the wave's
template <int LPR>
__device__ __forceinline__ unsigned long long row_lanes(int lane) {
    if constexpr (LPR == 64) return ~0ull;
    else return ((1ull << LPR) - 1) << (lane & ~(LPR - 1));
}
template <int LPR>
__device__ __forceinline__ bool row_any(bool v, int lane) { return (__ballot(v) & row_lanes<LPR>(lane)) != 0; }
__device__ __forceinline__ void route_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The shares to within ROUTE_SLACK of the true ones, from 32-bit exponentials: an argument of x is off by |x| 2^-23, v_exp_f32,
// v_rcp_f32, the sum and the product by 2^-22 or so each, all of it times p <= 1 with |x| p <= 0.4: 0.4 * 1.2e-7 + 3 * 2.4e-7.
constexpr double ROUTE_SLACK = 1e-6;
__device__ __forceinline__ float rough_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float rough_sigmoid(float s) { return __builtin_amdgcn_rcpf(1.0f + rough_exp(-s)); }

// log of the sigmoid, up to a constant the log of a softmax
__device__ __forceinline__ double log_share(double s, bool sigmoid) {
    return sigmoid ? __builtin_fmin(s, 0.0) - log1p(exp(-__builtin_fabs(s))) : s;
}

template <class S>
__device__ __forceinline__ double load_score(const RouteArgs& A, long long at) {
    return widen(((const S*)A.scores)[at]);
}
__device__ __forceinline__ double score_at(const RouteArgs& A, long long row, int f) {
    const long long at = row * A.rs + f * A.cs;
    switch (A.dtype) {
        case WN_F64: return load_score<double>(A, at);
        case WN_F32: return load_score<float>(A, at);
        case WN_F16: return load_score<f16_bits>(A, at);
    }
    return load_score<bf16_bits>(A, at);
}
// x[i] = score f0 + i of a row as it is in memory; past the last filter the value that score_scale makes -inf
template <class S, int LPR, int VPL>
__device__ __forceinline__ void load_chunk(double (&x)[VPL], const RouteArgs& A, long long row, int f0, double closed) {
    const S* p = (const S*)A.scores + row * A.rs + f0 * A.cs;
    if (A.cs == 1 && A.F == LPR * VPL) {
        S v[VPL];
        __builtin_memcpy(v, p, sizeof(v));                   // wide loads: the hardware takes any alignment
#pragma unroll
        for (int i = 0; i < VPL; i++) x[i] = widen(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int most = A.F - 1 - f0;                   // every load is made, from a score of the row: no branches
            const double v = widen(p[(i < most ? i : most) * A.cs]);
            x[i] = i <= most ? v : closed;
        }
    }
}
template <int LPR, int VPL>
__device__ __forceinline__ void load_row(double (&x)[VPL], const RouteArgs& A, long long row, int f0) {
    const double closed = A.score_scale > 0 ? minus_inf() : -minus_inf();
    switch (A.dtype) {
        case WN_F64: load_chunk<double, LPR, VPL>(x, A, row, f0, closed); break;
        case WN_F32: load_chunk<float, LPR, VPL>(x, A, row, f0, closed); break;
        case WN_F16: load_chunk<f16_bits, LPR, VPL>(x, A, row, f0, closed); break;
        default: load_chunk<bf16_bits, LPR, VPL>(x, A, row, f0, closed);
    }
}

// ---- sorted lists ---------------------------------------------------------------------------------------------
// Keys are doubles or unsigned 32-bit words.
__device__ __forceinline__ unsigned key_max(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned key_min(unsigned a, unsigned b) { return a < b ? a : b; }
__device__ __forceinline__ double key_none(double) { return minus_inf(); }
__device__ __forceinline__ unsigned key_none(unsigned) { return 0; }
// of lane (lane ^ M)
template <int M>
__device__ __forceinline__ double key_lane(double v, int lane) { return xlane<M>(v, lane); }
template <int M>
__device__ __forceinline__ unsigned key_lane(unsigned v, int lane) {
    if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);          // quad_perm [1,0,3,2]
    else if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);     // quad_perm [2,3,0,1]
    else if constexpr (M == 7) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);    // row_half_mirror
    else if constexpr (M == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, true);    // row_ror:8
    else return __shfl_xor(v, M, 64);
}

// a whole number per lane added up over the row
template <int LPR>
__device__ __forceinline__ int row_count(int v, int lane) {
    v += key_lane<1>((unsigned)v, lane);
    v += key_lane<2>((unsigned)v, lane);
    v += key_lane<7>((unsigned)v, lane);                     // the other four of eight
    v += key_lane<8>((unsigned)v, lane);
    if constexpr (LPR > 16) v += key_lane<16>((unsigned)v, lane);
    if constexpr (LPR > 32) v += key_lane<32>((unsigned)v, lane);
    return v;
}

template <class T>
__device__ __forceinline__ void larger_first(T& a, T& b) {
    const T hi = key_max(a, b);
    b = key_min(a, b);
    a = hi;
}
// v[0 .. N) is bitonic: into descending order
template <int N, class T>
__device__ __forceinline__ void bitonic_clean(T* v) {
    if constexpr (N > 1) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) larger_first(v[i], v[i + N / 2]);
        bitonic_clean<N / 2>(v);
        bitonic_clean<N / 2>(v + N / 2);
    }
}
template <int N, class T>
__device__ __forceinline__ void sort_descending(T* v) {
    if constexpr (N > 1) {
        sort_descending<N / 2>(v);
        sort_descending<N / 2>(v + N / 2);
#pragma unroll
        for (int i = 0; i < N / 2; i++) larger_first(v[i], v[N - 1 - i]);     // the second half is read backwards
        bitonic_clean<N / 2>(v);
        bitonic_clean<N / 2>(v + N / 2);
    }
}
// a = the K largest of a and b, both descending
template <int K, class T>
__device__ __forceinline__ void merge_lists(T (&a)[K], const T* b) {
#pragma unroll
    for (int i = 0; i < K; i++) a[i] = key_max(a[i], b[K - 1 - i]);
    bitonic_clean<K>(a);
}
// The same with the lists of two halves of 2 M lanes.  The exchange may be any that swaps the halves (every lane of a half
// has the half's list), which takes one move for half a row where its mirror image does.
template <int K, int M, class T>
__device__ __forceinline__ void merge_lanes(T (&a)[K], int lane) {
    constexpr int X = (M == 4) ? 7 : M;
    T b[K];
#pragma unroll
    for (int i = 0; i < K; i++) b[i] = key_lane<X>(a[i], lane);
    merge_lists<K>(a, b);
}
// The K largest of the LPR lanes' lists, descending, in every lane
template <int LPR, int K, class T>
__device__ __forceinline__ void largest_of_lanes(T (&top)[K], int lane) {
    merge_lanes<K, 1>(top, lane);
    merge_lanes<K, 2>(top, lane);
    merge_lanes<K, 4>(top, lane);
    merge_lanes<K, 8>(top, lane);
    if constexpr (LPR > 16) merge_lanes<K, 16>(top, lane);
    if constexpr (LPR > 32) merge_lanes<K, 32>(top, lane);
}
// The K largest of a lane's own values, descending.  v is destroyed.
template <int VPL, int K, class T>
__device__ __forceinline__ void largest_own(T (&v)[VPL], T (&top)[K]) {
    if constexpr (VPL <= K) {
        sort_descending<VPL>(v);
#pragma unroll
        for (int i = 0; i < K; i++) top[i] = i < VPL ? v[i < VPL ? i : 0] : key_none(v[0]);
    } else {
#pragma unroll
        for (int c = 0; c < VPL; c += K) sort_descending<K>(v + c);
#pragma unroll
        for (int i = 0; i < K; i++) top[i] = v[i];
#pragma unroll
        for (int c = K; c < VPL; c += K) merge_lists<K>(top, v + c);
    }
}
// A value with its filter's number in the low bits: of equal values the lower filter is the larger key.  -inf stays.
__device__ __forceinline__ double keyed(double c, int f) {
    const unsigned long long u = bits_of(__builtin_fmin(c, 1.7976931348623157e308) + 0.0);     // -0 is 0
    const unsigned flip = (unsigned)((int)(u >> 32) >> 31) & (unsigned)ROUTE_LOW;
    const double k = of_bits((u & ~ROUTE_LOW) | ((ROUTE_LOW ^ (unsigned)f) ^ flip));
    return c == minus_inf() ? c : k;
}
__device__ __forceinline__ int filter_of(double key) {
    const unsigned long long u = bits_of(key);
    const unsigned flip = (unsigned)((int)(u >> 32) >> 31) & (unsigned)ROUTE_LOW;
    return (int)(((unsigned)u & (unsigned)ROUTE_LOW) ^ (unsigned)ROUTE_LOW ^ flip);
}
__device__ __forceinline__ unsigned long long upper(double key) { return bits_of(key) & ~ROUTE_LOW; }

// ---- forward --------------------------------------------------------------------------------------------------

__device__ __forceinline__ double larger_of(double a, double b) { return key_max(a, b); }
__device__ __forceinline__ double smaller_of(double a, double b) { return key_min(a, b); }
__device__ __forceinline__ float larger_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ float smaller_of(float a, float b) { return __builtin_fminf(a, b); }

// of a >= b and v, the one in the middle
__device__ __forceinline__ double middle_of(double a, double b, double v) { return larger_of(b, smaller_of(a, v)); }
__device__ __forceinline__ float middle_of(float a, float b, float v) { return __builtin_amdgcn_fmed3f(a, b, v); }

// The groups that are kept, as a bit mask, from the row's values in LDS: a lane per group.
template <int LPR, class T>
__device__ __forceinline__ unsigned long long kept_groups(T slack, const RouteArgs& A, double* crow, int l, bool& doubt) {
    unsigned long long keep = 0;
    double* grow = crow + A.F;
    for (int g = l; g < A.groups; g += LPR) {
        double first = minus_inf(), second = minus_inf();
        for (int i0 = 0; i0 < A.per; i0 += 4) {              // four on their way at a time
            double v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = crow[g * A.per + min(i0 + i, A.per - 1)];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] = i0 + i < A.per ? v[i] : minus_inf();
                second = middle_of(first, second, v[i]);
                first = larger_of(first, v[i]);
            }
        }
        grow[g] = second > minus_inf() ? first + second : first;
    }
    route_lds_order();
    for (int g = l; g < A.groups; g += LPR) {
        const double mine = grow[g];
        int ahead = 0, surely = 0, perhaps = 0;
        for (int h0 = 0; h0 < A.groups; h0 += 4) {
            double other[4];
#pragma unroll
            for (int i = 0; i < 4; i++) other[i] = grow[min(h0 + i, A.groups - 1)];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int h = h0 + i;
                const bool there = h < A.groups;
                ahead += there && (other[i] > mine || (other[i] == mine && h < g));
                surely += there && other[i] > mine + 2 * slack;
                perhaps += there && other[i] >= mine - 2 * slack && h != g;
            }
        }
        doubt |= slack > 0 && mine > minus_inf() && surely < A.kept && perhaps >= A.kept;
        if (ahead < A.kept) keep |= 1ull << g;
    }
#pragma unroll
    for (int x = 1; x < LPR; x *= 2) keep |= __shfl_xor(keep, x, 64);
    route_lds_order();                                       // before the row's next values
    return keep;
}

// The lane's filters that are in a group that is kept, as a bit mask; c: the row's values, each within slack / 2 of the true one.  A group that is a
// whole number of lanes (a power of two) is reduced in registers; other sizes go through LDS, a lane per group.
// doubt: the values are too close to tell.
template <int LPR, int VPL, class T>
__device__ __forceinline__ unsigned choose_groups(const T (&c)[VPL], T slack, const RouteArgs& A, double* crow, int l,
                                                            int f0, int lane, bool& doubt) {
    const int lanes = A.per / VPL;                           // lanes per group, if that is what a group is
    if (lanes * VPL == A.per && (lanes & (lanes - 1)) == 0 && lanes > 0) {
        T first = (T)minus_inf(), second = (T)minus_inf();
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            second = middle_of(first, second, c[i]);          // first >= second
            first = larger_of(first, c[i]);
        }
        for (int m = 1; m < lanes; m *= 2) {
            const T f2 = __shfl_xor(first, m, 64), s2 = __shfl_xor(second, m, 64);
            second = larger_of(smaller_of(first, f2), larger_of(second, s2));
            first = larger_of(first, f2);
        }
        const T mine = second > (T)minus_inf() ? first + second : first;
        const int g = l / lanes;
        int ahead = 0, surely = 0, perhaps = 0;
        for (int h0 = 0; h0 < A.groups; h0 += 4) {           // four at a time on their way
            T other[4];
#pragma unroll
            for (int i = 0; i < 4; i++) other[i] = __shfl(mine, (lane - l) + ((h0 + i) * lanes & (LPR - 1)), 64);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int h = h0 + i;
                const bool there = h < A.groups;
                ahead += there && (other[i] > mine || (other[i] == mine && h < g));
                surely += there && other[i] > mine + 2 * slack;
                perhaps += there && other[i] >= mine - 2 * slack && h != g;
            }
        }
        doubt |= slack > 0 && g < A.groups && mine > (T)minus_inf() && surely < A.kept && perhaps >= A.kept;
        return ahead < A.kept ? ~0u : 0u;
    }
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        if (f0 + i < A.F) crow[f0 + i] = c[i];
    }
    route_lds_order();
    const unsigned long long keep = kept_groups<LPR, T>(slack, A, crow, l, doubt);
    unsigned own = 0;
#pragma unroll
    for (int i = 0; i < VPL; i++) {                          // (lanes past the last filter may name a group past the last: closed either way)
        own |= ((unsigned)(keep >> ((((unsigned)(f0 + i) * A.per_magic) >> 20) & 63u)) & 1u) << i;
    }
    return own;
}

// s = score_scale * x, in place; the largest of the row (softmax) and whether one of them is NaN or +inf
template <int LPR, int VPL>
__device__ __forceinline__ void scale_row(double (&x)[VPL], const RouteArgs& A, double& m, bool& bad, int lane) {
    m = minus_inf();
    bad = false;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        x[i] *= A.score_scale;
        bad |= !(x[i] <= 1.7976931348623157e308);
        m = __builtin_fmax(m, x[i]);
    }
    bad = row_any<LPR>(bad, lane);
    if (!A.sigmoid) m = row_max<LPR>(m, lane);
}
// The weights of a row, one chosen filter (or -1) per lane, and what leaves.
template <int LPR, int VPL>
__device__ __forceinline__ void finish_row(const RouteArgs& A, long long row, int f, bool bad, bool write, int l, int f0, int lane) {
    const bool have = f >= 0;
    const double s = have ? A.score_scale * score_at(A, row, f) : minus_inf();
    double w = 0;
    if (A.renorm) {
        // of one lane's weight each; lanes without one have u = 0
        double u, sum;
        if (A.sigmoid) {
            u = have ? route_sigmoid(s) : 0.0;
            sum = row_sum<LPR>(u, lane);
            if (__any(have && !(sum > 1e-250))) {            // shares that add up to nothing: from their logarithms
                const double lp = have ? log_share(s, true) : minus_inf(), top = row_max<LPR>(lp, lane);
                u = have ? route_exp(lp - top) : 0.0;
                sum = row_sum<LPR>(u, lane);
            }
        } else {
            const double top = row_max<LPR>(s, lane);
            u = have ? route_exp(s - top) : 0.0;
            sum = row_sum<LPR>(u, lane);
        }
        if (have) w = A.scale * (u / sum);
    } else if (A.sigmoid) {
        if (have) w = A.scale * route_sigmoid(s);
    } else {
        double all[VPL], m;
        bool unused;
        load_row<LPR, VPL>(all, A, row, f0);
        scale_row<LPR, VPL>(all, A, m, unused, lane);
        double Z = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++) Z += all[i] > minus_inf() ? route_exp(all[i] - m) : 0.0;
        Z = row_sum<LPR>(Z, lane);
        if (have) w = A.scale * (route_exp(s - m) / Z);
    }
    if (bad) w = __builtin_nan("");
    if (write && l < A.k) {
        A.idx[row * A.k + l] = f;
        A.w[row * A.k + l] = w;
    }
}

// A row whose values lie closer than what was compared can tell has ROUTE_DOUBT for its first index, and is chosen again by
// the next kernel (k_route_settle): in here, the rare way would cost the registers of every row and hold up the last.
constexpr int ROUTE_DOUBT = -2;
template <int LPR, int VPL>
__device__ __forceinline__ void route_row(const RouteArgs& A, long long row, int f, bool bad, bool doubt, bool live, int l, int f0, int lane) {
    doubt = row_any<LPR>(doubt, lane) && !bad;
    finish_row<LPR, VPL>(A, row, bad ? -1 : f, bad, live && !doubt, l, f0, lane);
    if (doubt && live && l == 0) A.idx[row * A.k] = ROUTE_DOUBT;
}
__device__ __forceinline__ void clear_counts(const RouteArgs& A) {
    if (A.counts && blockIdx.x == 0) {                       // added up by the last kernel
        for (int f = threadIdx.x; f < A.F; f += ROUTE_T) A.counts[f] = 0;
    }
}
// A workgroup that is alone, with no row left in doubt, counts what it wrote itself.
__device__ __forceinline__ void count_here(const RouteArgs& A) {
    if (!A.count_here) return;
    __syncthreads();                                         // the zeros and the indices are written
    for (int i = threadIdx.x; i < A.T * A.k; i += ROUTE_T) {
        const int f = A.idx[i];
        if (f >= 0) atomicAdd(&A.counts[f], 1);
    }
}

// 32- and 64-bit scores without a bias: 64-bit keys.  GROUPED: the groups are chosen by rough shares.
template <int LPR, int VPL, int K, bool GROUPED>
__global__ __launch_bounds__(ROUTE_T) void k_route64(RouteArgs A) {
    extern __shared__ __attribute__((aligned(16))) double route_lds[];
    constexpr int ROWS = ROUTE_T / LPR;
    const int lane = threadIdx.x & 63, sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    double* crow = route_lds + sub * (A.F + A.groups + 1);   // groups only
    // 24-bit scores are compared as they are: scaled, they could need the bits that the filter's number takes
    const bool as_read = A.dtype != WN_F64;
    clear_counts(A);
    for (long long base = (long long)blockIdx.x * ROWS; base < A.T; base += (long long)gridDim.x * ROWS) {
        const bool live = base + sub < A.T;
        const long long row = live ? base + sub : A.T - 1;
        int f0 = l * VPL;
        asm volatile("" : "+v"(f0));                         // what follows from it is not kept from row to row
        double c[VPL], keys[VPL], m;
        bool bad, doubt = false;
        load_row<LPR, VPL>(c, A, row, f0);
#pragma unroll
        for (int i = 0; i < VPL; i++) keys[i] = A.score_scale > 0 ? c[i] : -c[i];
        scale_row<LPR, VPL>(c, A, m, bad, lane);
#pragma unroll
        for (int i = 0; i < VPL; i++) keys[i] = (as_read && c[i] != minus_inf()) ? keys[i] : c[i];
        if constexpr (GROUPED) {
            double e[VPL], sum = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                e[i] = A.sigmoid ? rough_sigmoid((float)c[i]) : rough_exp((float)(c[i] - m));
                e[i] = c[i] > minus_inf() ? e[i] : 0.0;
                sum += e[i];
            }
            const double inv = A.sigmoid ? 1.0 : 1.0 / row_sum<LPR>(sum, lane);
#pragma unroll
            for (int i = 0; i < VPL; i++) e[i] = c[i] > minus_inf() ? e[i] * inv : minus_inf();
            const unsigned keep = choose_groups<LPR, VPL>(e, 2 * ROUTE_SLACK, A, crow, l, f0, lane, doubt);
#pragma unroll
            for (int i = 0; i < VPL; i++) keys[i] = (keep >> i) & 1 ? keys[i] : minus_inf();
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) c[i] = keys[i];
        double top[K], mine = minus_inf(), last = minus_inf();
#pragma unroll
        for (int i = 0; i < VPL; i++) keys[i] = keyed(keys[i], f0 + i);
        largest_own<VPL, K>(keys, top);
        largest_of_lanes<LPR, K>(top, lane);
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = (l == i && i < A.k) ? top[i] : mine;
            last = (i == A.k - 1) ? top[i] : last;
        }
        const int f = mine > minus_inf() ? filter_of(mine) : -1;
        if (!as_read) {
            // Values this close may have changed places.  Of the chosen ones neighbours are looked at, around the last of
            // them every value; equal ones stand in order of the filter already.  The bits given up are 2^-42 of a value, or
            // less than 1024 of the smallest numbers where values are no larger than 2^-1022.
            constexpr double SMALLEST = 2048 * 0x1p-1074;
            const double own = f >= 0 ? A.score_scale * score_at(A, row, f) : 0.0;
            const double next_own = __shfl_down(own, 1, 64), next = __shfl_down(mine, 1, 64);
            doubt |= l + 1 < A.k && next > minus_inf() && own != next_own &&
                     mine - next <= 0x1p-40 * __builtin_fmax(__builtin_fabs(mine), __builtin_fabs(next)) + SMALLEST;
            const double at_last = __shfl(own, (lane - l) + A.k - 1, 64), slack = 0x1p-40 * __builtin_fabs(last) + SMALLEST;
#pragma unroll
            for (int i = 0; i < VPL; i++) doubt |= last > minus_inf() && c[i] != at_last && c[i] >= last - slack && c[i] <= last + slack;
        }
        route_row<LPR, VPL>(A, row, f, bad, doubt, live, l, f0, lane);
    }
    count_here(A);
}

// With a bias, or 16-bit scores: 32-bit keys.  A 16-bit score stands in the upper half of its key as it is (in an order of
// unsigned numbers).  With a bias the upper bits are the rough share plus bias, as a fraction of the range that the biases
// leave for it.

// a lane's scores as they are in memory; those beyond the filters are others of the row
template <class S, int VPL>
__device__ __forceinline__ void fetch_chunk(S (&v)[VPL], const RouteArgs& A, long long row, int f0) {
    const S* p = (const S*)A.scores + row * A.rs + f0 * A.cs;
    const int most = A.F - 1 - f0;
    if (A.cs == 1 && A.F % VPL == 0) {                       // whole chunks, or none
        if (most < 0) p -= f0;
        __builtin_memcpy(v, p, sizeof(v));                   // wide loads: the hardware takes any alignment
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) v[i] = p[(i < most ? i : most) * A.cs];
    }
}
// s = scale * score as floats: finite ones within +-3e38, -inf for closed filters.  bad: a NaN or +inf among them.
template <class S, int VPL>
__device__ __forceinline__ void scale_chunk(float (&s)[VPL], const S (&v)[VPL], const RouteArgs& A, int f0, bool& bad) {
    const float scale = (float)A.score_scale;
    const int most = A.F - 1 - f0;
    bool odd = true;                                         // values that need a second look
    if constexpr (sizeof(S) < 8) {
        float large = 0;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            s[i] = (float)widen(v[i]) * scale;
            large += __builtin_fabsf(s[i]);                  // finite if they all are, and not too large
        }
        odd = !(large < 3e38f) || most < VPL - 1;
    }
    if (!__any(odd)) return;
    const float closed = A.score_scale > 0 ? -__builtin_huge_valf() : __builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        if constexpr (sizeof(S) == 8) {
            const double d = A.score_scale * v[i];
            bad |= i <= most && !(d <= 1.7976931348623157e308);
            s[i] = (i <= most && d != minus_inf()) ? (float)key_min(key_max(d, -3e38), 3e38) : -__builtin_huge_valf();
        } else {
            const float x = (float)widen(v[i]);
            bad |= i <= most && (x != x || x == -closed);
            s[i] = (i <= most && x != closed) ? __builtin_amdgcn_fmed3f(x * scale, -3e38f, 3e38f) : -__builtin_huge_valf();
        }
    }
}
// a 16-bit score as an unsigned number of the same order, -0 as 0
__device__ __forceinline__ unsigned ordered16(unsigned u) {
    u = (u == 0x8000u) ? 0 : u;
    return (u & 0x8000u) ? (u ^ 0xFFFFu) : (u | 0x8000u);
}
__device__ __forceinline__ unsigned bits16(f16_bits v) { return v.v; }
__device__ __forceinline__ unsigned bits16(bf16_bits v) { return v.v; }
__device__ __forceinline__ unsigned bits16(float) { return 0; }
__device__ __forceinline__ unsigned bits16(double) { return 0; }

// Three waves per SIMD and as many workgroups as that makes: 65536 x 256 bf16 scores with bias and groups 52 us (at 16 scores a
// lane with 68 bytes of scratch memory per lane, 64-bit scores 120 ... 132); two waves 55, one 74, four (with more of it) 93.
template <class S, int LPR, int VPL, int K>
__global__ __launch_bounds__(ROUTE_T, 3) void k_route32(RouteArgs A) {
    extern __shared__ __attribute__((aligned(16))) double route_lds[];
    constexpr int ROWS = ROUTE_T / LPR;
    constexpr unsigned LOW = LPR * VPL - 1;                  // bits of a key that hold the filter's number
    constexpr float STEPS = 0.99f * (float)(0xFFFFFFFFu / (LOW + 1));   // that the upper bits are cut into
    constexpr float NONE = -__builtin_huge_valf();
    const int lane = threadIdx.x & 63, sub = threadIdx.x / LPR, l = threadIdx.x % LPR;
    double* crow = route_lds + sub * (A.F + A.groups + 1);   // groups only
    const bool biased = A.bias != nullptr, grouped = A.kept < A.groups;
    // key = p * steps + place[i]: the share on top of where its filter's bias puts it
    float bias[VPL], place[VPL], b_min = 3e38f, b_max = -3e38f;
    bool wild = (biased || grouped) && !(__builtin_fabs(A.score_scale) >= 1e-30 && __builtin_fabs(A.score_scale) <= 1e30);
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int f = l * VPL + i;
        const double b = biased ? A.bias[f < A.F ? f : A.F - 1] : 0.0;
        bias[i] = b > minus_inf() ? (float)b : NONE;
        wild |= b > 1e30 || (b > minus_inf() && b < -1e30);
        if (bias[i] > NONE) { b_min = __builtin_fminf(b_min, bias[i]); b_max = __builtin_fmaxf(b_max, bias[i]); }
    }
    b_min = -(float)row_max<LPR>(-(double)b_min, lane);
    b_max = (float)row_max<LPR>((double)b_max, lane);
    wild = row_any<LPR>(wild, lane) || !(b_min <= b_max);    // biases that no range holds: every row goes the long way
    const float range = 1.0f + (b_max - b_min);
    const float steps = STEPS / range;
#pragma unroll
    for (int i = 0; i < VPL; i++) place[i] = (bias[i] - b_min) * steps + 1.0f;
    clear_counts(A);
    for (long long base = (long long)blockIdx.x * ROWS; base < A.T; base += (long long)gridDim.x * ROWS) {
        const bool live = base + sub < A.T;
        const long long row = live ? base + sub : A.T - 1;
        int f0 = l * VPL;
        asm volatile("" : "+v"(f0));                         // what follows from it is not kept from row to row
        float s[VPL], m = 0;
        unsigned keys[VPL], top[K];
        bool bad = false, doubt = wild;
        {
            S v[VPL];
            fetch_chunk<S, VPL>(v, A, row, f0);
            scale_chunk<S, VPL>(s, v, A, f0, bad);
            if (sizeof(S) == 2 && !biased) {
                // by the score itself: its order is that of the shares, and equal shares of different scores are not
                const unsigned flip = A.score_scale > 0 ? 0u : 0xFFFFu;
#pragma unroll
                for (int i = 0; i < VPL; i++) {
                    const unsigned o = ((ordered16(bits16(v[i])) ^ flip) << 16) | (LOW - (unsigned)(f0 + i));
                    keys[i] = s[i] > NONE ? o : 0u;
                }
            }
        }
        bad = row_any<LPR>(bad, lane);
        float slack = 0;
        if (biased || grouped) {
            float p[VPL];
            if (A.sigmoid) {
#pragma unroll
                for (int i = 0; i < VPL; i++) p[i] = rough_sigmoid(s[i]);
                slack = 2 * (float)ROUTE_SLACK;
            } else {
                m = s[0];
#pragma unroll
                for (int i = 1; i < VPL; i++) m = __builtin_fmaxf(m, s[i]);
                m = (float)row_max<LPR>((double)m, lane);
                float sum = 0;
#pragma unroll
                for (int i = 0; i < VPL; i++) {
                    p[i] = s[i] > NONE ? rough_exp(s[i] - m) : 0.0f;
                    sum += p[i];
                }
                const float inv = __builtin_amdgcn_rcpf((float)row_sum<LPR>((double)sum, lane));
#pragma unroll
                for (int i = 0; i < VPL; i++) p[i] *= inv;
                // a float score is off by its own 2^-23, and so is the logarithm of the share
                slack = 2 * ((float)ROUTE_SLACK + __builtin_fabsf(m) * 5e-7f);
            }
            if (biased) {
#pragma unroll
                for (int i = 0; i < VPL; i++) {
                    const unsigned o = ((unsigned)__builtin_fmaf(p[i], steps, place[i]) * (LOW + 1)) | (LOW - (unsigned)(f0 + i));
                    keys[i] = (s[i] > NONE && bias[i] > NONE) ? o : 0u;
                }
                slack += 2.4e-7f * __builtin_fmaxf(__builtin_fabsf(b_min), __builtin_fabsf(b_max));
            }
            if (grouped) {
#pragma unroll
                for (int i = 0; i < VPL; i++) p[i] = s[i] > NONE ? p[i] + bias[i] : NONE;
                const unsigned keep = choose_groups<LPR, VPL>(p, slack, A, crow, l, f0, lane, doubt);
#pragma unroll
                for (int i = 0; i < VPL; i++) keys[i] &= (unsigned)((int)(keep << (31 - i)) >> 31);
            }
        }
        unsigned mine = 0, last = 0;
        {
            unsigned v[VPL];
#pragma unroll
            for (int i = 0; i < VPL; i++) v[i] = keys[i];
            largest_own<VPL, K>(v, top);
        }
        largest_of_lanes<LPR, K>(top, lane);
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = (l == i && i < A.k) ? top[i] : mine;
            last = (i == A.k - 1) ? top[i] : last;
        }
        const int f = mine ? (int)(LOW - (mine & LOW)) : -1;
        if (biased) {
            // Values within the slack of each other are not told apart by their keys.  Of the chosen ones neighbours are
            // looked at, around the last of them every value.
            const unsigned near = (unsigned)__builtin_fminf(slack * steps + STEPS * 4.8e-7f + 2.0f, STEPS) * (LOW + 1) + LOW;
            const unsigned next = __shfl_down(mine, 1, 64), lo = last > near ? last - near : 1u;
            int within = 0;
#pragma unroll
            for (int i = 0; i < VPL; i++) within += keys[i] >= lo;
            within = row_count<LPR>(within, lane);
            doubt |= (l + 1 < A.k && next && mine - next <= near) || (last && within > A.k);
        }
        route_row<LPR, VPL>(A, row, f, bad, doubt, live, l, f0, lane);
    }
    count_here(A);
}

// A marked row in 64 bits and round by round, by one wave with the values in LDS: lane j < k returns its j-th filter.  Rows
// come here one at a time, so that a row's latency counts: for 256 scores with bias and groups some 2.8 k cycles for the
// scores, 3.8 k for the shares, 4.9 k for the groups and 0.9 k a round (two exchanges, a write and a read of LDS each).
__device__ __forceinline__ int choose_exactly(const RouteArgs& A, long long row, double* crow, int lane) {
    const bool shares = A.bias || A.kept < A.groups;
                double m = minus_inf(), Z = 0;
#pragma nounroll
                for (int f = lane; f < A.F; f += 64) {
                    const double v = A.score_scale * score_at(A, row, f);
                    m = key_max(m, v);
                    crow[f] = v;
                }
                route_lds_order();
                if (shares) {
                    if (!A.sigmoid) {
                        m = row_max<64>(m, lane);
#pragma nounroll
                        for (int f = lane; f < A.F; f += 64) Z += crow[f] > minus_inf() ? route_exp(crow[f] - m) : 0.0;
                        Z = row_sum<64>(Z, lane);
                    }
#pragma nounroll
                    for (int f = lane; f < A.F; f += 64) {
                        const double v0 = crow[f];
                        double v = A.sigmoid ? route_sigmoid(v0) : route_exp(v0 - m) / Z;
                        if (A.bias) v += A.bias[f];
                        crow[f] = (v0 > minus_inf() && v > minus_inf()) ? v : minus_inf();
                    }
                    route_lds_order();
                }
                if (A.kept < A.groups) {
                    bool doubt = false;
                    const unsigned long long keep = kept_groups<64, double>(0.0, A, crow, lane, doubt);
#pragma nounroll
                    for (int f = lane; f < A.F; f += 64) {
                        const bool open = (keep >> (((unsigned)f * A.per_magic) >> 20)) & 1;
                        if (!open) crow[f] = minus_inf();
                        else if (!A.bias && crow[f] > minus_inf()) crow[f] = A.score_scale * score_at(A, row, f);
                    }
                    route_lds_order();
                }
                // a lane keeps the best of its consecutive filters; only the one that gave it away looks again
                const int own = (A.F + 63) / 64;
                const auto look = [&](double& best, int& at) {
                    best = minus_inf();
                    for (int i0 = 0; i0 < own; i0 += 4) {    // four on their way at a time
                        double v[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] = crow[min(lane * own + i0 + i, A.F - 1)];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int f = lane * own + i0 + i;
                            const bool better = i0 + i < own && f < A.F && v[i] > best;
                            at = better ? f : at;
                            best = better ? v[i] : best;
                        }
                    }
                };
                double best;
                int at = 0, mine = -1;
                look(best, at);
#pragma nounroll
                for (int j = 0; j < A.k; j++) {
                    const double top = row_max<64>(best, lane);
                    if (!(top > minus_inf())) break;
                    const int first = __builtin_ctzll(__ballot(best == top));    // the lowest lane has the lowest filter
                    const int f = __builtin_amdgcn_readlane(at, first);
                    if (lane == j) mine = f;
                    if (lane == first) {
                        crow[f] = minus_inf();
                        look(best, at);
                    }
                }
    return mine;
}

// After k_route32 and k_route64: the rows that they marked (a workgroup's waves share its marked rows; equal values among
// 16-bit scores under equal biases come here too, and may be many), and counts[f] += entries of idx that name f, by a
// histogram per workgroup in LDS and one addition per filter (whole numbers, so that their order does not matter).
// 512 threads: with 1024 the registers spill, and setting up scratch memory alone takes every workgroup 8 k cycles (65536 x 256
// bf16 with bias and groups 71 us against 64; 65536 x 64 with bias and groups 43 against 35); 256 have too few waves for many
// marked rows (65536 x 1024 f32 with a bias: 197 us with 1024 threads, 208 with 512, 245 with 256).
constexpr int SETTLE_T = 512;
__global__ __launch_bounds__(SETTLE_T) void k_route_settle(RouteArgs A) {
    extern __shared__ __attribute__((aligned(16))) double route_lds[];
    __shared__ int hist[WN_MAX_EXPERTS], marked[SETTLE_T], marks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double* crow = route_lds + wave * (A.F + A.groups + 1);
    for (int f = threadIdx.x; f < A.F; f += SETTLE_T) hist[f] = 0;
    for (long long base = (long long)blockIdx.x * A.settle_rows; base < A.T; base += (long long)gridDim.x * A.settle_rows) {
        const int rows = (int)(A.T - base < A.settle_rows ? A.T - base : A.settle_rows);
        if (A.doubts) {
            __syncthreads();
            if (threadIdx.x == 0) marks = 0;
            __syncthreads();
            if ((int)threadIdx.x < rows && A.idx[(base + threadIdx.x) * A.k] == ROUTE_DOUBT) marked[atomicAdd(&marks, 1)] = threadIdx.x;
            __syncthreads();
            for (int i = wave; i < marks; i += SETTLE_T / 64) {
                const long long row = base + marked[i];
                const int f = choose_exactly(A, row, crow, lane);
                finish_row<64, WN_MAX_EXPERTS / 64>(A, row, f, false, true, lane, lane * (WN_MAX_EXPERTS / 64), lane);
            }
        }
        __syncthreads();
        if (A.counts) {
            for (int i = threadIdx.x; i < rows * A.k; i += SETTLE_T) {
                const int f = A.idx[base * A.k + i];
                if (f >= 0) atomicAdd(&hist[f], 1);
            }
        }
    }
    __syncthreads();
    if (!A.counts) return;
    for (int f = threadIdx.x; f < A.F; f += SETTLE_T) {
        if (hist[f]) atomicAdd(&A.counts[f], hist[f]);
    }
}

// ---- backward -------------------------------------------------------------------------------------------------

// Rounding twice, to a float and then to bf16, differs from rounding once only where the float is in the middle between two
// of the shorter type: one chunk in some thousand, which is then rounded the long way.
template <class S, int VPL>
__device__ __forceinline__ void narrow_chunk(S (&v)[VPL], const double (&ds)[VPL]) {
#pragma unroll
    for (int i = 0; i < VPL; i++) v[i] = narrow<S>(ds[i]);
}
template <int VPL>
__device__ __forceinline__ void narrow_chunk(bf16_bits (&v)[VPL], const double (&ds)[VPL]) {
    bool middle = false;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const float f = (float)ds[i];
        middle |= (__builtin_bit_cast(unsigned, f) & 0xFFFFu) == 0x8000u;
        v[i] = {__builtin_bit_cast(unsigned short, (__bf16)f)};
    }
    if (__any(middle)) {
#pragma unroll
        for (int i = 0; i < VPL; i++) v[i] = narrow<bf16_bits>(ds[i]);
    }
}
template <class S, int LPR, int VPL>
__device__ __forceinline__ void store_chunk(const double (&ds)[VPL], const RouteArgs& A, long long row, int f0) {
    S* p = (S*)A.dscores + row * A.rs + f0 * A.cs;
    S v[VPL];
    narrow_chunk(v, ds);
    if (A.cs == 1 && A.F == LPR * VPL) {
        __builtin_memcpy(p, v, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            if (f0 + i < A.F) p[i * A.cs] = v[i];
        }
    }
}

// What the chosen filters get on their own reaches the lanes that hold them through a row of LDS that is zero otherwise.
// Three waves per SIMD: 65536 x 256 bf16, full softmax, 43 us (at 16 scores a lane with 28 bytes of scratch memory per lane);
// two 56, four (with more of it) 51.
template <int LPR, int VPL>
__global__ __launch_bounds__(ROUTE_T, 3) void k_route_backward(RouteArgs A) {
    constexpr int ROWS = ROUTE_T / LPR;
    __shared__ __attribute__((aligned(16))) double own[ROWS][LPR * VPL];
    const int lane = threadIdx.x & 63, sub = threadIdx.x / LPR, l = threadIdx.x % LPR, f0 = l * VPL;
    const int lane0 = lane - l;
    double* mine = own[sub];
#pragma unroll
    for (int i = 0; i < VPL; i++) mine[f0 + i] = 0;
    route_lds_order();
    for (long long base = (long long)blockIdx.x * ROWS; base < A.T; base += (long long)gridDim.x * ROWS) {
        const bool live = base + sub < A.T;
        const long long row = live ? base + sub : A.T - 1;
        const int f = l < A.k ? A.idx_in[row * A.k + l] : -1;
        const bool have = f >= 0 && f < A.F;
        const double g = have ? A.scale * A.dw[row * A.k + l] : 0.0;
        const double s = have ? A.score_scale * score_at(A, row, f) : minus_inf();
        double ds[VPL], d = 0;                               // d: what the chosen filter of this lane gets on its own
#pragma unroll
        for (int i = 0; i < VPL; i++) ds[i] = 0;
        if (A.renorm) {
            const double lp = have ? log_share(s, A.sigmoid) : minus_inf();
            const double top = row_max<LPR>(lp, lane);
            const double u = (have && lp > minus_inf()) ? exp(lp - top) : 0.0;
            const double sum = row_sum<LPR>(u, lane);
            const double share = u > 0 ? u / sum : 0.0;
            const double mean = row_sum<LPR>(have ? share * g : 0.0, lane);
            d = have ? share * (g - mean) : 0.0;
            if (have && A.sigmoid) d *= 1.0 / (1.0 + exp(s));
        } else if (A.sigmoid) {
            const double e = exp(-__builtin_fabs(s)), t = 1.0 / (1.0 + e);
            d = have ? g * (e * t * t) : 0.0;                // p (1 - p)
        } else if (__any(have)) {
            double m = minus_inf(), Z = 0;
            load_row<LPR, VPL>(ds, A, row, f0);
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                ds[i] *= A.score_scale;
                m = key_max(m, ds[i]);
            }
            m = row_max<LPR>(m, lane);
            bool bad = false;
#pragma unroll
            for (int i = 0; i < VPL; i++) {
                bad |= !(ds[i] <= 1.7976931348623157e308);
                ds[i] = route_exp(ds[i] - m);                // (-inf: 0, and so is -inf - -inf)
                Z += ds[i];
            }
            Z = row_sum<LPR>(Z, lane);
            if (row_any<LPR>(bad, lane)) Z = __builtin_nan("");
            const double p = (have && s != minus_inf()) ? exp(s - m) / Z : 0.0;
            d = have ? g * p : 0.0;
            // a row without a chosen filter has no gradient, whatever its scores, nor has one without an open filter
            const double sum = row_sum<LPR>(d, lane);
            const double all = (row_any<LPR>(have, lane) && m > minus_inf()) ? -sum / Z * A.score_scale : 0.0;
#pragma unroll
            for (int i = 0; i < VPL; i++) ds[i] *= all;
        }
        d *= A.score_scale;
        // The lane that finds its own number where it left it speaks for its filter.  One that does not shares it: a filter
        // that is named twice (wn_route does not) gets both shares, in the order of the entries, from the first of them.
        if (have) mine[f] = l;
        route_lds_order();
        bool first = have && mine[have ? f : 0] == l;
        double sum = d;
        if (__any(have && !first)) {
            first = have;
            sum = 0;
            for (int j = 0; j < A.k; j++) {
                const int fj = __shfl(f, lane0 + j, 64);
                const double dj = __shfl(d, lane0 + j, 64);
                if (fj == f) {
                    sum += dj;
                    first &= j >= l;
                }
            }
        }
        if (first) mine[f] = sum;
        route_lds_order();
#pragma unroll
        for (int i = 0; i < VPL; i++) ds[i] += mine[f0 + i];
        route_lds_order();
        if (first) mine[f] = 0;
        if (live) {
            switch (A.dtype) {
                case WN_F64: store_chunk<double, LPR, VPL>(ds, A, row, f0); break;
                case WN_F32: store_chunk<float, LPR, VPL>(ds, A, row, f0); break;
                case WN_F16: store_chunk<f16_bits, LPR, VPL>(ds, A, row, f0); break;
                default: store_chunk<bf16_bits, LPR, VPL>(ds, A, row, f0);
            }
        }
    }
}

}  // namespace wn

namespace {

using wn::fail;

struct RouteClass { const void* forward; const void* backward; int lpr; };

// The forward kernel: 64-bit keys (with groups or without) for 32- and 64-bit scores without a bias, else 32-bit ones.
template <int LPR, int VPL, int K>
const void* route_kernel(int dtype, bool biased, bool grouped) {
    switch (dtype) {
        case WN_F16: return (const void*)&wn::k_route32<wn::f16_bits, LPR, VPL, K>;
        case WN_BF16: return (const void*)&wn::k_route32<wn::bf16_bits, LPR, VPL, K>;
    }
    if (biased) return dtype == WN_F64 ? (const void*)&wn::k_route32<double, LPR, VPL, K> : (const void*)&wn::k_route32<float, LPR, VPL, K>;
    return grouped ? (const void*)&wn::k_route64<LPR, VPL, K, true> : (const void*)&wn::k_route64<LPR, VPL, K, false>;
}
template <int LPR, int VPL>
RouteClass route_class_of(int k, int dtype, bool biased, bool grouped) {
    return {k <= 2   ? route_kernel<LPR, VPL, 2>(dtype, biased, grouped)
            : k <= 4 ? route_kernel<LPR, VPL, 4>(dtype, biased, grouped)
            : k <= 8 ? route_kernel<LPR, VPL, 8>(dtype, biased, grouped)
                     : route_kernel<LPR, VPL, 16>(dtype, biased, grouped),
            (const void*)&wn::k_route_backward<LPR, VPL>, LPR};
}
RouteClass route_class(int F, int k, int dtype, bool biased, bool grouped) {
    if (F <= 16) return route_class_of<16, 1>(k, dtype, biased, grouped);
    if (F <= 32) return route_class_of<16, 2>(k, dtype, biased, grouped);
    if (F <= 64) return route_class_of<16, 4>(k, dtype, biased, grouped);
    if (F <= 128) return route_class_of<16, 8>(k, dtype, biased, grouped);
    if (F <= 256) return route_class_of<16, 16>(k, dtype, biased, grouped);
    if (F <= 512) return route_class_of<32, 16>(k, dtype, biased, grouped);
    return route_class_of<64, 16>(k, dtype, biased, grouped);
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
    if (!(__builtin_fabs(r->score_scale) <= 1e100 && __builtin_fabs(r->score_scale) >= 1e-100))
        return fail(ctx, WN_ERR_ARG, "score_scale is zero, not finite, or beyond 1e-100 ... 1e100");
    if (T == 0) return WN_OK;
    const long long far = 1LL << 40;
    if (rs < 0 || cs < 0 || rs > far || cs > far) return fail(ctx, WN_ERR_ARG, "bad strides");
    // no two scores in one place: filters inside rows, or rows inside filters
    const bool rows_outside = (F == 1 || cs >= 1) && (T == 1 || rs > (F - 1) * cs);
    const bool rows_inside = (T == 1 || rs >= 1) && (F == 1 || (__int128)cs > (__int128)(T - 1) * rs);
    if (!rows_outside && !rows_inside) return fail(ctx, WN_ERR_ARG, "strides make scores overlap");
    if (!scores) return fail(ctx, WN_ERR_ARG, "null pointer");
    if (!wn::aligned_to(scores, es)) return fail(ctx, WN_ERR_ARG, "misaligned pointer");
    A.scores = scores; A.dtype = dtype; A.rs = rs; A.cs = cs;
    A.T = T; A.F = F; A.k = r->k;
    const bool grouped = r->groups_kept < r->groups;         // all groups kept: none, whatever their number
    A.groups = grouped ? r->groups : 1; A.kept = grouped ? r->groups_kept : 1; A.per = F / A.groups;
    A.per_magic = ((1u << 20) + A.per - 1) / A.per;
    A.sigmoid = r->score == WN_SCORE_SIGMOID; A.renorm = r->renormalise != 0;
    A.scale = r->scale; A.score_scale = r->score_scale;
    return WN_OK;
}

// The memory of scores, or of their gradients, as pieces of the direction whose elements lie closer together.
wn::Memory score_memory(const char* name, const void* at, const wn::RouteArgs& A) {
    const unsigned long long es = wn::element_bytes(A.dtype);
    const bool rows_outside = A.T == 1 || (A.F > 1 ? A.rs > A.cs : true);
    const unsigned long long inner = rows_outside ? (A.F - 1) * A.cs + 1 : (A.T - 1) * A.rs + 1;
    return {name, at, inner * es, (unsigned long long)(rows_outside ? A.T : A.F), (unsigned long long)(rows_outside ? A.rs : A.cs) * es};
}
// Whether gradients `by` elements behind the scores, at the same strides, lie on scores other than their own.
bool on_other_scores(long long by, const wn::RouteArgs& A) {
    if (by < 0) by = -by;
    const bool rows_outside = A.T == 1 || (A.F > 1 ? A.rs > A.cs : true);
    // outer and inner stride and counts: (T or F) pieces of (F or T) elements
    const long long so = rows_outside ? A.rs : A.cs, no = rows_outside ? A.T : A.F;
    const long long si = rows_outside ? A.cs : A.rs, ni = rows_outside ? A.F : A.T;
    if (by == 0) return false;
    const auto inside = [&](long long d) { return d == 0 || (ni > 1 && d % si == 0 && std::abs(d / si) < ni); };
    if (no == 1) return inside(by);
    const long long i = by / so;                             // inner pieces are shorter than so: piece i or the next
    return (i < no && inside(by - i * so)) || (i + 1 < no && inside(by - (i + 1) * so));
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
            const unsigned long long entries = (unsigned long long)T * A.k;
            rc = wn::refuse_overlaps(ctx, {{"idx", idx_dev, entries * 4}, {"w", w_dev, entries * 8}, {"counts", counts_dev, 4ull * F}},
                                     {score_memory("scores", scores_dev, A), {"bias", bias_dev, 8ull * F}});
            if (rc) return rc;
        } else if (!counts_dev) {
            return WN_OK;
        } else if (!wn::aligned_to(counts_dev, 4)) {
            return fail(ctx, WN_ERR_ARG, "misaligned pointer");
        }
        const RouteClass K = route_class(F, routing->k, dtype, bias_dev, routing->groups_kept < routing->groups);
        const int rows = wn::ROUTE_T / K.lpr;
        // as many workgroups as are on the chip at a time: what they set up (biases, the first instructions) serves more rows
        const long long grid = std::max(1LL, std::min<long long>(((long long)T + rows - 1) / rows, (long long)ctx->numCU * (F > 128 ? 3 : 6)));
        A.doubts = bias_dev || A.kept < A.groups || dtype == WN_F64;
        A.count_here = counts_dev && grid == 1 && !A.doubts;
        const size_t values = (size_t)(F + A.groups + 1) * sizeof(double);
        rc = wn::launch_kernel(ctx, K.forward, (unsigned)grid, wn::ROUTE_T, A.kept < A.groups ? rows * values : 0, A);
        if (rc || T == 0) return rc;
        if (!A.doubts && (!counts_dev || A.count_here)) return WN_OK;
        // rows spread over the chip, but no fewer than 256 to a workgroup, each of which adds to the counts
        A.settle_rows = (int)std::min<long long>(wn::SETTLE_T, std::max<long long>(256, ((long long)T + ctx->numCU - 1) / ctx->numCU));
        const long long sgrid = std::min<long long>(((long long)T + A.settle_rows - 1) / A.settle_rows, ctx->numCU);
        return wn::launch_kernel(ctx, (const void*)&wn::k_route_settle, (unsigned)sgrid, wn::SETTLE_T, A.doubts ? wn::SETTLE_T / 64 * values : 0, A);
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
        const unsigned long long entries = (unsigned long long)T * A.k;
        rc = wn::refuse_overlaps(ctx, {score_memory("dscores", dscores_dev, A)}, {{"idx", idx_dev, entries * 4}, {"dw", dw_dev, entries * 8}});
        if (rc) return rc;
        const long long es = (long long)wn::element_bytes(dtype);
        if (on_other_scores(((const char*)dscores_dev - (const char*)scores_dev) / es, A)) return fail(ctx, WN_ERR_ARG, "dscores overlaps scores of other places");
        A.idx_in = idx_dev; A.dw = dw_dev; A.dscores = dscores_dev;
        const RouteClass K = route_class(F, routing->k, dtype, false, false);
        const int rows = wn::ROUTE_T / K.lpr;
        const long long grid = std::min<long long>(((long long)T + rows - 1) / rows, (long long)ctx->numCU * 16);
        return wn::launch_kernel(ctx, K.backward, (unsigned)grid, wn::ROUTE_T, 0, A);
    });
}

}  // extern "C"
