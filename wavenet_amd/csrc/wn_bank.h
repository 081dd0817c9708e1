// Shared by the routed filter bank (wn_route.hip, wn_checkpoint.hip, wn_bank.hip, wn_bank_np.hip): argument blocks,
// element types, the 8-bit checkpoint format, and the host-side frame of an entry point.
#pragma once

#include <hip/hip_runtime.h>

#include <exception>
#include <initializer_list>
#include <string>

#include "wavenet_hip.h"
#include "wn_device.h"
#include "wn_internal.h"

namespace wn {

// ---- entry points -------------------------------------------------------------------------------------

// The context's device for the length of a call; the caller's device is current again afterwards.
struct DeviceScope {
    int before = -1;
    bool moved = false;
    hipError_t status;
    explicit DeviceScope(int device) {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before != device) {
            status = hipSetDevice(device);
            moved = status == hipSuccess;
        }
    }
    ~DeviceScope() {
        if (moved) (void)hipSetDevice(before);
    }
};

// Runs the body of an entry point: null context, device, and no exception past the C boundary.
template <class Body>
int entry(wn_context* ctx, Body body) noexcept {
    if (!ctx) return WN_ERR_ARG;
    try {
        DeviceScope scope(ctx->device);
        WN_HIP(ctx, scope.status);
        return body();
    } catch (const std::exception& e) {
        try {
            return fail(ctx, WN_ERR_HIP, e.what());
        } catch (...) {
        }
    } catch (...) {
    }
    return WN_ERR_HIP;
}

template <class Args>
int launch_kernel(wn_context* ctx, const void* func, unsigned grid, unsigned threads, size_t shmem, Args& args) {
    if (!func) return fail(ctx, WN_ERR_UNSUPPORTED, "no kernel compiled for this configuration");
    if (shmem > 64 * 1024) {
        size_t& have = ctx->lds_configured[func];
        if (have < shmem) {
            WN_HIP(ctx, hipFuncSetAttribute(func, hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem));
            have = shmem;
        }
    }
    void* p[] = {&args};
    WN_HIP(ctx, hipLaunchKernel(func, dim3(grid), dim3(threads), p, shmem, ctx->stream));
    return WN_OK;
}

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Memory of an argument: `pieces` of `bytes` each, `stride` bytes apart (at least a piece); a null pointer is none.
struct Memory {
    const char* name;
    const void* at;
    unsigned long long bytes, pieces = 1, stride = 0;
};
// whether the first, in one piece, shares a byte with the second
inline bool meets(const Memory& a, const Memory& b) {
    if (!a.at || !b.at || !a.bytes || !b.bytes || !b.pieces) return false;
    const unsigned long long x = (uintptr_t)a.at, y = (uintptr_t)b.at;
    // the first piece that ends behind the start of a
    const unsigned long long i = x < y + b.bytes ? 0 : b.pieces == 1 ? 1 : (x - y - b.bytes) / b.stride + 1;
    return i < b.pieces && y + i * b.stride < x + a.bytes;
}
// No output may lie in an input or in another output.  Either is in one piece, or all that it is compared with are.
inline int refuse_overlaps(wn_context* ctx, std::initializer_list<Memory> outputs, std::initializer_list<Memory> inputs) {
    const auto refuse = [&](const Memory& o, const Memory& m) {
        return fail(ctx, WN_ERR_ARG, std::string(o.name) + " overlaps " + m.name);
    };
    for (const Memory* o = outputs.begin(); o != outputs.end(); o++) {
        for (const Memory& i : inputs)
            if (o->pieces > 1 ? meets(i, *o) : meets(*o, i)) return refuse(*o, i);
        for (const Memory* p = o + 1; p != outputs.end(); p++)
            if (o->pieces > 1 ? meets(*p, *o) : meets(*o, *p)) return refuse(*o, *p);
    }
    return WN_OK;
}

inline size_t element_bytes(int dtype) {
    switch (dtype) {
        case WN_F64: return 8;
        case WN_F32: return 4;
        case WN_F16: case WN_BF16: return 2;
    }
    return 0;
}

// ---- element types: everything is computed in 64 bits, so that reading is exact and writing rounds once ----------

struct f16_bits { unsigned short v; };
struct bf16_bits { unsigned short v; };

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ double widen(float v) { return v; }
__device__ __forceinline__ double widen(f16_bits v) { return (double)(float)__builtin_bit_cast(_Float16, v.v); }
__device__ __forceinline__ double widen(bf16_bits v) { return (double)__builtin_bit_cast(float, (unsigned)v.v << 16); }

// d in 24 bits, rounded to odd: truncated, with the last bit set if anything was cut off.  Rounding that to 13 bits or
// fewer gives what rounding d itself gives, which rounding to the nearest float first does not.
__device__ __forceinline__ float round_to_odd(double d) {
    const float f = (float)d;
    if ((double)f == d || d != d) return f;
    unsigned u = __builtin_bit_cast(unsigned, f);
    if (__builtin_fabs((double)f) > __builtin_fabs(d)) u -= 1;
    return __builtin_bit_cast(float, u | 1u);
}
template <class S> __device__ __forceinline__ S narrow(double d);
template <> __device__ __forceinline__ double narrow<double>(double d) { return d; }
template <> __device__ __forceinline__ float narrow<float>(double d) { return (float)d; }
template <> __device__ __forceinline__ f16_bits narrow<f16_bits>(double d) {
    return {__builtin_bit_cast(unsigned short, (_Float16)round_to_odd(d))};
}
template <> __device__ __forceinline__ bf16_bits narrow<bf16_bits>(double d) {
    return {__builtin_bit_cast(unsigned short, (__bf16)round_to_odd(d))};
}

// ---- 8-bit checkpoints ------------------------------------------------------------------------------------
// Blocks of CKPT_BLOCK consecutive values share a float scale = largest magnitude / 127; a value is kept as the whole
// number q nearest to value / scale and read back as q * scale (7 bits times 24 bits: exact in a double).

constexpr int CKPT_BLOCK = 64;

// amax: the block's largest magnitude, any value not finite already replaced by a NaN
__device__ __forceinline__ float ckpt_scale(double amax) { return (float)(amax / 127.0); }
__device__ __forceinline__ int ckpt_quantise(double x, float scale) {
    if (!(scale > 0.0f && scale <= 3.402823466e38f)) return 0;   // nothing there, or a block that reads back as NaN
    const double r = __builtin_rint(x / (double)scale);
    return (int)__builtin_fmin(127.0, __builtin_fmax(-127.0, r));
}
// The same, unless odd is set, from inv = ckpt_inverse(scale): x * inv is within 2^-45 of x / scale, so that it rounds alike
// but next to the middle between two whole numbers.  Adding 1.5 * 2^52 leaves the nearest whole number in the low bits.
// Values that are not finite are odd, too.
__device__ __forceinline__ double ckpt_inverse(float scale) {
    return (scale > 0.0f && scale <= 3.402823466e38f) ? 1.0 / (double)scale : 0.0;
}
__device__ __forceinline__ int ckpt_quantise_fast(double x, double inv, bool& odd) {
    const double t = x * inv, s = t + 6755399441055744.0;
    odd |= !(__builtin_fabs(t - (s - 6755399441055744.0)) <= 0.499999) || __builtin_fabs(t) > 127.4;
    return __double2loint(s);
}
__device__ __forceinline__ void ckpt_quantise4(int (&b)[4], const double (&v)[4], float scale) {
    const double inv = ckpt_inverse(scale);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = ckpt_quantise_fast(v[i], inv, odd);
    if (__any(odd)) {
#pragma unroll
        for (int i = 0; i < 4; i++) b[i] = ckpt_quantise(v[i], scale);
    }
}
// larger of |a| and |b|, NaN losing: for values of which the odd ones are looked at again
__device__ __forceinline__ double ckpt_max_quick(double a, double b) {
    double r;
    asm("v_max_f64 %0, |%1|, |%2|" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
// |x|, or a NaN for what no scale can hold; the larger of two such magnitudes, NaN winning
__device__ __forceinline__ double ckpt_magnitude(double x) { return __builtin_fabs(x) <= 1.7976931348623157e308 ? __builtin_fabs(x) : __builtin_nan(""); }
__device__ __forceinline__ double ckpt_max(double a, double b) { return (a > b || a != a) ? a : b; }

// ---- routed transforms --------------------------------------------------------------------------------------

struct BankArgs {
    int B, lgR, lgC, k, F, N;
    const double* filters;   // [F][N] taps
    const int* idx;          // [B][k], null: every entry names filter 0
    const double* w;         // [B][k], null: ones
    const double* X;         // [B][n] examples (forward; backward unless a checkpoint is given)
    const signed char* q;    // backward: checkpoint of X, [B][n] whole numbers and one scale per block
    const float* qs;
    signed char* q_out;      // forward: checkpoint to write, optional
    float* qs_out;
    double* Y;               // forward: [B][n]
    const double* D;         // backward: errors on the coefficients
    double* dX;              // [B][n], optional
    double* dw;              // [B][k], optional
    double* grad;            // [B][k][N]
};

}  // namespace wn
