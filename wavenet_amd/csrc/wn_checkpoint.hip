// 8-bit checkpoints of activations on their own: wn_checkpoint_pack, wn_checkpoint_unpack.
#include <algorithm>

#include "wn_bank.h"

namespace wn {

struct CheckpointArgs {
    long long blocks;       // B * nb
    int n, nb;
    long long ld;           // elements between rows of the wide side
    const void* in;
    void* out;
    const signed char* q_in;
    const float* s_in;
    signed char* q_out;
    float* s_out;
};

// 16 lanes hold a block, 4 consecutive values each.
template <class S>
__global__ __launch_bounds__(256) void k_checkpoint_pack(CheckpointArgs A) {
    const int lane = threadIdx.x & 63, sub = lane & 15;
    for (long long base = (long long)blockIdx.x * 16; base < A.blocks; base += (long long)gridDim.x * 16) {
        const long long item = base + (threadIdx.x >> 4);
        const bool live = item < A.blocks;
        const long long row = live ? item / A.nb : 0;
        const int at = live ? (int)(item - row * A.nb) * CKPT_BLOCK + 4 * sub : 0;
        const S* x = (const S*)A.in + row * A.ld;
        double v[4], m = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = (live && at + i < A.n) ? widen(x[at + i]) : 0.0;
            m = ckpt_max(m, ckpt_magnitude(v[i]));
        }
        m = ckpt_max(m, xlane<1>(m, lane));
        m = ckpt_max(m, xlane<2>(m, lane));
        m = ckpt_max(m, xlane<4>(m, lane));
        m = ckpt_max(m, xlane<8>(m, lane));
        const float scale = ckpt_scale(m);
        if (!live) continue;
        signed char* q = A.q_out + row * A.n + at;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (at + i < A.n) q[i] = (signed char)ckpt_quantise(v[i], scale);
        }
        if (sub == 0) A.s_out[item] = scale;
    }
}

template <class S>
__global__ __launch_bounds__(256) void k_checkpoint_unpack(CheckpointArgs A) {
    const int sub = threadIdx.x & 15;
    for (long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4); item < A.blocks; item += (long long)gridDim.x * 16) {
        const long long row = item / A.nb;
        const int at = (int)(item - row * A.nb) * CKPT_BLOCK + 4 * sub;
        const double scale = (double)A.s_in[item];
        const signed char* q = A.q_in + row * A.n + at;
        S* x = (S*)A.out + row * A.ld + at;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (at + i < A.n) x[i] = narrow<S>((double)q[i] * scale);
        }
    }
}

}  // namespace wn

namespace {

const void* kernel_for(bool pack, int dtype) {
    switch (dtype) {
        case WN_F64: return pack ? (const void*)&wn::k_checkpoint_pack<double> : (const void*)&wn::k_checkpoint_unpack<double>;
        case WN_F32: return pack ? (const void*)&wn::k_checkpoint_pack<float> : (const void*)&wn::k_checkpoint_unpack<float>;
        case WN_F16: return pack ? (const void*)&wn::k_checkpoint_pack<wn::f16_bits> : (const void*)&wn::k_checkpoint_unpack<wn::f16_bits>;
        case WN_BF16: return pack ? (const void*)&wn::k_checkpoint_pack<wn::bf16_bits> : (const void*)&wn::k_checkpoint_unpack<wn::bf16_bits>;
    }
    return nullptr;
}

int run(wn_context* ctx, bool pack, const void* wide, int dtype, int B, int n, long long ld, const void* q, const void* scales,
        wn::CheckpointArgs& A) {
    const size_t es = wn::element_bytes(dtype);
    if (!es) return wn::fail(ctx, WN_ERR_ARG, "unknown element type " + std::to_string(dtype));
    if (B < 0 || n < 0) return wn::fail(ctx, WN_ERR_ARG, "bad counts");
    if (B == 0 || n == 0) return WN_OK;
    if (ld < n && B > 1) return wn::fail(ctx, WN_ERR_ARG, "rows of " + std::to_string(n) + " values lie " + std::to_string(ld) + " apart");
    if (!wide || !q || !scales) return wn::fail(ctx, WN_ERR_ARG, "null pointer");
    if (!wn::aligned_to(wide, es) || !wn::aligned_to(scales, 4)) return wn::fail(ctx, WN_ERR_ARG, "misaligned pointer");
    if (ld > (1LL << 40)) return wn::fail(ctx, WN_ERR_UNSUPPORTED, "rows too far apart");
    A.n = n;
    A.nb = (n + wn::CKPT_BLOCK - 1) / wn::CKPT_BLOCK;
    A.blocks = (long long)B * A.nb;
    A.ld = ld;
    const long long grid = std::min<long long>((A.blocks + 15) / 16, (long long)ctx->numCU * 64);
    return wn::launch_kernel(ctx, kernel_for(pack, dtype), (unsigned)grid, 256, 0, A);
}

}  // namespace

extern "C" {

int wn_checkpoint_pack(wn_context* ctx, const void* X_dev, int dtype, int B, int n, long long row_stride, signed char* q_dev,
                       float* scale_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::CheckpointArgs A = {};
        A.in = X_dev; A.q_out = q_dev; A.s_out = scale_dev;
        return run(ctx, true, X_dev, dtype, B, n, row_stride, q_dev, scale_dev, A);
    });
}

int wn_checkpoint_unpack(wn_context* ctx, const signed char* q_dev, const float* scale_dev, int dtype, int B, int n,
                         long long row_stride, void* X_dev) {
    return wn::entry(ctx, [&]() -> int {
        wn::CheckpointArgs A = {};
        A.out = X_dev; A.q_in = q_dev; A.s_in = scale_dev;
        return run(ctx, false, X_dev, dtype, B, n, row_stride, q_dev, scale_dev, A);
    });
}

}  // extern "C"
