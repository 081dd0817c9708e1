// 8-bit checkpoints of activations on their own: wn_checkpoint_pack, wn_checkpoint_unpack.
#include <algorithm>

#include "wn_bank.h"

namespace wn {

struct CheckpointArgs {
    unsigned blocks;        // rows * nb, below 2^31
    int n;
    unsigned nb;
    long long ld;           // elements between rows of the wide side
    const void* in;
    void* out;
    const signed char* q_in;
    const float* s_in;
    signed char* q_out;
    float* s_out;
};

// 16 lanes hold a block, 4 consecutive values each, moved as one piece where the row has them all (the hardware takes any
// alignment).  Blocks are numbered row by row; a workgroup goes through 16 at a time.  32-bit arithmetic finds a block's row:
// the number of blocks is below 2^31 or the launch is cut (run, below).
template <class S>
__global__ __launch_bounds__(256) void k_checkpoint_pack(CheckpointArgs A) {
    const int lane = threadIdx.x & 63, sub = lane & 15;
    for (unsigned base = blockIdx.x * 16; base < A.blocks; base += gridDim.x * 16) {
        const unsigned item = base + (threadIdx.x >> 4);
        const bool live = item < A.blocks;
        const unsigned row = live ? item / A.nb : 0;
        const int at = live ? (int)(item - row * A.nb) * CKPT_BLOCK + 4 * sub : 0, left = live ? A.n - at : 0;
        const S* x = (const S*)A.in + (long long)row * A.ld + at;
        S raw[4] = {};
        if (left >= 4) {
            __builtin_memcpy(raw, x, sizeof(raw));
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++) {
                if (i < left) raw[i] = x[i];
            }
        }
        double v[4], m = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = widen(raw[i]);
            m = ckpt_max(m, ckpt_magnitude(v[i]));
        }
        m = ckpt_max(m, xlane<1>(m, lane));
        m = ckpt_max(m, xlane<2>(m, lane));
        m = ckpt_max(m, xlane<4>(m, lane));
        m = ckpt_max(m, xlane<8>(m, lane));
        const float scale = ckpt_scale(m);
        int b[4];
        ckpt_quantise4(b, v, scale);
        signed char* q = A.q_out + (size_t)row * A.n + at;
        if (left >= 4) {
            const unsigned word = (b[0] & 0xFF) | (b[1] & 0xFF) << 8 | (b[2] & 0xFF) << 16 | (unsigned)b[3] << 24;
            __builtin_memcpy(q, &word, 4);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++) {
                if (i < left) q[i] = (signed char)b[i];
            }
        }
        if (live && sub == 0) A.s_out[item] = scale;
    }
}

template <class S>
__global__ __launch_bounds__(256) void k_checkpoint_unpack(CheckpointArgs A) {
    const int sub = threadIdx.x & 15;
    for (unsigned item = blockIdx.x * 16 + (threadIdx.x >> 4); item < A.blocks; item += gridDim.x * 16) {
        const unsigned row = item / A.nb;
        const int at = (int)(item - row * A.nb) * CKPT_BLOCK + 4 * sub, left = A.n - at;
        const double scale = (double)A.s_in[item];
        const signed char* q = A.q_in + (size_t)row * A.n + at;
        S* x = (S*)A.out + (long long)row * A.ld + at;
        if (left >= 4) {
            signed char b[4];
            __builtin_memcpy(b, q, 4);
            S v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = narrow<S>((double)b[i] * scale);
            __builtin_memcpy(x, v, sizeof(v));
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++) {
                if (i < left) x[i] = narrow<S>((double)q[i] * scale);
            }
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
    A.nb = ((unsigned)n + wn::CKPT_BLOCK - 1) / wn::CKPT_BLOCK;
    const wn::Memory values = {"X", wide, n * es, (unsigned long long)B, ld * es}, whole = {"q", q, (unsigned long long)B * n},
                     parts = {"scale", scales, (unsigned long long)B * A.nb * 4};
    const int rc = pack ? wn::refuse_overlaps(ctx, {whole, parts}, {values}) : wn::refuse_overlaps(ctx, {values}, {whole, parts});
    if (rc) return rc;
    A.ld = ld;
    const int rows = (int)std::min<long long>(B, (1LL << 31) / A.nb - 1);   // of a launch; a row has at most 2^25 blocks
    for (int first = 0; first < B; first += rows) {
        A.blocks = (unsigned)std::min(rows, B - first) * A.nb;
        const unsigned grid = std::min<unsigned>((A.blocks + 15) / 16, (unsigned)ctx->numCU * 32);
        const int rc = wn::launch_kernel(ctx, kernel_for(pack, dtype), grid, 256, 0, A);
        if (rc) return rc;
        const size_t wide = (size_t)rows * ld * es, narrow = (size_t)rows * n, scale = (size_t)rows * A.nb;
        if (pack) { A.in = (const char*)A.in + wide; A.q_out += narrow; A.s_out += scale; }
        else { A.out = (char*)A.out + wide; A.q_in += narrow; A.s_in += scale; }
        if (first > B - rows) break;                        // (first + rows may pass the largest int)
    }
    return WN_OK;
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
