// Instantiates the routed transforms for one compiled tap count (-DWN_NP=2|4|8|16|32) and exports their addresses:
// kind 0 forward, 1 backward; size class as in wn_fused_np.hip.  wn_kernel_bank64_np<taps>: the kernels of 64x64 examples, kind
// 0 forward, 1 backward from the examples, 2 backward from a checkpoint; wn_kernel_bank_line_np<taps>: those of signals of
// 64 M samples, M = 2, 4, 8, 16.
#include "wn_bank_lines.h"

#ifndef WN_NP
#error "compile with -DWN_NP=<taps>"
#endif

#define WN_CAT2(a, b) a##b
#define WN_CAT(a, b) WN_CAT2(a, b)
#define WN_KERNELS(T, Q) return kind ? (const void*)&wn::k_bank_backward<WN_NP, T, Q> : (const void*)&wn::k_bank_forward<WN_NP, T, Q>

extern "C" const void* WN_CAT(wn_kernel_bank_np, WN_NP)(int kind, int sc) {
    switch (sc) {
        case 0: WN_KERNELS(64, 1);
        case 1: WN_KERNELS(64, 3);
        case 2: WN_KERNELS(64, 4);
        case 3: WN_KERNELS(256, 3);
        case 4: WN_KERNELS(512, 3);
    }
    return nullptr;
}

extern "C" const void* WN_CAT(wn_kernel_bank64_np, WN_NP)(int kind) {
    switch (kind) {
        case 0: return (const void*)&wn::k_bank_forward64<WN_NP>;
        case 1: return (const void*)&wn::k_bank_backward64<WN_NP, false>;
        case 2: return (const void*)&wn::k_bank_backward64<WN_NP, true>;
    }
    return nullptr;
}

template <int M>
static const void* line_kernel(int kind) {
    switch (kind) {
        case 0: return (const void*)&wn::k_bank_forward_line<WN_NP, M>;
        case 1: return (const void*)&wn::k_bank_backward_line<WN_NP, M, false>;
        case 2: return (const void*)&wn::k_bank_backward_line<WN_NP, M, true>;
    }
    return nullptr;
}
extern "C" const void* WN_CAT(wn_kernel_bank_line_np, WN_NP)(int kind, int M) {
    switch (M) {
        case 2: return line_kernel<2>(kind);
        case 4: return line_kernel<4>(kind);
        case 8: return line_kernel<8>(kind);
        case 16: return line_kernel<16>(kind);
    }
    return nullptr;
}
