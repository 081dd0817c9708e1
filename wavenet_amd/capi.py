"""ctypes binding of the C ABI declared in include/wavenet_hip.h.

Device buffers are passed as integer addresses (e.g. torch.Tensor.data_ptr()); torch is only
used by callers for device memory and streams, never for the arithmetic.
"""
import ctypes as C
import functools
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))

WN_OK = 0
WN_ERR_ARG, WN_ERR_BAD_SHAPE, WN_ERR_BAD_FILTER, WN_ERR_UNSUPPORTED = 1, 2, 3, 4
WN_ERR_HIP, WN_ERR_COMM, WN_ERR_NONFINITE, WN_ERR_STATE = 5, 6, 7, 8
WN_MAX_TAPS = 32
WN_MAX_FUSED = 4096
WN_F64, WN_F32, WN_F16, WN_BF16 = 0, 1, 2, 3
WN_SCORE_SOFTMAX, WN_SCORE_SIGMOID = 0, 1
WN_MAX_EXPERTS, WN_MAX_TOPK, WN_MAX_GROUPS = 1024, 16, 64

_dp = C.POINTER(C.c_double)
_vp = C.c_void_p


class Routing(C.Structure):
    """wn_routing of include/wavenet_hip.h."""
    _fields_ = [("score", C.c_int), ("k", C.c_int), ("groups", C.c_int), ("groups_kept", C.c_int), ("renormalise", C.c_int),
                ("scale", C.c_double), ("score_scale", C.c_double)]


# name -> (restype, argtypes); every symbol include/wavenet_hip.h declares
SIGNATURES = {
    "wn_create": (C.c_int, [C.c_int, C.POINTER(_vp)]),
    "wn_destroy": (C.c_int, [_vp]),
    "wn_set_stream": (C.c_int, [_vp, _vp]),
    "wn_synchronize": (C.c_int, [_vp]),
    "wn_last_error": (C.c_char_p, [_vp]),
    "wn_status_string": (C.c_char_p, [C.c_int]),
    "wn_malloc": (C.c_int, [_vp, C.POINTER(_vp), C.c_size_t]),
    "wn_free": (C.c_int, [_vp, _vp]),
    "wn_memcpy_h2d": (C.c_int, [_vp, _vp, _vp, C.c_size_t]),
    "wn_memcpy_d2h": (C.c_int, [_vp, _vp, _vp, C.c_size_t]),
    "wn_set_filter": (C.c_int, [_vp, _dp, C.c_int]),
    "wn_get_filter": (C.c_int, [_vp, _dp, C.POINTER(C.c_int)]),
    "wn_set_momentum": (C.c_int, [_vp, _dp, C.c_int]),
    "wn_get_momentum": (C.c_int, [_vp, _dp, C.POINTER(C.c_int)]),
    "wn_lowpass_operator": (C.c_int, [_dp, C.c_int, C.c_uint, _dp]),
    "wn_highpass_operator": (C.c_int, [_dp, C.c_int, C.c_uint, _dp]),
    "wn_forward": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp, _vp]),
    "wn_inverse": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "wn_backprop": (C.c_int, [_vp, _vp, _vp, _vp, _vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp]),
    "wn_sparse_term": (C.c_int, [_vp, _vp, C.c_int, C.c_int, _vp]),
    "wn_sparse_term_deriv": (C.c_int, [_vp, _vp, C.c_int, C.c_int, _vp, _vp]),
    "wn_reg_term": (C.c_int, [_dp, C.c_int, C.c_int, _dp]),
    "wn_reg_term_deriv": (C.c_int, [_dp, C.c_int, C.c_int, _dp]),
    "wn_sparse_cost_grid": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _dp, C.c_int, C.c_int, _vp]),
    "wn_route": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, C.c_longlong, C.c_longlong, C.POINTER(Routing), _vp, _vp, _vp, _vp]),
    "wn_route_backward": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, C.c_longlong, C.c_longlong, C.POINTER(Routing), _vp, _vp, _vp]),
    "wn_checkpoint_pack": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, C.c_longlong, _vp, _vp]),
    "wn_checkpoint_unpack": (C.c_int, [_vp, _vp, _vp, C.c_int, C.c_int, C.c_int, C.c_longlong, _vp]),
    "wn_forward_routed": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp, C.c_int, C.c_int, _vp, _vp, C.c_int, _vp, _vp, _vp]),
    "wn_backprop_routed": (C.c_int, [_vp, _vp, _vp, _vp, _vp, C.c_int, C.c_int, C.c_int, _vp, C.c_int, C.c_int, _vp, _vp, C.c_int,
                                     _vp, _vp, _vp, _vp]),
    "wn_generate_uniform": (C.c_int, [_vp, C.c_ulonglong, C.c_longlong, C.c_int, C.c_int, C.c_int, _vp]),
    "wn_generate_needle": (C.c_int, [_vp, C.c_ulonglong, C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_double, _vp]),
    "wn_generate_calorimeter": (C.c_int, [_vp, C.c_ulonglong, C.c_longlong, C.c_int, C.c_int, C.c_int,
                                          C.POINTER(C.c_int), _dp, C.c_int, C.c_int, _vp]),
    "wn_get_device": (C.c_int, [_vp, C.POINTER(C.c_int)]),
    "wn_generate_gaussian": (C.c_int, [_vp, C.c_ulonglong, C.c_longlong, C.c_int, C.c_int, C.c_int, _dp, _vp]),
    "wn_train_batch": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp]),
    "wn_train_batch_static": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "wn_sums": (C.c_int, [_vp, C.POINTER(_vp), C.POINTER(C.c_int)]),
    "wn_get_sums": (C.c_int, [_vp, _dp, C.POINTER(C.c_int)]),
    "wn_set_sums_buffer": (C.c_int, [_vp, _vp]),
    "wn_profile_begin": (C.c_int, [_vp, C.c_int]),
    "wn_profile_collect": (C.c_int, [_vp, C.POINTER(C.c_float), C.c_int, C.POINTER(C.c_int)]),
    "wn_apply_update": (C.c_int, [_vp, C.c_double, C.c_double, C.c_double, C.c_double, C.c_int]),
    "wn_train_step": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, C.c_double, C.c_double, C.c_double, C.c_double, C.c_int]),
    "wn_num_updates": (C.c_int, [_vp, C.POINTER(C.c_int)]),
    "wn_get_logs": (C.c_int, [_vp, C.c_int, C.c_int, _dp, _dp]),
    "wn_get_updates": (C.c_int, [_vp, C.c_int, C.c_int, C.POINTER(C.c_int), _dp, _dp, _dp]),
    "wn_clear_logs": (C.c_int, [_vp]),
    "wn_comm_unique_id": (C.c_int, [_vp]),
    "wn_comm_init": (C.c_int, [_vp, _vp, C.c_int, C.c_int]),
    "wn_comm_destroy": (C.c_int, [_vp]),
    "wn_allreduce_sums": (C.c_int, [_vp]),
    "wn_comm_init_all": (C.c_int, [C.POINTER(_vp), C.c_int]),
    "wn_allreduce_sums_all": (C.c_int, [C.POINTER(_vp), C.c_int]),
}


class WavenetError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"[wn status {status}] {message}")
        self.status = status


def lib_path():
    """The library next to this package, unless WAVENET_HIP_LIBRARY names another build of it."""
    return os.environ.get("WAVENET_HIP_LIBRARY") or os.path.join(_HERE, "lib", "libwavenet_hip.so")


_lib = None


def load_library():
    """Load libwavenet_hip.so and type every entry point.  Raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    try:
        # torch bundles its own libamdhip64 under the same soname as /opt/rocm's; whichever is
        # mapped first serves the whole process, and a process that ends up with both cannot
        # see the GPU from the second.  Callers use torch for device memory, so let it go first.
        import torch  # noqa: F401
    except ImportError:
        pass
    path = lib_path()
    if not os.path.exists(path):
        raise ImportError(
            f"{path} not found: build it with `make -C wavenet_amd/csrc` (or __graft_entry__.build()). "
            "There is no CPU fallback.")
    lib = C.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _addr(x):
    """Device address of a torch tensor, or an int/None passed through."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _hd(a):
    a = np.ascontiguousarray(a, dtype=np.float64)
    return a, a.ctypes.data_as(_dp)


_TYPE_CODES = {"float64": WN_F64, "float32": WN_F32, "float16": WN_F16, "bfloat16": WN_BF16}


_type_names = {}


def _type_name(x):
    name = _type_names.get(x.dtype)
    if name is None:
        name = _type_names[x.dtype] = str(x.dtype).rsplit(".", 1)[-1]
    return name


def _dtype_code(x, dtype):
    """Element type code: of a tensor, or of an address by the code or name given with it (default float64)."""
    if x is not None and not isinstance(x, int):
        name = _type_name(x)
        if name not in _TYPE_CODES:
            raise ValueError(f"element type {name} is not one of {sorted(_TYPE_CODES)}")
        if dtype is not None and _TYPE_CODES[name] != _TYPE_CODES.get(dtype, dtype):
            raise ValueError(f"element type is {name}, not {dtype}")
        return _TYPE_CODES[name]
    if dtype is None:
        return WN_F64
    return _TYPE_CODES.get(dtype, dtype)


def _strided(x, rows, row_stride, cols, col_stride):
    """Whether a tensor that is not contiguous holds value (r, c) where the strides say: both have to be strides of its
    dimensions, or of neighbouring dimensions that make one."""
    if x.dim() == 2 and x.stride() == (row_stride, col_stride):
        return x.shape[0] >= rows and x.shape[1] >= cols
    dims = [(n, s) for n, s in zip(x.shape, x.stride()) if n > 1]
    runs, n, s = [], 0, 0
    for m, t in reversed(dims):
        n, s = (n * m, s) if n and t == n * s else (m, t)
        runs.append((n, s))
    return all(count <= 1 or any(s == stride and n >= count for n, s in dims + runs)
               for count, stride in ((rows, row_stride), (cols, col_stride)))


def _out_of_step(x, count, widths):
    """Whether a tensor of rows, with more elements than the `count` of the table it is taken for, has rows of another width."""
    return x.numel() != count and x.dim() > 1 and x.shape[0] > 1 and x.numel() // x.shape[0] not in widths


# --- host-only entry points ----------------------------------------------------------------------

def reg_term(a, wavelet=True):
    lib = load_library()
    a, pa = _hd(a)
    out = C.c_double(0)
    st = lib.wn_reg_term(pa, len(a), int(wavelet), C.byref(out))
    if st:
        raise WavenetError(st, lib.wn_status_string(st).decode())
    return out.value


def reg_term_deriv(a, wavelet=True):
    lib = load_library()
    a, pa = _hd(a)
    g = np.empty_like(a)
    st = lib.wn_reg_term_deriv(pa, len(a), int(wavelet), g.ctypes.data_as(_dp))
    if st:
        raise WavenetError(st, lib.wn_status_string(st).decode())
    return g


def dense_operator(a, size, highpass=False):
    """LowpassOperator(a, size) / HighpassOperator(a, size) as a 2^size x 2^(size+1) numpy matrix."""
    lib = load_library()
    a, pa = _hd(a)
    nr, nc = 1 << size, 2 << size
    M = np.empty(nr * nc)
    fn = lib.wn_highpass_operator if highpass else lib.wn_lowpass_operator
    st = fn(pa, len(a), size, M.ctypes.data_as(_dp))
    if st:
        raise WavenetError(st, lib.wn_status_string(st).decode())
    return M.reshape((nr, nc), order="F").copy()


class Context:
    """One context per (process, device): filter state, stream, scratch, communicator."""

    def __init__(self, device=0, stream=None):
        self.lib = load_library()
        h = _vp()
        st = self.lib.wn_create(int(device), C.byref(h))
        if st:
            raise WavenetError(st, self.lib.wn_last_error(None).decode())
        self._h = h
        self.device = device
        if stream is not None:
            self.set_stream(stream)

    def close(self):
        if getattr(self, "_h", None):
            self.lib.wn_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st):
        if st:
            raise WavenetError(st, self.lib.wn_last_error(self._h).decode())

    def set_stream(self, stream):
        """stream: integer hipStream_t (torch.cuda.current_stream().cuda_stream) or None."""
        self._check(self.lib.wn_set_stream(self._h, stream))

    def synchronize(self):
        self._check(self.lib.wn_synchronize(self._h))

    # filter ----------------------------------------------------------------------------------
    def set_filter(self, a):
        a, pa = _hd(a)
        self._check(self.lib.wn_set_filter(self._h, pa, len(a)))

    def filter(self):
        n = C.c_int(0)
        self._check(self.lib.wn_get_filter(self._h, None, C.byref(n)))
        a = np.empty(n.value)
        self._check(self.lib.wn_get_filter(self._h, a.ctypes.data_as(_dp), C.byref(n)))
        return a

    def set_momentum(self, p):
        p, pp = _hd(p)
        self._check(self.lib.wn_set_momentum(self._h, pp, len(p)))

    def momentum(self):
        n = C.c_int(0)
        self._check(self.lib.wn_get_momentum(self._h, None, C.byref(n)))
        p = np.empty(n.value)
        self._check(self.lib.wn_get_momentum(self._h, p.ctypes.data_as(_dp), C.byref(n)))
        return p

    # transforms (device buffers: torch tensors or addresses) ----------------------------------
    def forward(self, X, B, R, Cc, Y=None, Prow=None, Y1=None, Pcol=None):
        self._check(self.lib.wn_forward(self._h, _addr(X), B, R, Cc, _addr(Y), _addr(Prow), _addr(Y1), _addr(Pcol)))

    def inverse(self, Y, B, R, Cc, X):
        self._check(self.lib.wn_inverse(self._h, _addr(Y), B, R, Cc, _addr(X)))

    def backprop(self, Delta, X, Prow, Y1, Pcol, B, R, Cc, grad, din=None):
        self._check(self.lib.wn_backprop(self._h, _addr(Delta), _addr(X), _addr(Prow), _addr(Y1), _addr(Pcol),
                                         B, R, Cc, _addr(grad), _addr(din)))

    def sparse_term(self, Y, B, n, S):
        self._check(self.lib.wn_sparse_term(self._h, _addr(Y), B, n, _addr(S)))

    def sparse_term_deriv(self, Y, B, n, Delta, S=None):
        self._check(self.lib.wn_sparse_term_deriv(self._h, _addr(Y), B, n, _addr(Delta), _addr(S)))

    def sparse_cost_grid(self, X, B, R, Cc, filters, S):
        """S[f * B + e] = sparse term of example e under filter f; filters: (F, N) numpy array."""
        f = np.ascontiguousarray(filters, dtype=np.float64)
        assert f.ndim == 2
        self._check(self.lib.wn_sparse_cost_grid(self._h, _addr(X), B, R, Cc, f.ctypes.data_as(_dp), f.shape[0],
                                                 f.shape[1], _addr(S)))

    # routed filter bank ---------------------------------------------------------------------------
    def _buffer(self, name, x, count, wanted=None, strides=None, widths=None):
        """Address of an argument.  A tensor has to lie on the context's GPU and hold `count` elements of the type, densely,
        or with `strides` (rows, row_stride, cols, col_stride) reach the last of them, with these strides unless it is
        contiguous; an address is taken as it is.  widths: what the rows of a tensor with room to spare may be wide."""
        if x is None or isinstance(x, int):
            return x
        if x.get_device() != self.device:                      # (-1 off the GPU)
            raise ValueError(f"{name} is on {x.device}, the context on GPU {self.device}")
        if wanted is not None and _type_name(x) != wanted:
            raise ValueError(f"{name} holds {_type_name(x)}, not {wanted}")
        if strides is None:
            if not x.is_contiguous():
                raise ValueError(f"{name} is not contiguous")
            held = x.numel()
            if held < count:
                raise ValueError(f"{name} holds {held} elements, {count} are needed")
            if widths is not None and held != count and _out_of_step(x, count, widths):
                raise ValueError(f"{name} is {held // x.shape[0]} wide, not {widths[0]}")
            return x.data_ptr()
        rows, row_stride, cols, col_stride = strides
        span = (rows - 1) * row_stride + (cols - 1) * col_stride + 1 if rows > 0 and cols > 0 else 0
        dense = x.is_contiguous()
        if not dense or x.numel() < span:
            if not dense and span > 0 and not _strided(x, *strides):
                raise ValueError(f"{name} has strides {tuple(x.stride())}, not {row_stride} between rows and {col_stride} in them")
            held = x.untyped_storage().nbytes() // x.element_size() - x.storage_offset()
            if held < span:
                raise ValueError(f"{name} ends {held} elements after its start, {span} are needed")
        return x.data_ptr()

    @staticmethod
    @functools.lru_cache(maxsize=64)
    def _routing(k, score, groups, groups_kept, renormalise, scale, score_scale):
        code = {"softmax": WN_SCORE_SOFTMAX, "sigmoid": WN_SCORE_SIGMOID}.get(score, score)
        if not isinstance(code, int):
            raise ValueError(f"score is {score!r}, not 'softmax' or 'sigmoid'")
        return Routing(code, int(k), int(groups), int(groups if groups_kept is None else groups_kept), int(bool(renormalise)),
                       float(scale), float(score_scale))

    def route(self, scores, T, F, idx, w, k=1, score="softmax", bias=None, groups=1, groups_kept=None, renormalise=True,
              scale=1.0, score_scale=1.0, counts=None, row_stride=None, col_stride=1, dtype=None):
        """wn_route: the k filters of each of T rows of F scores, and their weights.

        scores: tensor (its element type is used) or address (dtype: "float64", "float32", "float16" or "bfloat16");
        score (t, f) lies t * row_stride + f * col_stride elements from the start (default: dense rows).
        idx: int32 [T][k], w: float64 [T][k], bias: float64 [F], counts: int32 [F]."""
        rs = F * col_stride if row_stride is None else row_stride
        at = (T, rs, F, col_stride)
        r = self._routing(k, score, groups, groups_kept, renormalise, scale, score_scale)
        self._check(self.lib.wn_route(
            self._h, self._buffer("scores", scores, 0, strides=at), _dtype_code(scores, dtype), T, F, rs, col_stride, C.byref(r),
            self._buffer("bias", bias, F, "float64"), self._buffer("idx", idx, T * k, "int32", None, (k, 1)),
            self._buffer("w", w, T * k, "float64", None, (k, 1)), self._buffer("counts", counts, F, "int32")))

    def route_backward(self, scores, T, F, idx, dw, dscores, k=1, score="softmax", groups=1, groups_kept=None, renormalise=True,
                       scale=1.0, score_scale=1.0, row_stride=None, col_stride=1, dtype=None):
        """wn_route_backward: gradient dw of the weights -> gradient of the scores, laid out as the scores."""
        rs = F * col_stride if row_stride is None else row_stride
        at = (T, rs, F, col_stride)
        r = self._routing(k, score, groups, groups_kept, renormalise, scale, score_scale)
        code = _dtype_code(scores, dtype)
        if _dtype_code(dscores, dtype if isinstance(dscores, int) else None) != code and dscores is not None and not isinstance(dscores, int):
            raise ValueError("dscores and scores differ in type")
        self._check(self.lib.wn_route_backward(
            self._h, self._buffer("scores", scores, 0, strides=at), code, T, F, rs, col_stride, C.byref(r),
            self._buffer("idx", idx, T * k, "int32", None, (k, 1)), self._buffer("dw", dw, T * k, "float64", None, (k, 1)),
            self._buffer("dscores", dscores, 0, strides=at)))

    def checkpoint_pack(self, X, B, n, q, scales, row_stride=None, dtype=None):
        """wn_checkpoint_pack: B rows of n values as int8 q[B][n] and float32 scales[B][ceil(n / 64)]."""
        rs = n if row_stride is None else row_stride
        self._check(self.lib.wn_checkpoint_pack(
            self._h, self._buffer("X", X, 0, strides=(B, rs, n, 1)), _dtype_code(X, dtype), B, n, rs,
            self._buffer("q", q, B * n, "int8"), self._buffer("scales", scales, B * -(-n // 64), "float32")))

    def checkpoint_unpack(self, q, scales, B, n, X, row_stride=None, dtype=None):
        """wn_checkpoint_unpack: the values a checkpoint stands for, in the type of X."""
        rs = n if row_stride is None else row_stride
        self._check(self.lib.wn_checkpoint_unpack(
            self._h, self._buffer("q", q, B * n, "int8"), self._buffer("scales", scales, B * -(-n // 64), "float32"),
            _dtype_code(X, dtype), B, n, rs, self._buffer("X", X, 0, strides=(B, rs, n, 1))))

    def _bank(self, filters, F, N):
        """(filters, F, N): a tensor [F][N] says both numbers; None is the context's own filter."""
        if filters is None and N is None:
            n = C.c_int(0)
            self._check(self.lib.wn_get_filter(self._h, None, C.byref(n)))
            return None, 1 if F is None else F, n.value
        if filters is not None and not isinstance(filters, int) and filters.dim() == 2:
            F = filters.shape[0] if F is None else F
            N = filters.shape[1] if N is None else N
        if F is None or N is None:
            raise ValueError("the number of filters and of taps is not known: pass a tensor [F][N], or F and N")
        return self._buffer("filters", filters, F * N, "float64", None, (N,)), F, N

    @staticmethod
    def _entries(idx, w, k):
        for x in (idx, w):
            if k is None and x is not None and not isinstance(x, int) and x.dim() == 2:
                k = x.shape[1]
        return 1 if k is None else k

    def forward_routed(self, X, B, R, Cc, filters, idx, w, Y, k=None, q=None, scales=None, F=None, N=None):
        """wn_forward_routed: Y[e] = sum_j w[e][j] forward(X[e] under filters[idx[e][j]]).

        filters: float64 [F][N] (None: the context's filter); idx: int32 [B][k] (None: filter 0); w: float64 [B][k]
        (None: ones); q, scales: where to keep the checkpoint of X, if wanted."""
        filters, F, N = self._bank(filters, F, N)
        k, n = self._entries(idx, w, k), R * Cc
        self._check(self.lib.wn_forward_routed(
            self._h, self._buffer("X", X, B * n, "float64"), B, R, Cc, filters, F, N, self._buffer("idx", idx, B * k, "int32", None, (k, 1)),
            self._buffer("w", w, B * k, "float64", None, (k, 1)), k, self._buffer("Y", Y, B * n, "float64"), self._buffer("q", q, B * n, "int8"),
            self._buffer("scales", scales, B * -(-n // 64), "float32")))

    def backprop_routed(self, Delta, B, R, Cc, filters, idx, w, grad, X=None, q=None, scales=None, dfilters=None, dw=None, dX=None,
                        k=None, F=None, N=None):
        """wn_backprop_routed: errors Delta on Y -> grad[B][k][N], dfilters[F][N], dw[B][k], dX[B][n], at the examples X or at
        the checkpoint (q, scales) that forward_routed or checkpoint_pack kept."""
        filters, F, N = self._bank(filters, F, N)
        k, n = self._entries(idx, w, k), R * Cc
        self._check(self.lib.wn_backprop_routed(
            self._h, self._buffer("Delta", Delta, B * n, "float64"), self._buffer("X", X, B * n, "float64"),
            self._buffer("q", q, B * n, "int8"), self._buffer("scales", scales, B * -(-n // 64), "float32"), B, R, Cc, filters, F, N,
            self._buffer("idx", idx, B * k, "int32", None, (k, 1)), self._buffer("w", w, B * k, "float64", None, (k, 1)), k,
            self._buffer("grad", grad, B * k * N, "float64", None, (k * N, N)), self._buffer("dfilters", dfilters, F * N, "float64", None, (N,)),
            self._buffer("dw", dw, B * k, "float64", None, (k, 1)), self._buffer("dX", dX, B * n, "float64")))

    # generators ---------------------------------------------------------------------------------
    def generate_uniform(self, X, B, R, Cc, seed=1, first=0):
        self._check(self.lib.wn_generate_uniform(self._h, seed, first, B, R, Cc, _addr(X)))

    def generate_needle(self, X, B, R, Cc, seed=1, first=0, threshold=0.995):
        self._check(self.lib.wn_generate_needle(self._h, seed, first, B, R, Cc, threshold, _addr(X)))

    def generate_calorimeter(self, X, B, R, Cc, seed=1, first=0, mean_deposits=None, jets=2, jet_deposits=30):
        """Same images as generators.calorimeter(...)[first:first + B], written in device layout."""
        from . import generators as G
        if mean_deposits is None:
            mean_deposits = max(1.0, 200.0 * (R * Cc) / 4096.0)
        ptab = np.ascontiguousarray(G._poisson_table(float(mean_deposits)), dtype=np.int32)
        etab = np.ascontiguousarray(G._EXP_TABLE, dtype=np.float64)
        self._check(self.lib.wn_generate_calorimeter(self._h, seed, first, B, R, Cc, ptab.ctypes.data_as(C.POINTER(C.c_int)),
                                                     etab.ctypes.data_as(_dp), jets, jet_deposits, _addr(X)))

    def generate_gaussian(self, X, B, R, Cc, seed=1, first=0):
        """wn_generate_gaussian: the sequence of generators.gaussian, written on the device."""
        from .generators import GAUSS_EXP_TABLE
        tab = np.ascontiguousarray(GAUSS_EXP_TABLE, dtype=np.float64)
        self._check(self.lib.wn_generate_gaussian(self._h, seed, first, B, R, Cc, tab.ctypes.data_as(_dp), _addr(X)))

    # training -----------------------------------------------------------------------------------
    def train_batch(self, X, B, R, Cc, grad=None, S=None):
        self._check(self.lib.wn_train_batch(self._h, _addr(X), B, R, Cc, _addr(grad), _addr(S)))

    def train_batch_static(self, X, B, R, Cc, sums):
        """wn_train_batch_static: no allocation; sums: device tensor/address of N + 2 doubles."""
        self._check(self.lib.wn_train_batch_static(self._h, _addr(X), B, R, Cc, _addr(sums)))

    def sums_ptr(self):
        p = _vp()
        n = C.c_int(0)
        self._check(self.lib.wn_sums(self._h, C.byref(p), C.byref(n)))
        return p.value, n.value

    def sums(self):
        n = C.c_int(0)
        self._check(self.lib.wn_get_sums(self._h, None, C.byref(n)))
        s = np.empty(n.value)
        self._check(self.lib.wn_get_sums(self._h, s.ctypes.data_as(_dp), C.byref(n)))
        return s

    def set_sums_buffer(self, buf):
        """buf: device tensor/address of >= WN_MAX_TAPS + 2 doubles, or None for the context's own."""
        self._check(self.lib.wn_set_sums_buffer(self._h, _addr(buf)))

    def profile_begin(self, max_records):
        self._check(self.lib.wn_profile_begin(self._h, int(max_records)))

    def profile_collect(self, capacity=4096):
        ms = (C.c_float * capacity)()
        n = C.c_int(0)
        self._check(self.lib.wn_profile_collect(self._h, ms, capacity, C.byref(n)))
        return np.array(ms[:n.value], dtype=np.float64)

    def apply_update(self, batch_total, lambda_sum, alpha, inertia_eff=0.0, wavelet=True):
        self._check(self.lib.wn_apply_update(self._h, float(batch_total), float(lambda_sum), float(alpha),
                                             float(inertia_eff), int(wavelet)))

    def train_step(self, X, B, R, Cc, batch_total, lambda_sum, alpha, inertia_eff=0.0, wavelet=True):
        """wn_train_step: train_batch + (all-reduce over the context's communicator) + apply_update, one submission."""
        self._check(self.lib.wn_train_step(self._h, _addr(X), B, R, Cc, float(batch_total), float(lambda_sum),
                                           float(alpha), float(inertia_eff), int(wavelet)))

    def num_updates(self):
        n = C.c_int(0)
        self._check(self.lib.wn_num_updates(self._h, C.byref(n)))
        return n.value

    def logs(self, first=0, count=None):
        if count is None:
            count = self.num_updates() - first
        N = len(self.filter())
        F = np.empty((count, N))
        Cs = np.empty(count)
        self._check(self.lib.wn_get_logs(self._h, first, count, F.ctypes.data_as(_dp), Cs.ctypes.data_as(_dp)))
        return F, Cs

    def updates(self, first=0, max_count=1024):
        """wn_get_updates: (steps, filters[count][N], costs[count], momentum[N], rejected) in one readback."""
        N = len(self.filter())
        F = np.empty((max_count, N))
        Cs = np.empty(max_count)
        P = np.empty(N)
        n = C.c_int(0)
        st = self.lib.wn_get_updates(self._h, first, max_count, C.byref(n), F.ctypes.data_as(_dp), Cs.ctypes.data_as(_dp),
                                     P.ctypes.data_as(_dp))
        if st not in (0, WN_ERR_NONFINITE):
            self._check(st)
        count = max(0, min(max_count, n.value - first))
        return n.value, F[:count], Cs[:count], P, st == WN_ERR_NONFINITE

    def clear_logs(self):
        self._check(self.lib.wn_clear_logs(self._h))

    # communicator ---------------------------------------------------------------------------------
    def comm_unique_id(self):
        buf = (C.c_char * 128)()
        st = self.lib.wn_comm_unique_id(buf)
        if st:
            raise WavenetError(st, self.lib.wn_last_error(None).decode())
        return bytes(buf)

    def comm_init(self, unique_id, nranks, rank):
        buf = (C.c_char * 128).from_buffer_copy(unique_id)
        self._check(self.lib.wn_comm_init(self._h, buf, nranks, rank))

    def allreduce_sums(self):
        self._check(self.lib.wn_allreduce_sums(self._h))
