"""ctypes binding of the C ABI declared in include/fsw.h (libfsw_hip.so).

This is the foreign-function stub a maintainer of the reference would add to call the MI355X path without the
PyTorch extension; tensors are only used as owners of device memory (data_ptr) and of the current stream.
The library is never built from here: a missing libfsw_hip.so is an error, not a reason to fall back.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libfsw_hip.so")

BF16, FP16 = 0, 1
OK = 0
E_NULL, E_DTYPE, E_SHAPE, E_LD, E_ALIGN, E_WORKSPACE, E_LAUNCH, E_DEVICE, E_VARIANT, E_STATIC_LIMIT = range(-1, -11, -1)

# name -> (restype, argtypes); the list the loader test checks against include/fsw.h
_i, _i64, _vp, _sz, _cp = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_char_p
_rows = [_vp, _i64, _i64]  # rows [token][head][channel]: base, token stride, head stride


class KvCache(ctypes.Structure):
    """fsw_kv_cache of include/fsw.h."""
    _fields_ = [("k", _vp), ("v", _vp), ("pages", _i64), ("page_size", _i64), ("page_stride", _i64), ("head_stride", _i64),
                ("token_stride", _i64)]


class KvCache8(ctypes.Structure):
    """fsw_kv_cache8 of include/fsw.h."""
    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("pages", _i64), ("page_size", _i64), ("page_stride", _i64),
                ("head_stride", _i64), ("token_stride", _i64), ("scale_page_stride", _i64), ("scale_head_stride", _i64),
                ("scale_token_stride", _i64)]


_kvp = ctypes.POINTER(KvCache)
_kvp8 = ctypes.POINTER(KvCache8)
_f = ctypes.c_float
PROTOTYPES = {
    "fsw_validate_gateup": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64]),
    "fsw_gateup": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    "fsw_gateup_f32out": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    "fsw_validate_down": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64]),
    "fsw_down_workspace_bytes": (_sz, [_i, _i64, _i64, _i64]),
    "fsw_down": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _sz, _vp]),
    "fsw_mlp_workspace_bytes": (_sz, [_i, _i64, _i64, _i64]),
    "fsw_mlp": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _sz, _vp]),
    "fsw_mlp_static_max_bytes": (_sz, []),
    "fsw_mlp_static": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    "fsw_blocked_bytes": (_sz, [_i64, _i64]),
    "fsw_block_rows": (_i, [_i, _i64, _i64, _vp, _i64, _vp, _vp]),
    "fsw_prepack_w13": (_i, [_i, _i64, _i64, _vp, _i64, _vp, _vp]),
    "fsw_prepack_w2": (_i, [_i, _i64, _i64, _vp, _i64, _vp, _vp]),
    "fsw_gateup_blocked": (_i, [_i, _i64, _i64, _i64, _vp, _vp, _i64, _i, _vp, _i64, _vp]),
    "fsw_gateup_hblocked": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _i, _vp, _vp]),
    "fsw_down_blocked": (_i, [_i, _i64, _i64, _i64, _vp, _vp, _i64, _i, _vp, _i64, _vp]),
    "fsw_gateup_workspace_bytes": (_sz, [_i, _i64, _i64, _i64]),
    "fsw_gateup_ws": (_i, [_i, _i64, _i64, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _sz, _vp]),
    "fsw_validate_kv_append": (_i, [_i] + [_i64] * 5 + _rows * 3 + [_vp, _i64, _vp, _vp] + _rows * 2 + [_kvp]),
    "fsw_kv_append": (_i, [_i] + [_i64] * 5 + [_i] + _rows * 3 + [_vp, _i64, _vp, _vp] + _rows * 2 + [_kvp, _vp]),
    "fsw_validate_attn_decode": (_i, [_i] + [_i64] * 4 + _rows + [_kvp, _vp, _i64, _vp, _i64, ctypes.c_float] + _rows),
    "fsw_attn_decode_workspace_bytes": (_sz, [_i] + [_i64] * 5),
    "fsw_attn_decode": (_i, [_i] + [_i64] * 4 + _rows + [_kvp, _vp, _i64, _vp, _i64, ctypes.c_float] + _rows + [_vp, _sz, _vp]),
    "fsw_validate_attn_prompt": (_i, [_i] + [_i64] * 6 + _rows * 3 + [_vp, _vp, ctypes.c_float] + _rows),
    "fsw_attn_prompt_rows": (_i, [_i] + [_i64] * 5),
    "fsw_attn_prompt": (_i, [_i] + [_i64] * 6 + _rows * 3 + [_vp, _vp, ctypes.c_float] + _rows + [_vp]),
    "fsw_validate_kv_append8": (_i, [_i] + [_i64] * 5 + _rows * 3 + [_vp, _i64, _vp, _vp] + _rows * 3 + [_kvp8]),
    "fsw_kv_append8": (_i, [_i] + [_i64] * 5 + [_i] + _rows * 3 + [_vp, _i64, _vp, _vp] + _rows * 3 + [_kvp8, _vp]),
    "fsw_validate_kv_read": (_i, [_i] + [_i64] * 4 + [_kvp, _vp, _i64, _i64, _vp] + _rows * 2),
    "fsw_validate_kv_read8": (_i, [_i] + [_i64] * 4 + [_kvp8, _vp, _i64, _i64, _vp] + _rows * 2),
    "fsw_kv_read": (_i, [_i] + [_i64] * 4 + [_kvp, _vp, _i64, _i64, _vp] + _rows * 2 + [_vp]),
    "fsw_kv_read8": (_i, [_i] + [_i64] * 4 + [_kvp8, _vp, _i64, _i64, _vp] + _rows * 2 + [_vp]),
    "fsw_validate_attn_decode8": (_i, [_i] + [_i64] * 4 + _rows + [_kvp8, _vp, _i64, _vp, _i64, _f] + _rows),
    "fsw_attn_decode8_workspace_bytes": (_sz, [_i] + [_i64] * 5),
    "fsw_attn_decode8": (_i, [_i] + [_i64] * 4 + _rows + [_kvp8, _vp, _i64, _vp, _i64, _f] + _rows + [_vp, _sz, _vp]),
    "fsw_validate_attn_shared": (_i, [_i] + [_i64] * 4 + _rows + [_kvp, _vp, _i64, _vp, _i64, _vp, _i64, _f] + _rows),
    "fsw_validate_attn_shared8": (_i, [_i] + [_i64] * 4 + _rows + [_kvp8, _vp, _i64, _vp, _i64, _vp, _i64, _f] + _rows),
    "fsw_attn_shared_workspace_bytes": (_sz, [_i] + [_i64] * 6),
    "fsw_attn_shared8_workspace_bytes": (_sz, [_i] + [_i64] * 6),
    "fsw_attn_shared_rows": (_i, [_i] + [_i64] * 6),
    "fsw_attn_shared8_rows": (_i, [_i] + [_i64] * 6),
    "fsw_attn_shared": (_i, [_i] + [_i64] * 4 + _rows + [_kvp, _vp, _i64, _vp, _i64, _vp, _i64, _f] + _rows + [_vp, _sz, _vp]),
    "fsw_attn_shared8": (_i, [_i] + [_i64] * 4 + _rows + [_kvp8, _vp, _i64, _vp, _i64, _vp, _i64, _f] + _rows + [_vp, _sz, _vp]),
    "fsw_validate_add_norm": (_i, [_i, _i64, _i64] + [_vp, _i64] * 3 + [_vp, _vp, _f, _f] + [_vp, _i64] * 2),
    "fsw_add_norm": (_i, [_i, _i64, _i64] + [_vp, _i64] * 3 + [_vp, _vp, _f, _f] + [_vp, _i64] * 2 + [_vp]),
    "fsw_strerror": (_cp, [_i]),
    "fsw_last_hip_error": (_i, []),
    "fsw_decode_barrier_failures": (_i, []),
    "fsw_version": (_i, []),
    "fsw_set_variant": (_i, [_i, _i]),
    "fsw_variant_name": (_cp, [_i, _i, _i64, _i64, _i64]),
}

# the benchmark's measurement kernels live in a library of their own (include/fsw_probe.h)
PROBE_LIB_PATH = os.path.join(HERE, "libfsw_probe.so")
PROBE_PROTOTYPES = {
    "fsw_probe_mfma": (_i, [_i, _i, _vp, _vp, _i, _vp]),
    "fsw_probe_read": (_i, [_vp, _sz, _vp, _i, _vp]),
}

_lib = None
_probe_lib = None


class FswError(RuntimeError):
    """An FSW_E_* code from the library (RuntimeError, the failure mode of the reference's TORCH_CHECKs)."""

    def __init__(self, code, text):
        super().__init__("%s (code %d)" % (text, code))
        self.code = code


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                "%s is missing: build it with `python setup.py build_hip` in %s" % (LIB_PATH, HERE))
        # torch ships its own HIP runtime: when it is installed, load it first, so that this process holds one
        # runtime only (loaded the other way round, the library's launches fail with FSW_E_DEVICE)
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in PROTOTYPES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


def probe_lib():
    """libfsw_probe.so (measurement kernels for bench.py), loaded after the product library."""
    global _probe_lib
    if _probe_lib is None:
        lib()
        if not os.path.exists(PROBE_LIB_PATH):
            raise FileNotFoundError("%s is missing: build it with `python setup.py build_hip` in %s" % (PROBE_LIB_PATH, HERE))
        L = ctypes.CDLL(PROBE_LIB_PATH)
        for name, (res, args) in PROBE_PROTOTYPES.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _probe_lib = L
    return _probe_lib


def strerror(code):
    return lib().fsw_strerror(code).decode()


def check(code):
    if code != OK:
        raise FswError(code, strerror(code))


def dtype_code(t):
    import torch
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.float16:
        return FP16
    raise FswError(E_DTYPE, strerror(E_DTYPE))


def _stream(t):
    import torch
    return torch.cuda.current_stream(t.device).cuda_stream


def _ld(t):
    """Row stride in elements; degenerate shapes (one row, empty rows) report the row length."""
    if t.shape[0] > 1 and t.shape[1] > 0:
        return t.stride(0)
    return t.shape[1]


def _check_operands(first, *others, out=None, out_shape=None, workspace=None):
    """The guards of the PyTorch operator surface, for callers of the raw C ABI: 2-D device tensors with a unit
    inner stride, all on one device; `out` of the same type with the expected shape; `workspace` a uint8 device
    tensor. A transposed view passes a leading-dimension test and would be read as if it were row-major."""
    import torch
    for t in (first,) + others + ((out,) if out is not None else ()):
        if t.dim() != 2:
            raise FswError(E_SHAPE, "fsw: operands must be 2-D")
        if not t.is_cuda:
            raise FswError(E_DEVICE, "fsw: operands must be device tensors")
        if t.device != first.device:
            raise FswError(E_DEVICE, "fsw: operands live on different devices")
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise FswError(E_LD, "fsw: operands must be contiguous in their last dimension")
        if t.shape[0] > 1 and t.shape[1] > 0 and t.stride(0) < t.shape[1]:
            raise FswError(E_LD, "fsw: overlapping rows")
    if out is not None:
        if out.dtype != first.dtype or tuple(out.shape) != tuple(out_shape):
            raise FswError(E_SHAPE, "fsw: `out` must be a %s tensor of shape %s" % (first.dtype, tuple(out_shape)))
    if workspace is not None:
        if workspace.dtype != torch.uint8 or not workspace.is_cuda or workspace.device != first.device or \
                not workspace.is_contiguous():
            raise FswError(E_WORKSPACE, "fsw: workspace must be a contiguous uint8 tensor on the operands' device")


def gateup(X, W13, out=None):
    """H[M, ff] = up * silu(gate) through fsw_gateup on the current stream. X [M,K], W13 [2ff,K] device tensors."""
    import torch
    code = dtype_code(X)
    if W13.dtype != X.dtype:
        raise FswError(E_DTYPE, "fsw: X and W13 differ in element type")
    _check_operands(X, W13)
    M, K = X.shape
    N = W13.shape[0]
    if W13.shape[1] != K:
        raise FswError(E_SHAPE, "fsw: X is [M, K] and W13 is [2 ff, K]: K differs")
    if out is None:
        out = torch.empty((M, N // 2), dtype=X.dtype, device=X.device)
    _check_operands(X, out=out, out_shape=(M, N // 2))
    with torch.cuda.device(X.device):
        check(lib().fsw_gateup(code, M, N, K, X.data_ptr(), _ld(X), W13.data_ptr(), _ld(W13), out.data_ptr(),
                               _ld(out), _stream(X)))
    return out


def gateup_f32out(X, W13, out=None):
    """H[M, ff] as float32, the gated fp32 value unrounded, through fsw_gateup_f32out."""
    import torch
    code = dtype_code(X)
    if W13.dtype != X.dtype:
        raise FswError(E_DTYPE, "fsw: X and W13 differ in element type")
    _check_operands(X, W13)
    M, K = X.shape
    N = W13.shape[0]
    if W13.shape[1] != K:
        raise FswError(E_SHAPE, "fsw: X is [M, K] and W13 is [2 ff, K]: K differs")
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.float32, device=X.device)
    if out.dtype != torch.float32 or tuple(out.shape) != (M, N // 2):
        raise FswError(E_SHAPE, "fsw: `out` must be a float32 tensor of shape %s" % ((M, N // 2),))
    _check_operands(out)
    with torch.cuda.device(X.device):
        check(lib().fsw_gateup_f32out(code, M, N, K, X.data_ptr(), _ld(X), W13.data_ptr(), _ld(W13), out.data_ptr(),
                                      _ld(out), _stream(X)))
    return out


def down(H, W2, out=None):
    """Y[M, D] = H @ W2.T through fsw_down on the current stream. H [M,FF], W2 [D,FF] device tensors."""
    import torch
    code = dtype_code(H)
    if W2.dtype != H.dtype:
        raise FswError(E_DTYPE, "fsw: H and W2 differ in element type")
    _check_operands(H, W2)
    M, FF = H.shape
    D = W2.shape[0]
    if W2.shape[1] != FF:
        raise FswError(E_SHAPE, "fsw: H is [M, FF] and W2 is [D, FF]: FF differs")
    if out is None:
        out = torch.empty((M, D), dtype=H.dtype, device=H.device)
    _check_operands(H, out=out, out_shape=(M, D))
    nbytes = lib().fsw_down_workspace_bytes(code, M, D, FF)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=H.device) if nbytes else None
    with torch.cuda.device(H.device):
        check(lib().fsw_down(code, M, D, FF, H.data_ptr(), _ld(H), W2.data_ptr(), _ld(W2), out.data_ptr(), _ld(out),
                             ws.data_ptr() if ws is not None else None, nbytes, _stream(H)))
    return out


def mlp_workspace(X, FF):
    import torch
    M, D = X.shape
    nbytes = lib().fsw_mlp_workspace_bytes(dtype_code(X), M, D, FF)
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=X.device)


def mlp(X, W13, W2, out=None, workspace=None):
    """Y = (silu(X @ Wg) * (X @ Wu)) @ Wd through fsw_mlp. `workspace` (uint8 device tensor) may be reused."""
    import torch
    code = dtype_code(X)
    if W13.dtype != X.dtype or W2.dtype != X.dtype:
        raise FswError(E_DTYPE, "fsw: X, W13 and W2 differ in element type")
    _check_operands(X, W13, W2)
    M, D = X.shape
    FF = W13.shape[0] // 2
    if W13.shape[1] != D or tuple(W2.shape) != (D, FF):
        raise FswError(E_SHAPE, "fsw: X is [M, d], W13 is [2 ff, d] and W2 is [d, ff]")
    if out is None:
        out = torch.empty((M, D), dtype=X.dtype, device=X.device)
    if workspace is None:
        workspace = mlp_workspace(X, FF)
    _check_operands(X, out=out, out_shape=(M, D), workspace=workspace)
    with torch.cuda.device(X.device):
        check(lib().fsw_mlp(code, M, D, FF, X.data_ptr(), _ld(X), W13.data_ptr(), _ld(W13), W2.data_ptr(), _ld(W2),
                            out.data_ptr(), _ld(out), workspace.data_ptr(), workspace.numel(), _stream(X)))
    return out


def mlp_static(X, W13, W2, out):
    """fsw_mlp_static: the forward with the library's own static scratch; `out` is required (nothing is allocated)."""
    import torch
    code = dtype_code(X)
    if W13.dtype != X.dtype or W2.dtype != X.dtype:
        raise FswError(E_DTYPE, "fsw: X, W13 and W2 differ in element type")
    _check_operands(X, W13, W2)
    M, D = X.shape
    FF = W13.shape[0] // 2
    if W13.shape[1] != D or tuple(W2.shape) != (D, FF):
        raise FswError(E_SHAPE, "fsw: X is [M, d], W13 is [2 ff, d] and W2 is [d, ff]")
    _check_operands(X, out=out, out_shape=(M, D))
    with torch.cuda.device(X.device):
        check(lib().fsw_mlp_static(code, M, D, FF, X.data_ptr(), _ld(X), W13.data_ptr(), _ld(W13), W2.data_ptr(),
                                   _ld(W2), out.data_ptr(), _ld(out), _stream(X)))
    return out


class Blocked:
    """A panel-blocked device copy of a row-major [rows, k] matrix (fsw.h: blocks of [256 rows][32 elements])."""

    def __init__(self, buf, rows, k, dtype):
        self.buf, self.rows, self.k, self.dtype = buf, rows, k, dtype

    def data_ptr(self):
        return self.buf.data_ptr()


def _blocked_empty(rows, k, like):
    import torch
    n = lib().fsw_blocked_bytes(rows, k)
    return Blocked(torch.empty(max(n, 16), dtype=torch.uint8, device=like.device), rows, k, like.dtype)


def block_rows(A, kind="rows"):
    """Row-major device matrix -> Blocked. kind: "rows" (X, H, W2) or "w13" (up/gate rows de-interleaved per panel)."""
    import torch
    _check_operands(A)
    rows, k = A.shape
    out = _blocked_empty(rows, k, A)
    fn = {"rows": lib().fsw_block_rows, "w13": lib().fsw_prepack_w13, "w2": lib().fsw_prepack_w2}[kind]
    with torch.cuda.device(A.device):
        check(fn(dtype_code(A), rows, k, A.data_ptr(), _ld(A), out.data_ptr(), _stream(A)))
    return out


def unblock(B):
    """Blocked -> row-major torch tensor (host-side index arithmetic on the device buffer; for tests)."""
    import torch
    panels, nkt = (B.rows + 255) // 256, (B.k + 31) // 32
    t = B.buf[: panels * nkt * 256 * 64].view(B.dtype).view(panels, nkt, 256, 32)
    return t.permute(0, 2, 1, 3).reshape(panels * 256, nkt * 32)[: B.rows, : B.k].contiguous()


def gateup_blocked(Xb, W13, row_major_out=False):
    """Gate/up of a Blocked X: returns a Blocked H, or a row-major tensor with row_major_out. W13: row-major tensor
    or a Blocked from block_rows(W13, "w13")."""
    import torch
    wb = isinstance(W13, Blocked)
    N = W13.rows if wb else W13.shape[0]
    like = Xb.buf
    if row_major_out:
        H = torch.empty((Xb.rows, N // 2), dtype=Xb.dtype, device=like.device)
        ldh = max(N // 2, 1)
    else:
        H = Blocked(torch.empty(max(lib().fsw_blocked_bytes(Xb.rows, N // 2), 16), dtype=torch.uint8,
                                device=like.device), Xb.rows, N // 2, Xb.dtype)
        ldh = 0
    code = BF16 if Xb.dtype == torch.bfloat16 else FP16
    with torch.cuda.device(like.device):
        check(lib().fsw_gateup_blocked(code, Xb.rows, N, Xb.k, Xb.data_ptr(), W13.data_ptr(), 0 if wb else _ld(W13),
                                       1 if wb else 0, H.data_ptr(), ldh, _stream(like)))
    return H


def gateup_hblocked(X, W13):
    """Gate/up of a row-major X written as a Blocked H (what fsw_mlp runs in the large-tile regime). W13: row-major
    tensor or a Blocked from block_rows(W13, "w13")."""
    import torch
    _check_operands(X)
    wb = isinstance(W13, Blocked)
    if not wb:
        _check_operands(X, W13)
    N = W13.rows if wb else W13.shape[0]
    M, K = X.shape
    H = _blocked_empty(M, N // 2, X)
    with torch.cuda.device(X.device):
        check(lib().fsw_gateup_hblocked(dtype_code(X), M, N, K, X.data_ptr(), _ld(X), W13.data_ptr(),
                                        0 if wb else _ld(W13), 1 if wb else 0, H.data_ptr(), _stream(X)))
    return H


def down_blocked(Hb, W2, out=None):
    """Row-major Y = Blocked H @ W2.T. W2: row-major tensor or a Blocked from block_rows(W2, "w2")."""
    import torch
    wb = isinstance(W2, Blocked)
    D = W2.rows if wb else W2.shape[0]
    like = Hb.buf
    if out is None:
        out = torch.empty((Hb.rows, D), dtype=Hb.dtype, device=like.device)
    code = BF16 if Hb.dtype == torch.bfloat16 else FP16
    with torch.cuda.device(like.device):
        check(lib().fsw_down_blocked(code, Hb.rows, D, Hb.k, Hb.data_ptr(), W2.data_ptr(), 0 if wb else _ld(W2),
                                     1 if wb else 0, out.data_ptr(), _ld(out), _stream(like)))
    return out


def _row_args(t):
    """Base, token stride and head stride of a [tokens, heads, channels] device tensor."""
    return t.data_ptr(), _step(t, 0), _step(t, 1)


def _step(t, dim):
    """Stride of a dimension; one that is never stepped along may hold anything."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


def _check_rows(first, *others):
    for t in (first,) + others:
        if t.dim() != 3:
            raise FswError(E_SHAPE, "fsw: rows must be [tokens, heads, channels]")
        if not t.is_cuda or t.device != first.device:
            raise FswError(E_DEVICE, "fsw: operands must be device tensors on one device")
        if t.dtype != first.dtype:
            raise FswError(E_DTYPE, "fsw: operands differ in element type")
        if t.shape[2] > 1 and t.stride(2) != 1:
            raise FswError(E_LD, "fsw: channels must be contiguous")


def _check_int32(like, *arrays):
    import torch
    for t in arrays:
        if t.dtype != torch.int32:
            raise FswError(E_DTYPE, "fsw: positions, slots, pages, lengths and offsets are int32")
        if not t.is_cuda or t.device != like.device:
            raise FswError(E_DEVICE, "fsw: operands must be device tensors on one device")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise FswError(E_LD, "fsw: int32 arrays must be contiguous")


def kv_cache(k_cache, v_cache):
    """fsw_kv_cache of two [pages, heads, page_size, channels] device tensors with the same strides (any order of dimensions
    whose channels are contiguous)."""
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape or \
            any(_step(k_cache, i) != _step(v_cache, i) for i in range(3)):
        raise FswError(E_SHAPE, "fsw: the caches must be [pages, heads, page_size, channels] with the same strides")
    if k_cache.shape[3] > 1 and k_cache.stride(3) != 1:
        raise FswError(E_LD, "fsw: channels must be contiguous")
    return KvCache(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0], k_cache.shape[2], _step(k_cache, 0),
                   _step(k_cache, 1), _step(k_cache, 2))


def kv_append(q, k, v, cos_sin, positions, slots, k_cache, v_cache, interleaved=False, q_out=None, k_out=None):
    """Rotated copies of q [T, Hq, D] and k [T, Hkv, D]; rotated k, and v, go to their slots of the caches (fsw_kv_append).
    k_out=False: rotated keys go to the cache only, the second result is None."""
    import torch
    code = dtype_code(q)
    _check_rows(q, k, v)
    _check_int32(q, positions, slots)
    cache = kv_cache(k_cache, v_cache)
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != k.shape or tuple(k_cache.shape[1::2]) != (Hkv, D):
        raise FswError(E_SHAPE, "fsw: q is [T, Hq, D], k and v are [T, Hkv, D], the caches [pages, Hkv, page_size, D]")
    if positions.shape != (T,) or slots.shape != (T,) or cos_sin.dim() != 2:
        raise FswError(E_SHAPE, "fsw: positions and slots are [T], cos_sin is [rows, rot]")
    if cos_sin.dtype != torch.float32 or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise FswError(E_DTYPE, "fsw: cos_sin is float32, the caches have the rows' element type")
    if any(t.device != q.device for t in (cos_sin, k_cache, v_cache)):
        raise FswError(E_DEVICE, "fsw: operands live on different devices")
    if not cos_sin.is_contiguous():
        raise FswError(E_LD, "fsw: cos_sin must be contiguous")
    q_out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device) if q_out is None else q_out
    if k_out is False:
        k_out = None
    elif k_out is None:
        k_out = torch.empty((T, Hkv, D), dtype=q.dtype, device=q.device)
    _check_rows(q, q_out, *([] if k_out is None else [k_out]))
    if q_out.shape != q.shape or (k_out is not None and k_out.shape != k.shape):
        raise FswError(E_SHAPE, "fsw: q_out and k_out have the shapes of q and k")
    with torch.cuda.device(q.device):
        check(lib().fsw_kv_append(code, T, Hq, Hkv, D, cos_sin.shape[1], int(interleaved), *_row_args(q), *_row_args(k),
                                  *_row_args(v), cos_sin.data_ptr(), cos_sin.shape[0], positions.data_ptr(), slots.data_ptr(),
                                  *_row_args(q_out), *((None, 0, 0) if k_out is None else _row_args(k_out)), ctypes.byref(cache),
                                  _stream(q)))
    return q_out, k_out


def attn_decode(q, k_cache, v_cache, block_table, lengths, max_len, scale, out=None, workspace=None):
    """Attention of one token per sequence, q [B, Hq, D], over the paged caches (fsw_attn_decode). `workspace` (uint8 device
    tensor) may be reused."""
    import torch
    code = dtype_code(q)
    _check_rows(q)
    _check_int32(q, block_table, lengths)
    cache = kv_cache(k_cache, v_cache)
    B, Hq, D = q.shape
    Hkv = k_cache.shape[1]
    if k_cache.shape[3] != D or block_table.dim() != 2 or block_table.shape[0] != B or lengths.shape != (B,):
        raise FswError(E_SHAPE, "fsw: q is [B, Hq, D], the caches [pages, Hkv, page_size, D], block_table [B, width], lengths [B]")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise FswError(E_DTYPE, "fsw: the caches have the queries' element type")
    if k_cache.device != q.device or v_cache.device != q.device:
        raise FswError(E_DEVICE, "fsw: operands live on different devices")
    if block_table.shape[1] * k_cache.shape[2] < max_len:
        raise FswError(E_LD, "fsw: block_table is narrower than max_len")
    out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device) if out is None else out
    _check_rows(q, out)
    if out.shape != q.shape:
        raise FswError(E_SHAPE, "fsw: `out` has the shape of q")
    nbytes = lib().fsw_attn_decode_workspace_bytes(code, B, Hq, Hkv, D, max_len)
    if workspace is None and nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    if workspace is not None and (workspace.dtype != torch.uint8 or workspace.device != q.device or not workspace.is_contiguous()):
        raise FswError(E_WORKSPACE, "fsw: workspace must be a contiguous uint8 tensor on the operands' device")
    ld = block_table.stride(0) if B > 1 else block_table.shape[1]
    with torch.cuda.device(q.device):
        check(lib().fsw_attn_decode(code, B, Hq, Hkv, D, *_row_args(q), ctypes.byref(cache), block_table.data_ptr(), ld,
                                    lengths.data_ptr(), max_len, scale, *_row_args(out),
                                    workspace.data_ptr() if workspace is not None else None,
                                    workspace.numel() if workspace is not None else 0, _stream(q)))
    return out


def attn_prompt(q, k, v, cu_q, cu_k, scale, out=None):
    """Causal attention of packed sequences, q [Tq, Hq, D], k and v [Tk, Hkv, D], offsets [B + 1] (fsw_attn_prompt)."""
    import torch
    code = dtype_code(q)
    _check_rows(q, k, v)
    _check_int32(q, cu_q, cu_k)
    Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[:2]
    if k.shape[2] != D or v.shape != k.shape or cu_q.dim() != 1 or cu_q.numel() < 1 or cu_k.shape != cu_q.shape:
        raise FswError(E_SHAPE, "fsw: q is [Tq, Hq, D], k and v are [Tk, Hkv, D], offsets are [B + 1]")
    out = torch.empty((Tq, Hq, D), dtype=q.dtype, device=q.device) if out is None else out
    _check_rows(q, out)
    if out.shape != q.shape:
        raise FswError(E_SHAPE, "fsw: `out` has the shape of q")
    with torch.cuda.device(q.device):
        check(lib().fsw_attn_prompt(code, Tq, Tk, cu_q.numel() - 1, Hq, Hkv, D, *_row_args(q), *_row_args(k), *_row_args(v),
                                    cu_q.data_ptr(), cu_k.data_ptr(), scale, *_row_args(out), _stream(q)))
    return out


def kv_cache8(k_cache, v_cache, k_scale, v_scale):
    """fsw_kv_cache8 of two float8_e4m3fn tensors [pages, heads, page_size, channels] and their float8_e8m0fnu scales [pages, heads,
    page_size], each pair with the same strides."""
    import torch
    c = kv_cache(k_cache, v_cache)
    if k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != k_cache.dtype or \
            k_scale.dtype != torch.float8_e8m0fnu or v_scale.dtype != k_scale.dtype:
        raise FswError(E_DTYPE, "fsw: the caches are float8_e4m3fn, their scales float8_e8m0fnu")
    if k_scale.shape != k_cache.shape[:3] or v_scale.shape != k_scale.shape or any(_step(k_scale, i) != _step(v_scale, i) for i in range(3)):
        raise FswError(E_SHAPE, "fsw: the scales must be [pages, heads, page_size] with the same strides")
    return KvCache8(c.k, c.v, k_scale.data_ptr(), v_scale.data_ptr(), c.pages, c.page_size, c.page_stride, c.head_stride, c.token_stride,
                    _step(k_scale, 0), _step(k_scale, 1), _step(k_scale, 2))


def _check_caches(caches, *kinds):
    """`caches` are two tensors of the rows' type, or four of 8 bits and their scales, where `kinds` has that number."""
    if len(caches) not in kinds:
        raise FswError(E_SHAPE, "fsw: the caches are %s" % " or ".join({2: "(k, v)", 4: "(k, v, k_scale, v_scale)"}[n] for n in kinds))


def _cache_of(like, caches, dtype, heads, channels):
    """A cache's structure from (k, v) or (k, v, k_scale, v_scale), checked against the rows it goes with."""
    if any(not t.is_cuda or t.device != like.device for t in caches):
        raise FswError(E_DEVICE, "fsw: operands must be device tensors on one device")
    c = kv_cache(*caches) if len(caches) == 2 else kv_cache8(*caches)
    if len(caches) == 2 and (caches[0].dtype != dtype or caches[1].dtype != dtype):
        raise FswError(E_DTYPE, "fsw: the caches have the rows' element type")
    if tuple(caches[0].shape[1::2]) != (heads, channels):
        raise FswError(E_SHAPE, "fsw: the caches are [pages, Hkv, page_size, D]")
    return ctypes.byref(c)


def kv_append8(q, k, v, cos_sin, positions, slots, caches, interleaved=False, q_out=None, k_out=None, v_out=None):
    """Rotated q, and k and v as the cache in 8 bits holds them; `caches` is (k, v, k_scale, v_scale) (fsw_kv_append8). k_out=False,
    v_out=False: the cache only, the result is None."""
    import torch
    _check_caches(caches, 4)
    code = dtype_code(q)
    _check_rows(q, k, v)
    _check_int32(q, positions, slots)
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != k.shape or positions.shape != (T,) or slots.shape != (T,) or cos_sin.dim() != 2:
        raise FswError(E_SHAPE, "fsw: q is [T, Hq, D], k and v are [T, Hkv, D], positions and slots [T], cos_sin [rows, rot]")
    if cos_sin.dtype != torch.float32:
        raise FswError(E_DTYPE, "fsw: cos_sin is float32")
    if cos_sin.device != q.device:
        raise FswError(E_DEVICE, "fsw: operands live on different devices")
    if not cos_sin.is_contiguous():
        raise FswError(E_LD, "fsw: cos_sin must be contiguous")
    cache = _cache_of(q, caches, q.dtype, Hkv, D)
    q_out, k_out, v_out = (None if o is False else torch.empty(r.shape, dtype=r.dtype, device=r.device) if o is None else o
                           for o, r in ((q_out, q), (k_out, k), (v_out, v)))
    for o, r in ((q_out, q), (k_out, k), (v_out, v)):
        if o is not None:
            _check_rows(q, o)
            if o.shape != r.shape:
                raise FswError(E_SHAPE, "fsw: q_out, k_out and v_out have the shapes of q, k and v")
    outs = [_row_args(o) if o is not None else (None, 0, 0) for o in (q_out, k_out, v_out)]
    with torch.cuda.device(q.device):
        check(lib().fsw_kv_append8(code, T, Hq, Hkv, D, cos_sin.shape[1], int(interleaved), *_row_args(q), *_row_args(k), *_row_args(v),
                                   cos_sin.data_ptr(), cos_sin.shape[0], positions.data_ptr(), slots.data_ptr(), *outs[0], *outs[1],
                                   *outs[2], cache, _stream(q)))
    return q_out, k_out, v_out


def kv_read(caches, block_table, cu, tokens, dtype=None, k_out=None, v_out=None):
    """Keys and values [tokens, Hkv, D] of sequences whose offsets are cu [B + 1], out of their pages (fsw_kv_read; with scales among
    `caches` fsw_kv_read8, whose results are of `dtype`)."""
    import torch
    _check_caches(caches, 2, 4)
    eight = len(caches) == 4
    like = caches[0]
    if like.dim() != 4:
        raise FswError(E_SHAPE, "fsw: the caches are [pages, Hkv, page_size, D]")
    dtype = dtype if eight else like.dtype
    _check_int32(like, block_table, cu)
    Hkv, D = like.shape[1::2]
    cache = _cache_of(like, caches, dtype, Hkv, D)
    if cu.dim() != 1 or cu.numel() < 1 or block_table.dim() != 2 or block_table.shape[0] != cu.numel() - 1:
        raise FswError(E_SHAPE, "fsw: block_table is [B, width], offsets are [B + 1]")
    k_out, v_out = (torch.empty((tokens, Hkv, D), dtype=dtype, device=like.device) if o is None else o for o in (k_out, v_out))
    _check_rows(k_out, v_out)
    if k_out.shape != (tokens, Hkv, D) or v_out.shape != k_out.shape or k_out.dtype != dtype or k_out.device != like.device:
        raise FswError(E_SHAPE, "fsw: k_out and v_out are [tokens, Hkv, D]")
    B, width = block_table.shape
    f = lib().fsw_kv_read8 if eight else lib().fsw_kv_read
    with torch.cuda.device(like.device):
        check(f(dtype_code(k_out), tokens, B, Hkv, D, cache, block_table.data_ptr(), block_table.stride(0) if B > 1 else width, width,
                cu.data_ptr(), *_row_args(k_out), *_row_args(v_out), _stream(like)))
    return k_out, v_out


def _attend(q, caches, prefix, prefix_len, block_table, lengths, max_len, scale, out, workspace):
    import torch
    code = dtype_code(q)
    _check_rows(q)
    _check_int32(q, block_table, lengths, *([] if prefix is None else [prefix]))
    B, Hq, D = q.shape
    if caches[0].dim() != 4 or block_table.dim() != 2 or block_table.shape[0] != B or lengths.shape != (B,):
        raise FswError(E_SHAPE, "fsw: q is [B, Hq, D], the caches [pages, Hkv, page_size, D], block_table [B, width], lengths [B]")
    Hkv, page = caches[0].shape[1:3]
    cache = _cache_of(q, caches, q.dtype, Hkv, D)
    if block_table.shape[1] * page < max_len:
        raise FswError(E_LD, "fsw: block_table is narrower than max_len")
    if prefix is not None and (prefix.dim() != 1 or prefix.numel() * page < prefix_len):
        raise FswError(E_LD, "fsw: prefix has fewer pages than prefix_len needs")
    out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device) if out is None else out
    _check_rows(q, out)
    if out.shape != q.shape:
        raise FswError(E_SHAPE, "fsw: `out` has the shape of q")
    L, head = lib(), [code, B, Hq, Hkv, D]
    if prefix is None:
        f, first, nbytes = L.fsw_attn_decode8, [], L.fsw_attn_decode8_workspace_bytes(*head, max_len)
    else:
        f, size = (L.fsw_attn_shared8, L.fsw_attn_shared8_workspace_bytes) if len(caches) == 4 else \
            (L.fsw_attn_shared, L.fsw_attn_shared_workspace_bytes)
        first, nbytes = [prefix.data_ptr(), prefix_len], size(*head, prefix_len, max_len)
    if workspace is None and nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    if workspace is not None and (workspace.dtype != torch.uint8 or workspace.device != q.device or not workspace.is_contiguous()):
        raise FswError(E_WORKSPACE, "fsw: workspace must be a contiguous uint8 tensor on the operands' device")
    with torch.cuda.device(q.device):
        check(f(*head, *_row_args(q), cache, *first, block_table.data_ptr(), block_table.stride(0) if B > 1 else block_table.shape[1],
                lengths.data_ptr(), max_len, scale, *_row_args(out), workspace.data_ptr() if workspace is not None else None,
                workspace.numel() if workspace is not None else 0, _stream(q)))
    return out


def attn_decode8(q, caches, block_table, lengths, max_len, scale, out=None, workspace=None):
    """Attention of one token per sequence over the caches (k, v, k_scale, v_scale) in 8 bits (fsw_attn_decode8)."""
    _check_caches(caches, 4)
    return _attend(q, caches, None, 0, block_table, lengths, max_len, scale, out, workspace)


def attn_shared(q, caches, prefix, prefix_len, block_table, lengths, max_len, scale, out=None, workspace=None):
    """Attention of one token per sequence over a prefix that all share, in pages prefix [n], and its own tokens, over (k, v) or
    (k, v, k_scale, v_scale) (fsw_attn_shared, fsw_attn_shared8)."""
    _check_caches(caches, 2, 4)
    if prefix is None:
        raise FswError(E_NULL, "fsw: prefix is an int32 tensor of pages; without one there is attn_decode, attn_decode8")
    return _attend(q, caches, prefix, prefix_len, block_table, lengths, max_len, scale, out, workspace)


def add_norm(x, y=None, gate=None, post=None, pre=None, scale=1.0, eps=1e-5, x_out=None, h=None):
    """(x', h) of rows x, y [M, D]: x' = x + scale * gate * norm(y) * post, h = norm(x') * pre (fsw_add_norm). gate: [D] or [M, D].
    Without y: (None, norm(x) * pre). x_out=False, h=False: not computed, None."""
    import torch
    code = dtype_code(x)
    if gate is not None and gate.dim() not in (1, 2):
        raise FswError(E_SHAPE, "fsw: gate is [D] or [M, D]")
    rows = [t for t in (y, gate if gate is not None and gate.dim() == 2 else None) if t is not None]
    _check_operands(x, *rows)
    M, D = x.shape
    if any(t.shape != x.shape for t in rows):
        raise FswError(E_SHAPE, "fsw: x, y and a gate of rows are [M, D]")
    for t in (post, pre, gate if gate is not None and gate.dim() == 1 else None):
        if t is not None and (t.shape != (D,) or (D > 1 and t.stride(0) != 1)):
            raise FswError(E_SHAPE, "fsw: weights are [D], contiguous")
    x_out, h = (None if o is False else torch.empty_like(x, memory_format=torch.contiguous_format) if o is None else o for o in (x_out, h))
    x_out = None if y is None else x_out
    for o in (x_out, h):
        if o is not None:
            _check_operands(x, out=o, out_shape=(M, D))
    for t in (y, gate, post, pre):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise FswError(E_DTYPE, "fsw: operands differ in element type or device")
    two = lambda t: (t.data_ptr(), _ld(t)) if t is not None else (None, 0)  # noqa: E731
    one = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    gate_args = two(gate) if gate is not None and gate.dim() == 2 else (one(gate), 0)
    with torch.cuda.device(x.device):
        check(lib().fsw_add_norm(code, M, D, *two(x), *two(y), *gate_args, one(post), one(pre), scale, eps, *two(x_out), *two(h), _stream(x)))
    return x_out, h


def set_variant(family, variant):
    check(lib().fsw_set_variant(family, variant))


def decode_barrier_failures():
    """Single-launch decode forwards whose device-wide barrier gave up since the last call (synchronous)."""
    n = lib().fsw_decode_barrier_failures()
    if n < 0:
        check(n)
    return n


def variant_name(family, dtype, M, n, k):
    return lib().fsw_variant_name(family, dtype, M, n, k).decode()
