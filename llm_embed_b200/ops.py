"""Stand-alone operators of newer encoder layers over libllmembed_cuda, beside
embed.QWeight (le_qgemm_device): the e4m3 product with a scale for each block
of 128 (F8Weight) and its quantiser, the norm of query and key heads with the
position rotation (Rope), and differential attention (DiffAttention).

As with embed.QWeight the calls take device addresses, enqueue their work on
`stream` and return; the formulas, shapes and limits are in
include/llmembed.h.  Without a `stream` all of them go to the legacy default
stream, so one call's result may be the next one's input (a framework whose
current stream has the handle 0 means that one: pass LEGACY_STREAM).  `stream` 0
is the handle's own stream (the quantiser has no handle: the legacy one), which
orders neither with that nor with another handle's.  Element types are "f32",
"f16", "bf16" and "e4m3".
"""
from __future__ import annotations

import ctypes as C
import struct
import threading

import numpy as np

from . import embed
from .embed import LE_EINVAL, LlmEmbedError, _check

LEGACY_STREAM = 1  # cudaStreamLegacy
TYPES = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}
PAIRINGS = {"interleaved": 0, "half": 1}


# The argument structures of include/llmembed.h, field by field (packing one
# takes a fraction of the time that building a ctypes.Structure does).
_F8GEMM_ARGS = struct.Struct("@PPPPqqqiii4x").pack
_QK_NORM_ARGS = struct.Struct("@PPPPPPPqqqqiiiiif").pack
_DIFFATTN_ARGS = struct.Struct("@PPPPPqqqqiiii").pack

_lib = None
_lib_lock = threading.Lock()


def lib() -> C.CDLL:
    """The CUDA library with the operators' signatures."""
    global _lib
    if _lib is None:
        with _lib_lock:
            if _lib is None:
                L = embed.lib()
                vp, i, i64 = C.c_void_p, C.c_int, C.c_int64
                out = C.POINTER(vp)
                L.le_f8_quantize_device.argtypes = [i, i, vp, i64, i, i, vp, vp, vp]
                L.le_f8weight_create.argtypes = [i, vp, vp, i, i, out]
                L.le_f8weight_quantize.argtypes = [i, vp, i, i, out]
                L.le_f8weight_read.argtypes = [vp, vp, vp]
                L.le_f8gemm_workspace.argtypes = [vp, i, i, C.POINTER(i64)]
                L.le_f8gemm_tile.argtypes = [i, i]
                L.le_f8gemm_device.argtypes = [vp, vp, vp]
                L.le_rope_create.argtypes = [i, i, i, C.c_double, i, out]
                L.le_qk_norm_device.argtypes = [vp, vp, vp]
                L.le_diffattn_create.argtypes = [i, i, i, i, vp, i, C.c_float, vp, C.c_float, out]
                L.le_diffattn_device.argtypes = [vp, vp, vp]
                for name in ("f8weight", "rope", "diffattn"):
                    getattr(L, f"le_{name}_sync").argtypes = [vp]
                    getattr(L, f"le_{name}_free").argtypes = [vp]
                _lib = L
    return _lib


def _id(table: dict, name: str, what: str) -> int:
    try:
        return table[name]
    except (KeyError, TypeError):
        raise LlmEmbedError(LE_EINVAL, f"{what} {name!r} is none of {', '.join(table)}") from None


def _i32(**sizes) -> None:
    """Refuse sizes that a C int does not hold (ctypes would cut them)."""
    for name, v in sizes.items():
        if not -(1 << 31) <= v < 1 << 31:
            raise LlmEmbedError(LE_EINVAL, f"{name} {v} does not fit 32 bits")


def _run(fn, h, pack, stream: int, *args) -> None:
    """fn(handle, packed arguments, stream), its code checked."""
    try:
        packed = pack(*args)
    except (struct.error, TypeError) as e:
        raise LlmEmbedError(LE_EINVAL, f"argument out of range or of another type: {e}") from None
    rc = fn(h, packed, stream or None)
    if rc:
        _check(rc)


class _Handle:
    _name = ""

    def __init__(self, h):
        self._h = h.value

    def sync(self) -> None:
        """Wait for the device; raise on a failure that a kernel of an earlier call reported."""
        _check(getattr(lib(), f"le_{self._name}_sync")(self._h))

    def close(self) -> None:
        if getattr(self, "_h", None):
            getattr(lib(), f"le_{self._name}_free")(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def f8_quantize_device(d_x: int, x_type: str, M: int, K: int, d_q: int, d_scales: int, ldx: int = 0, dev: int = 0,
                       stream: int = LEGACY_STREAM) -> None:
    """x [M][K] -> e4m3 bytes [M][K] and scales [ceil(K/128)][M] (le_f8_quantize_device)."""
    _i32(M=M, K=K, dev=dev)
    rc = (_lib or lib()).le_f8_quantize_device(dev, _id(TYPES, x_type, "type"), d_x, ldx, M, K, d_q, d_scales,
                                               stream or None)
    if rc:
        _check(rc)


class F8Weight(_Handle):
    """An e4m3 weight [N][K] with a scale for each block of 128 x 128: y = x . W^T."""

    _name = "f8weight"

    def __init__(self, wq, scales, N: int, K: int, dev: int = 0):
        """wq (bytes) and scales (float32): numpy arrays or host or device addresses."""
        _i32(N=N, K=K, dev=dev)
        wp, _w = _address(wq, np.uint8, N * K)
        sp, _s = _address(scales, np.float32, -(-N // 128) * -(-K // 128))
        h = C.c_void_p()
        _check(lib().le_f8weight_create(dev, wp, sp, N, K, C.byref(h)))
        super().__init__(h)
        self.N, self.K = N, K

    @classmethod
    def from_float(cls, w: np.ndarray, dev: int = 0) -> "F8Weight":
        """Quantise float32 w [N][K] (le_f8weight_quantize)."""
        w = np.ascontiguousarray(w, np.float32)
        if w.ndim != 2:
            raise LlmEmbedError(LE_EINVAL, f"w has {w.ndim} dimensions, not 2")
        _i32(N=w.shape[0], K=w.shape[1], dev=dev)
        h = C.c_void_p()
        _check(lib().le_f8weight_quantize(dev, w.ctypes.data, w.shape[0], w.shape[1], C.byref(h)))
        self = cls.__new__(cls)
        _Handle.__init__(self, h)
        self.N, self.K = w.shape
        return self

    def read(self) -> tuple[np.ndarray, np.ndarray]:
        """The weight's bytes [N][K] and scales."""
        q = np.empty((self.N, self.K), np.uint8)
        s = np.empty((-(-self.N // 128), -(-self.K // 128)), np.float32)
        _check(lib().le_f8weight_read(self._h, q.ctypes.data, s.ctypes.data))
        return q, s

    def workspace_bytes(self, M: int, x_type: str) -> int:
        _i32(M=M)
        n = C.c_int64(0)
        _check(lib().le_f8gemm_workspace(self._h, M, _id(TYPES, x_type, "type"), C.byref(n)))
        return n.value

    def matmul_device(self, d_x: int, M: int, d_y: int, x_type: str = "f16", y_type: str = "f16", ldx: int = 0,
                      ldy: int = 0, d_x_scales: int = 0, d_work: int = 0, work_bytes: int = 0,
                      stream: int = LEGACY_STREAM) -> None:
        """y [M][N] = x [M][K] . W^T; x is quantised in the call, or e4m3 with d_x_scales."""
        _run((_lib or lib()).le_f8gemm_device, self._h, _F8GEMM_ARGS, stream, d_x, d_x_scales, d_y, d_work, work_bytes,
             ldx, ldy, M, _id(TYPES, x_type, "type"), _id(TYPES, y_type, "type"))


def _address(a, dtype, n: int):
    if isinstance(a, int):
        return a, None
    a, dtype = np.ascontiguousarray(a), np.dtype(dtype)
    # Bytes may be of any type of one byte; other values are what they are.
    if a.dtype != dtype and (a.dtype.itemsize != 1 or dtype.itemsize != 1) or a.size != n:
        raise LlmEmbedError(LE_EINVAL, f"expected {n} values of {dtype.name}, not {a.size} of {a.dtype.name}")
    return a.ctypes.data, a


class Rope(_Handle):
    """Rotation table; qk_norm_device norms and rotates query and key heads."""

    _name = "rope"

    def __init__(self, max_pos: int, rot_dim: int, base: float = 10000.0, pairing: str = "interleaved", dev: int = 0):
        _i32(max_pos=max_pos, rot_dim=rot_dim, dev=dev)
        h = C.c_void_p()
        _check(lib().le_rope_create(dev, max_pos, rot_dim, base, _id(PAIRINGS, pairing, "pairing"), C.byref(h)))
        super().__init__(h)

    def qk_norm_device(self, dtype: str, n_tokens: int, q_heads: int, k_heads: int, head_dim: int, d_q: int, d_k: int,
                       d_positions: int, d_q_out: int, d_k_out: int, q_stride: int = 0, k_stride: int = 0,
                       q_out_stride: int = 0, k_out_stride: int = 0, d_q_weight: int = 0, d_k_weight: int = 0,
                       eps: float = 1e-6, stream: int = LEGACY_STREAM) -> None:
        _run((_lib or lib()).le_qk_norm_device, self._h, _QK_NORM_ARGS, stream, d_q, d_k, d_q_out, d_k_out, d_q_weight,
             d_k_weight, d_positions, q_stride, k_stride, q_out_stride, k_out_stride, _id(TYPES, dtype, "type"),
             n_tokens, q_heads, k_heads, head_dim, eps)


class DiffAttention(_Handle):
    """Differential attention with its learned weights."""

    _name = "diffattn"

    def __init__(self, heads: int, kv_heads: int, head_dim: int, lambdas, lambda_init: float, norm_weight=None,
                 eps: float = 1e-5, dev: int = 0):
        """lambdas [4][head_dim] or [heads][4][head_dim] (lq1, lk1, lq2, lk2); norm_weight [2 * head_dim] or None."""
        _i32(heads=heads, kv_heads=kv_heads, head_dim=head_dim, dev=dev)
        lam = np.ascontiguousarray(lambdas, np.float32)
        if heads < 1 or head_dim < 1:
            raise LlmEmbedError(LE_EINVAL, f"heads {heads} and head_dim {head_dim} must be positive")
        if lam.size != 4 * head_dim and lam.size != heads * 4 * head_dim:
            raise LlmEmbedError(LE_EINVAL, f"lambdas have {lam.size} values, not [4][{head_dim}] for one or {heads} heads")
        nw = None if norm_weight is None else np.ascontiguousarray(norm_weight, np.float32)
        if nw is not None and nw.size != 2 * head_dim:
            raise LlmEmbedError(LE_EINVAL, f"norm_weight has {nw.size} values, not {2 * head_dim}")
        h = C.c_void_p()
        _check(lib().le_diffattn_create(dev, heads, kv_heads, head_dim, lam.ctypes.data, lam.size // (4 * head_dim),
                                        lambda_init, None if nw is None else nw.ctypes.data, eps, C.byref(h)))
        super().__init__(h)

    def run_device(self, dtype: str, d_q: int, d_k: int, d_v: int, d_offsets: int, nseq: int, n_tokens: int,
                   max_len: int, d_out: int, q_stride: int = 0, k_stride: int = 0, v_stride: int = 0,
                   out_stride: int = 0, stream: int = LEGACY_STREAM) -> None:
        _run((_lib or lib()).le_diffattn_device, self._h, _DIFFATTN_ARGS, stream, d_q, d_k, d_v, d_out, d_offsets,
             q_stride, k_stride, v_stride, out_stride, _id(TYPES, dtype, "type"), nseq, n_tokens, max_len)
