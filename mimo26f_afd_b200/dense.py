"""Dense operators around the routed experts, over the C ABI: projections with MXFP4 weights in the checkpoint layout (a
shared expert, a first dense layer) and the step between two blocks (rank sum, norms, gate, residual).

Where the reference has cuBLAS projections on the coordinator (crates/mimo26-coordinator/src/gpu_dense.rs) and separate
launches for the rank sum, the residual add and the norm (kernels/glue.cu), these work on the expert weights' own format and
in one pass. Arguments are device buffers (anything with ``data_ptr()`` or an address); work is enqueued on ``stream`` (an
address; None = the default stream) and nothing is synchronised.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading

from . import _native
from .expert import X_BF16, ExpertError, _check, _ptr

GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_ELEMENT = 0, 1, 2, 3
Y_BF16, Y_F32 = 0, 1


# struct m26b_linear_args and struct m26b_block_norm_args of the header
_LINEAR_ARGS = struct.Struct("@4PQP2QI3i")
_NORM_ARGS = struct.Struct("@14P3Q3f2I7i")
_local = threading.local()


def _err():
    """This thread's error buffer and its address (a decode step makes several calls per layer; a fresh buffer each costs more
    than the rest of the check)."""
    try:
        return _local.err
    except AttributeError:
        buf = C.create_string_buffer(256)
        _local.err = buf, C.addressof(buf)
        return _local.err


def _addr(x) -> int:
    if x is None:
        return 0
    if type(x) is int:
        return x
    try:
        return x.data_ptr()
    except AttributeError:
        return _ptr(x)


def _any_addr(x):
    """The address of a buffer of no rows: an empty tensor has none, and any stands for it, since nothing is read or written."""
    return x if x is None or type(x) is int else _addr(x) or 1 << 20


class Linear:
    """One prepared MXFP4 matrix (``new``: y = x W^T) or gated pair (``gated``: silu(x Wg^T) * (x Wu^T)) on the current
    device. Weights ``w`` u8 [n, k/2], scales ``s`` u8 [n, k/32]; the sources may be freed afterwards."""

    def __init__(self, handle: int, n: int, k: int):
        self._h, self.n, self.k = C.c_void_p(handle), n, k

    @classmethod
    def new(cls, w, s, n: int, k: int) -> "Linear":
        out, err = C.c_void_p(), C.create_string_buffer(256)
        _check(_native.lib().m26b_linear_new(_ptr(w), _ptr(s), n, k, C.byref(out), err, 256), err)
        return cls(out.value, n, k)

    @classmethod
    def gated(cls, gate_w, gate_s, up_w, up_s, n: int, k: int) -> "Linear":
        out, err = C.c_void_p(), C.create_string_buffer(256)
        _check(_native.lib().m26b_linear_new_gated(_ptr(gate_w), _ptr(gate_s), _ptr(up_w), _ptr(up_s), n, k, C.byref(out), err, 256), err)
        return cls(out.value, n, k)

    def workspace_bytes(self, rows: int) -> int:
        """Device bytes ``linear_dev`` needs for ``rows`` tokens."""
        return int(_native.lib().m26b_linear_workspace_bytes(self._h, rows))

    def set_wait_us(self, us: int) -> None:
        """Bound of a call's wait for its own tensor-core work (default about 200,000 us); later calls that exceed it put code 3
        into their fault word."""
        if not 0 < us < 1 << 32 or _native.lib().m26b_linear_set_wait_us(self._h, us):
            raise ExpertError(1, "m26b linear: bad wait bound or handle")

    def close(self) -> None:
        if self._h:
            _native.lib().m26b_linear_free(self._h)
            self._h = C.c_void_p(0)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _nbytes(buf) -> int:
    n = getattr(buf, "nbytes", None)
    if n is None:
        raise ExpertError(1, "m26b linear: pass workspace_bytes with a workspace address")
    return int(n)


def linear_dev(layer: Linear, x, rows: int, y, *, x_dtype: int = X_BF16, x_scales=None, x_pitch: int = 0, y_dtype: int = Y_BF16,
               y_pitch: int = 0, workspace=None, workspace_bytes=None, fault=None, stream=None) -> None:
    """y [rows, n] from x [rows, k] (BF16, or E4M3 with ``x_scales`` [rows, k/32]); pitches in elements, 0 = dense rows.
    ``workspace`` holds ``layer.workspace_bytes(rows)`` bytes and serves one call at a time; ``fault`` is one int32 / uint32
    that receives code 3 if a bounded wait inside the kernel ran out."""
    if workspace_bytes is None:
        workspace_bytes = 0 if workspace is None else _nbytes(workspace)
    try:
        args = _LINEAR_ARGS.pack(_addr(x), _addr(x_scales), _addr(y), _addr(workspace), workspace_bytes, _addr(fault), x_pitch, y_pitch, rows,
                                 x_dtype, y_dtype, 0)
    except (struct.error, OverflowError) as e:        # a negative or oversized number
        raise ExpertError(1, f"m26b linear: bad arguments ({e})") from None
    buf, at = _err()
    rc = _native.lib().m26b_linear_dev(layer._h, args, _addr(stream), at, 256)
    if rc:
        _check(rc, buf)


def block_norm_dev(planes, residual, rows: int, width: int, *, post_w=None, gate=None, gate_kind: int = GATE_NONE, y_dtype: int = 0,
                   y_pitch: int = 0, y_scale: float = 1.0, h_dtype: int = 1, h_pitch: int = 0, residual_scale: float = 1.0, pre_w=None,
                   w_dtype: int = 1, eps: float = 1e-6, h_out=None, n_out=None, n_dtype: int = 0, n_pitch: int = 0, stream=None) -> None:
    """u = sum of ``planes`` in order, normed with ``post_w`` if given; h = residual_scale * residual + y_scale * gate * u into
    ``h_out``; n = the RMS norm of h (times ``pre_w``) into ``n_out``. dtypes 0 = BF16, 1 = FP32; pitches in elements, 0 =
    dense rows; ``planes`` a sequence of up to eight device buffers (empty: norm of the residual alone). No rows are no work; the
    other arguments are checked all the same, and empty tensors are fine."""
    n = len(planes)
    if not rows:
        planes = [_any_addr(p) for p in planes]
        gate, residual, h_out, n_out = _any_addr(gate), _any_addr(residual), _any_addr(h_out), _any_addr(n_out)
    if n > 8:
        raise ExpertError(1, "m26b block norm: bad arguments")
    try:
        if n == 1:
            args = _NORM_ARGS.pack(_addr(planes[0]), 0, 0, 0, 0, 0, 0, 0, _addr(post_w), _addr(gate), _addr(residual), _addr(pre_w), _addr(h_out),
                                   _addr(n_out), y_pitch, h_pitch, n_pitch, y_scale, residual_scale, eps, rows, width, 1, gate_kind, y_dtype,
                                   h_dtype, n_dtype, w_dtype, 0)
        else:
            args = _NORM_ARGS.pack(*map(_addr, planes), *_PAD[n], _addr(post_w), _addr(gate), _addr(residual), _addr(pre_w), _addr(h_out),
                                   _addr(n_out), y_pitch, h_pitch, n_pitch, y_scale, residual_scale, eps, rows, width, n, gate_kind, y_dtype,
                                   h_dtype, n_dtype, w_dtype, 0)
    except (struct.error, OverflowError) as e:        # a negative or oversized number
        raise ExpertError(1, f"m26b block norm: bad arguments ({e})") from None
    buf, at = _err()
    rc = _native.lib().m26b_block_norm_dev(args, _addr(stream), at, 256)
    if rc:
        _check(rc, buf)


_PAD = [(0,) * (8 - i) for i in range(9)]
