"""The 8-bit integer (W8A8) linear path: row quantisers that feed it and the integer matrix product.

A token row ``y`` becomes int8 codes with one fp32 scale, ``s = max(max|y| / 127, 2^-120)``, ``q = rint(y / s)``, half to even.
``quantize_act_int8`` rounds the exact quotient ``127 y / max|y|``; the norm and SwiGLU, whose ``y`` are rounded fp32 values,
round ``y * (1 / s)``, which is within 2^-16 of ``y / s``. A weight row (output channel) is quantised by the exact quotient
too, once, at load (``codec.quantize_int8``, ``QLinear.from_dense(w, "int8")``). The product
``out[i, m] = (sum_k q[i, k] c[m, k]) * s[i] * row_scale[m]`` has an exact integer sum, so it depends neither on the batch
width nor on how the kernel splits K.

No result of a token depends on the other rows of the call, on their number or on where its row lies: the norm sums a row's
squares in one order that goes by the width alone.

A row that holds an infinity or a NaN gets scale NaN and codes 0: all that is computed from it is NaN.

Wrappers check their arguments before anything is enqueued (``KernelError``), launch on the current stream of the
tensors' device, and allocate only what the caller does not hand in. Rows ``>= n`` of every buffer stay as they are.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from ..models.weights import QLinear
from . import lib as _lib
from .lib import KernelError, c_float, c_int, c_ll, c_void_p, empty_beside as _empty

MAX_K = 131071                 # 128 * 128 * K must stay below 2^31
MAX_ROWS = 1 << 27
# fp32 squares below 2^-126 flush to zero: beside an eps of 2^-100 that is 2^-26 of mean + eps; a smaller one may become zero itself
EPS_MIN, EPS_MAX = 2.0 ** -100, 2.0 ** 127
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_BF16, _INT8 = (torch.bfloat16,), (torch.int8,)


@dataclass
class Int8Act:
    """Quantised tokens: ``q`` int8 ``[rows, k]`` (row pitch a multiple of 16 bytes), ``scale`` fp32 ``[rows]``."""
    q: torch.Tensor
    scale: torch.Tensor


def act_buffers(rows: int, k: int, device) -> Int8Act:
    """Buffers a quantiser can write into (``out=``) and ``linear_int8`` can read."""
    if k & 15:
        q = torch.empty_strided((rows, k), ((k + 15) & ~15, 1), dtype=torch.int8, device=device)
    else:
        q = torch.empty(rows, k, dtype=torch.int8, device=device)
    return Int8Act(q, torch.empty(rows, dtype=torch.float32, device=device))


# argument types of the C entries, set once so that plain ints and floats convert without wrapper objects
_P, _I, _L, _F = c_void_p, c_int, c_ll, c_float
_TYPES = {"vg_quant_int8": (_P, _L, _I, _I, _I, _P, _L, _P, _P, _P),
          "vg_swiglu_int8": (_P, _L, _I, _I, _P, _L, _P, _P, _P),
          "vg_add_rmsnorm_int8": (_P, _L, _P, _L, _P, _I, _I, _F, _I, _P, _L, _P, _P, _L, _P, _P),
          "vg_dequant_int8": (_P, _L, _P, _P, _L, _I, _I, _I, _P, _P),
          "vg_gemm_int8": (_P, _L, _P, _P, _L, _P, _P, _L, _I, _I, _I, _I, _P, _P)}
_fns = {}
_err = {}                      # device index -> address of the device's error word


def _fn(name: str):
    f = getattr(_lib.lib(), name)
    f.argtypes = _TYPES[name]
    f.restype = c_int
    _fns[name] = f
    return f


def _err_word(index: int) -> int:
    if index < 0:
        raise KernelError("the 8-bit integer path runs on CUDA tensors")
    device = torch.device("cuda", index)
    if torch.cuda.is_current_stream_capturing() and device not in _lib._err_words:
        # made here, the word would be cleared by every replay instead of once
        raise KernelError("call the 8-bit integer path once before capturing it: its error word does not exist yet")
    p = _err[index] = _lib.err_word(device).data_ptr()
    return p


def _launch(name: str, index: int, *args):
    """Enqueues on the current stream of device ``index``; every entry ends with (error word, stream)."""
    err = _err.get(index) or _err_word(index)
    fn = _fns.get(name) or _fn(name)
    if index != _lib.current_index():
        with torch.cuda.device(index):
            _lib.check(fn(*args, err, _lib.raw_stream(index)), name)
        return
    _lib.check(fn(*args, err, _lib.raw_stream(index)), name)


def _input(t: torch.Tensor, what: str, dtypes, n: Optional[int]):
    """Rows to process, row width and row pitch of a call's main argument."""
    shape = t.shape
    if len(shape) != 2:
        raise KernelError(f"{what}: expected a matrix, got shape {tuple(shape)}")
    rows, cols = shape
    if n is None:
        n = rows
    if not 0 <= n <= rows or n > MAX_ROWS:
        raise KernelError(f"{what}: {n} rows asked for, the tensor has {rows}")
    if t.dtype not in dtypes:
        raise KernelError(f"{what}: dtype {t.dtype} is not supported")
    ld, inner = t.stride()
    if inner != 1 or ld < cols:
        ld = _pitch(t, what, n, cols)
    return n, cols, ld


def _pitch(t: torch.Tensor, what: str, rows: int, cols: int) -> int:
    """Row pitch of a matrix whose strides are not plainly row-major: single rows and columns may have any."""
    ld, inner = t.stride()
    if (inner != 1 and cols > 1) or (ld < cols and rows > 1):
        raise KernelError(f"{what}: rows must be contiguous and must not overlap (strides {t.stride()})")
    return ld if rows > 1 else max(ld, cols)


def _matrix(t: torch.Tensor, what: str, dtypes, rows: int, cols: int, index: int) -> int:
    """Row pitch of a 2-D row-major argument that has to hold ``rows`` x ``cols`` elements."""
    if t.dtype not in dtypes:
        raise KernelError(f"{what}: dtype {t.dtype} is not supported")
    shape = t.shape
    if len(shape) != 2 or shape[0] < rows or shape[1] != cols:
        raise KernelError(f"{what}: shape {tuple(shape)}, expected at least {rows} rows of {cols}")
    if t.get_device() != index:
        raise KernelError(f"{what} is on {t.device}, expected CUDA device {index}")
    ld, inner = t.stride()
    return ld if inner == 1 and ld >= cols else _pitch(t, what, rows, cols)


def _vector(t: torch.Tensor, what: str, size: int, index: int, least: bool = False):
    shape = t.shape
    if t.dtype is not torch.float32 or len(shape) != 1 or (shape[0] < size if least else shape[0] != size) \
            or t.get_device() != index or not t.is_contiguous():
        raise KernelError(f"{what}: expected {size} contiguous fp32 values on CUDA device {index}, "
                          f"got {t.dtype} {tuple(shape)} on {t.device}")


def _out(out: Optional[Int8Act], n: int, k: int, like: torch.Tensor):
    """The quantisers' output buffers and their row pitch."""
    if k < 1 or k > MAX_K:
        raise KernelError(f"row width {k} is outside 1 .. {MAX_K}")
    if out is None:
        ld = (k + 15) & ~15
        return Int8Act(_empty(like, (n, k), (ld, 1), torch.int8), _empty(like, (n,), (1,), torch.float32)), ld
    index = like.get_device()
    ld = _matrix(out.q, "out.q", _INT8, n, k, index)
    _vector(out.scale, "out.scale", n, index, least=True)
    return out, ld


def quantize_act_int8(x: torch.Tensor, n: Optional[int] = None, out: Optional[Int8Act] = None) -> Int8Act:
    """Quantise rows ``x[:n]`` (bf16 / f16 / f32 ``[rows, k]``)."""
    n, k, ld = _input(x, "x", _DTYPE, n)
    out, ldq = _out(out, n, k, x)
    if n:
        _launch("vg_quant_int8", x.get_device(), x.data_ptr(), ld, _DTYPE[x.dtype], n, k, out.q.data_ptr(), ldq, out.scale.data_ptr())
    return out


def swiglu_int8(gu: torch.Tensor, n: Optional[int] = None, inter: Optional[int] = None, out: Optional[Int8Act] = None) -> Int8Act:
    """``silu(gate) * up`` of ``gu[:n] = [gate | up]`` (bf16 ``[rows, 2 * inter]``), quantised."""
    n, cols, ld = _input(gu, "gu", _BF16, n)
    if inter is None:
        inter = cols // 2
    if cols != 2 * inter:
        raise KernelError(f"gu: {cols} columns, expected 2 * {inter}")
    out, ldq = _out(out, n, inter, gu)
    if n:
        _launch("vg_swiglu_int8", gu.get_device(), gu.data_ptr(), ld, n, inter, out.q.data_ptr(), ldq, out.scale.data_ptr())
    return out


def add_rmsnorm_int8(res: torch.Tensor, delta: Optional[torch.Tensor], w: torch.Tensor, eps: float, n: Optional[int] = None,
                     out: Optional[Int8Act] = None, out16: Optional[torch.Tensor] = None, plus_one: bool = True) -> Int8Act:
    """``res[:n] += delta[:n]`` (bf16, in place, when delta is given), then RMSNorm with weights ``w`` (``1 + w`` with
    ``plus_one``) quantised; the normed rows also go to ``out16`` (f16, saturating) when it is given."""
    n, h, ld = _input(res, "res", _BF16, n)
    dev = res.get_device()
    if not EPS_MIN <= eps <= EPS_MAX:
        raise KernelError(f"eps must be in 2^-100 .. 2^127, got {eps}")
    out, ldq = _out(out, n, h, res)
    ldd = ldo = 0
    if delta is not None:
        ldd = _matrix(delta, "delta", _BF16, n, h, dev)
    if out16 is not None:
        ldo = _matrix(out16, "out16", (torch.float16,), n, h, dev)
    _vector(w, "w", h, dev)
    if n:
        _launch("vg_add_rmsnorm_int8", dev, res.data_ptr(), ld, 0 if delta is None else delta.data_ptr(), ldd, w.data_ptr(), n, h,
                eps, 1 if plus_one else 0, out.q.data_ptr(), ldq, out.scale.data_ptr(),
                0 if out16 is None else out16.data_ptr(), ldo)
    return out


def dequantize_act_int8(act: Int8Act, n: Optional[int] = None, out: Optional[torch.Tensor] = None,
                        dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values rows ``act.q[:n]`` stand for, in bf16, f16 (saturating) or f32 (``out``'s type when it is given)."""
    q = act.q
    n, k, ldq = _input(q, "act.q", _INT8, n)
    dev = q.get_device()
    if k < 1 or k > MAX_K:
        raise KernelError(f"row width {k} is outside 1 .. {MAX_K}")
    _vector(act.scale, "act.scale", n, dev, least=True)
    if out is None:
        if dtype not in _DTYPE:
            raise KernelError(f"dtype {dtype} is not supported")
        out = _empty(q, (n, k), (k, 1), dtype)
        ldo = k
    else:
        ldo = _matrix(out, "out", _DTYPE, n, k, dev)
    if n:
        _launch("vg_dequant_int8", dev, q.data_ptr(), ldq, act.scale.data_ptr(), out.data_ptr(), ldo, _DTYPE[out.dtype], n, k)
    return out


def linear_int8(q: QLinear, act: Int8Act, n: Optional[int] = None, out: Optional[torch.Tensor] = None,
                out_f32: bool = False) -> torch.Tensor:
    """``out[:n] = act @ W^T`` for an ``int8`` linear, bf16 or fp32 (``out``'s type when it is given). Codes of both sides are
    read in place: rows must start on 16-byte boundaries (``codec.rows16`` re-lays a matrix whose rows do not)."""
    if q.fmt != "int8":
        raise KernelError(f"linear_int8 takes int8 weights, got {q.fmt}")
    n, cols, ldq = _input(act.q, "act.q", _INT8, n)
    m, k, dev = q.m, q.k, act.q.get_device()
    if k < 1 or k > MAX_K or m < 1:
        raise KernelError(f"weights [{m}, {k}]: K must be in 1 .. {MAX_K}")
    if cols != k:
        raise KernelError(f"act.q: {cols} columns, the weights have {k}")
    ldw = _matrix(q.codes, "codes", _INT8, m, k, dev)
    if m == 1:
        ldw = (k + 15) & ~15
    if n <= 1:
        ldq = (k + 15) & ~15
    wp, qp = q.codes.data_ptr(), act.q.data_ptr()
    if (ldw | ldq | wp | qp) & 15:
        raise KernelError("int8 rows must start on 16-byte boundaries (codec.rows16)")
    _vector(q.row_scale, "row_scale", m, dev)
    _vector(act.scale, "act.scale", n, dev, least=True)
    if out is None:
        out = _empty(act.q, (n, m), (m, 1), torch.float32 if out_f32 else torch.bfloat16)
        ldo = m
    else:
        ldo = _matrix(out, "out", (torch.bfloat16, torch.float32), n, m, dev)
    if n:
        _launch("vg_gemm_int8", dev, wp, ldw, q.row_scale.data_ptr(), qp, ldq, act.scale.data_ptr(), out.data_ptr(), ldo,
                1 if out.dtype == torch.float32 else 0, m, k, n)
    return out
