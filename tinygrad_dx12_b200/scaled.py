"""8-bit activations between packed projections: block-scaled rows, the RMS norm that makes them, and
products of them with packed weights.

tinygrad-dx12 has no counterpart: its packed path ends at one matmul (``src/tinygrad_dx12/codegen/
linalg.py:136-223``). ``matmul`` takes 16-bit activations and decodes the weights; here both sides stay
as they are stored, E4M3 codes of the activations beside FP4 / FP6 codes of the weights, each with a power
of two for every 32 values, and the tensor cores multiply them so:

    x8, h = rms_norm(y, weight, residual=h, dtype=torch.float8_e4m3fn)      add, norm, quantise
    m8    = scaled_linear(x8, gate_up, activation="silu", gated=True, dtype=torch.float8_e4m3fn)
    h     = scaled_linear(m8, down, residual=h)

Everything runs in the library's kernels on the current stream; there is no CPU path. No gradients: results carry
none, whatever their operands ask for.

Which product to take: ``scaled_linear`` for many tokens (several times ``matmul``'s rate), for an epilogue and for
experts; at one or two tokens ``matmul`` streams the weights as fast or faster, on 16-bit activations (one token x 57344 x
8192 49 us and 52, x 8192 x 8192 11 and 18; eight 83 and 52, 18 and 18).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .attention import _REAL, _call, _elsewhere
from .packed import PackedTensor, _require_cuda

BLOCK = 32
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
ROWS_TOKENS, ROWS_PAIRS, ROWS_PLAN = 0, 1, 2  # B200_ROWS_*
SCALED_FORMATS = ("fp4_e2m1", "fp6_e2m3", "fp6_e3m2")
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_RESULTS = {**_REAL, _E4M3: _lib.DT["fp8e4m3"]}


class NormArgs(ctypes.Structure):
    """``b200_norm_args``."""

    _fields_ = [("x", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("total", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("y", ctypes.c_void_p), ("y_scales", ctypes.c_void_p),
                ("rows", ctypes.c_int64), ("cols", ctypes.c_int64), ("x_stride", ctypes.c_int64),
                ("residual_stride", ctypes.c_int64), ("total_stride", ctypes.c_int64), ("x_dtype", ctypes.c_int32),
                ("total_dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32), ("y_dtype", ctypes.c_int32),
                ("normalize", ctypes.c_int32), ("eps", ctypes.c_float)]


class ScaledArgs(ctypes.Structure):
    """``b200_scaled_args``."""

    _fields_ = [("x", ctypes.c_void_p), ("x_scales", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("residual_stride", ctypes.c_int64),
                ("y", ctypes.c_void_p), ("y_scales", ctypes.c_void_p), ("scratch", ctypes.c_void_p),
                ("offsets", ctypes.c_void_p), ("order", ctypes.c_void_p), ("experts", ctypes.c_int64),
                ("fan", ctypes.c_int32), ("x_rows", ctypes.c_int32), ("y_rows", ctypes.c_int32), ("bias_dtype", ctypes.c_int32),
                ("residual_dtype", ctypes.c_int32), ("y_dtype", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("gated", ctypes.c_int32), ("general", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class BlockScaled:
    """Rows of 8-bit values: ``codes`` float8_e4m3fn (..., dim) and ``scales`` float8_e8m0fnu (..., dim / 32),
    a power of two for every 32 values along the last axis. ``quantize`` and ``rms_norm`` make them."""

    __slots__ = ("_codes", "_scales", "_raw", "shape", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != _E4M3 or scales.dtype != _E8M0:
            raise ValueError("block-scaled rows are float8_e4m3fn codes with float8_e8m0fnu scales")
        if codes.dim() < 1 or codes.shape[-1] % BLOCK:
            raise ValueError(f"block-scaled rows are whole blocks of {BLOCK}")
        expected = (*codes.shape[:-1], codes.shape[-1] // BLOCK)
        if tuple(scales.shape) != expected:
            raise ValueError(f"scales must have shape {expected}")
        if scales.device != codes.device:
            raise _elsewhere("scales", scales, codes.device)
        self._codes, self._scales, self._raw, self.shape, self.device = codes, scales, None, codes.shape, codes.device

    @classmethod
    def _empty(cls, shape, device) -> "BlockScaled":
        """Codes and, behind them, scales in one allocation, which a small call's host time is made of; the tensors
        are made when asked for. (Scales begin on a multiple of 32 bytes, as codes are whole blocks.)"""
        x = object.__new__(cls)
        n = math.prod(shape)
        x._raw = torch.empty(n + n // BLOCK, dtype=torch.uint8, device=device)
        x._codes, x._scales, x.shape, x.device = None, None, torch.Size(shape), x._raw.device
        return x

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._raw[: math.prod(self.shape)].view(_E4M3).view(self.shape)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._raw[math.prod(self.shape):].view(_E8M0).view(*self.shape[:-1], self.shape[-1] // BLOCK)
        return self._scales

    def __repr__(self) -> str:
        return f"BlockScaled(shape={tuple(self.shape)}, device={self.device})"

    def _pointers(self):
        """Addresses of contiguous codes and scales on the boundaries that the kernels ask for, and what keeps them."""
        if self._raw is not None:
            codes = self._raw.data_ptr()
            return codes, codes + math.prod(self.shape), None
        codes, scales = self._codes, self._scales
        if not codes.is_contiguous() or codes.data_ptr() % 16:
            codes = codes.clone(memory_format=torch.contiguous_format)
        if not scales.is_contiguous() or scales.data_ptr() % 4:
            scales = scales.clone(memory_format=torch.contiguous_format)
        return codes.data_ptr(), scales.data_ptr(), (codes, scales)

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """What the codes stand for, rounded once (bfloat16 and float32 hold every value whose scale lies in
        [2^-100, 2^100])."""
        if dtype not in _REAL:
            raise ValueError(f"values are float16, bfloat16 or float32, not {dtype}")
        if self.device.type != "cuda":
            _require_cuda(self.codes, "block-scaled rows")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        n = math.prod(self.shape)
        if n:
            codes, scales, keep = self._pointers()
            cols = self.shape[-1]
            _call("b200_scaled_values", self.device, codes, scales, n // cols, cols, out.data_ptr(), _REAL[dtype])
        return out


def _flat(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """t (..., cols) as (rows, cols) with contiguous rows; a copy where its axes do not fold."""
    if t.dim() != 2:
        t = t.reshape(rows, cols)
    return t if t.stride(1) == 1 or cols == 1 else t.contiguous()


def _norm(x, weight, eps, residual, total, dtype, normalize):
    device, shape = x.device, x.shape
    cols = shape[-1]
    rows = x.numel() // cols if cols else 0
    y = BlockScaled._empty(shape, device) if dtype == _E4M3 else torch.empty(shape, dtype=dtype, device=device)
    if rows and cols:
        flat = _flat(x, rows, cols)
        r = r_ptr = t_ptr = w_ptr = ys_ptr = None
        r_stride = t_stride = t_dtype = w_dtype = 0
        if residual is not None:
            r = _flat(residual, rows, cols)
            r_ptr, r_stride, t_ptr, t_stride, t_dtype = r.data_ptr(), r.stride(0), total.data_ptr(), cols, _REAL[residual.dtype]
        if weight is not None:
            w_ptr, w_dtype = weight.data_ptr(), _REAL[weight.dtype]
        if dtype == _E4M3:
            y_ptr, ys_ptr, _ = y._pointers()
        else:
            y_ptr = y.data_ptr()
        a = NormArgs(flat.data_ptr(), r_ptr, t_ptr, w_ptr, y_ptr, ys_ptr, rows, cols, flat.stride(0), r_stride, t_stride,
                     _REAL[x.dtype], t_dtype, w_dtype, _RESULTS[dtype], normalize, eps)
        _call("b200_rms_norm", device, ctypes.byref(a))
    return y


def quantize(x: torch.Tensor) -> BlockScaled:
    """``x`` (..., dim), float16, bfloat16 or float32, in 8 bits; dim a multiple of 32.

    A block of 32 values along the last axis gets the smallest power of two that is not below max|x| / 448 as
    its scale, held within [2^-100, 2^100], and each value the E4M3 code nearest to x / scale, ties to even,
    held at 448. A NaN makes its block's scale NaN."""
    if x.dtype not in _REAL or x.dim() < 1:
        raise ValueError(f"quantize takes float16, bfloat16 or float32 rows, not {x.dtype}")
    if x.shape[-1] % BLOCK:
        raise ValueError(f"block-scaled rows are whole blocks of {BLOCK}, not {x.shape[-1]} values")
    _require_cuda(x, "quantize's input")
    return _norm(x, None, 0.0, None, None, _E4M3, 0)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, residual: torch.Tensor | None = None,
             dtype: torch.dtype | None = None, total: torch.Tensor | None = None):
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last axis, in fp32, rounded once.

    x (..., dim): float16, bfloat16 or float32, any strides. ``weight`` (dim,) of one of these types. (Fastest, one reading
    of x: dim a multiple of 8, results of the residual's or x's own type or in 8 bits, residuals of x's type or fp32 x.)
    ``dtype``: the result's, x's by default; ``torch.float8_e4m3fn`` gives ``BlockScaled`` rows, quantised from
    fp32 as ``quantize`` does (dim a multiple of 32).

    With ``residual`` (x's shape) the norm is of ``residual + x``, rounded to the residual's type, which comes back
    too: ``y, total``. It is written into ``total`` when given (contiguous, of the residual's shape and type; it
    may be the residual itself). No gradients."""
    if x.dtype not in _REAL or x.dim() < 1:
        raise ValueError(f"rms_norm takes float16, bfloat16 or float32 rows, not {x.dtype}")
    dtype = x.dtype if dtype is None else dtype
    if dtype not in _RESULTS:
        raise ValueError(f"rms_norm gives float16, bfloat16, float32 or float8_e4m3fn, not {dtype}")
    if dtype == _E4M3 and x.shape[-1] % BLOCK:
        raise ValueError(f"block-scaled rows are whole blocks of {BLOCK}, not {x.shape[-1]} values")
    device = x.device
    if device.type != "cuda":
        _require_cuda(x, "rms_norm's input")
    if weight is not None:
        if weight.dtype not in _REAL or weight.shape != x.shape[-1:]:
            raise ValueError(f"weight must be float16, bfloat16 or float32 of shape ({x.shape[-1]},)")
        if weight.device != device:
            raise _elsewhere("weight", weight, device)
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if residual is None:
        if total is not None:
            raise ValueError("total needs a residual")
        return _norm(x, weight, eps, None, None, dtype, 1)
    if residual.dtype not in _REAL or residual.shape != x.shape:
        raise ValueError("residual must be float16, bfloat16 or float32 of x's shape")
    if residual.device != device:
        raise _elsewhere("residual", residual, device)
    if total is None:
        total = torch.empty(residual.shape, dtype=residual.dtype, device=device)
    elif total.shape != residual.shape or total.dtype != residual.dtype or total.device != device or not total.is_contiguous():
        raise ValueError("total must be contiguous, of the residual's shape, type and device")
    return _norm(x, weight, eps, residual, total, dtype, 1), total


def _check_weights(w: PackedTensor, dims: int, what: str) -> None:
    if not isinstance(w, PackedTensor) or len(w.shape) != dims:
        raise ValueError(f"{what} takes a PackedTensor of {dims} dimensions")
    if w.format not in SCALED_FORMATS:
        raise ValueError(f"{what} takes FP4 or FP6 weights, not {w.format}")
    if w.scales is None or w.scales.dtype != _E8M0 or w.block_size != BLOCK or w.cols < 1 or w.cols % BLOCK:
        raise ValueError(f"{what} takes weights with float8_e8m0fnu scales in whole blocks of {BLOCK}")
    if w.device.type != "cuda":
        _require_cuda(w.data, "packed data")


def _check_product(x, w, activation, gated, dtype, what):
    """Columns of the result."""
    if not isinstance(x, BlockScaled):
        raise ValueError(f"{what} takes BlockScaled activations (quantize, rms_norm)")
    if x.shape[-1] != w.cols:
        raise ValueError(f"activations of {x.shape[-1]} values do not fit weights of {w.cols}")
    if x.device != w.device:
        raise _elsewhere("activations", x, w.device)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    if dtype not in _RESULTS:
        raise ValueError(f"{what} gives float16, bfloat16, float32 or float8_e4m3fn, not {dtype}")
    cols = w.shape[-2]
    if gated:
        if cols % 2:
            raise ValueError("gated weights hold as many gate rows as up rows")
        cols //= 2
    if dtype == _E4M3 and cols % BLOCK:
        raise ValueError(f"block-scaled rows are whole blocks of {BLOCK}, not {cols} values")
    return cols


def _check_bias(bias, shape, device, name="bias"):
    if bias is None:
        return None
    if bias.dtype not in _REAL or tuple(bias.shape) != tuple(shape):
        raise ValueError(f"{name} must be float16, bfloat16 or float32 of shape {tuple(shape)}")
    if bias.device != device:
        raise _elsewhere(name, bias, device)
    return bias if bias.is_contiguous() else bias.contiguous()


def _args(x, xs, rows, y, ys, y_dtype, bias, activation, gated, residual=None, plan=None, x_rows=0, y_rows=1, general=False,
          scratch=None) -> ScaledArgs:
    """Arguments of one product: pointers of x and y, checked operands."""
    b_ptr = r_ptr = o_ptr = p_ptr = None
    b_dtype = r_dtype = r_stride = experts = fan = 0
    if bias is not None:
        b_ptr, b_dtype = bias.data_ptr(), _REAL[bias.dtype]
    if residual is not None:
        r_ptr, r_stride, r_dtype = residual.data_ptr(), residual.stride(0), _REAL[residual.dtype]
    if plan is not None:
        o_ptr, p_ptr, experts, fan = plan.offsets.data_ptr(), plan.rows.data_ptr(), plan.experts, plan.indices.shape[1]
    return ScaledArgs(x, xs, rows, b_ptr, r_ptr, r_stride, y, ys, scratch, o_ptr, p_ptr, experts, fan, x_rows, y_rows, b_dtype,
                      r_dtype, y_dtype, ACTIVATIONS[activation], int(gated), int(general), 0)


def _scratch_bytes(desc, a: ScaledArgs, w: PackedTensor) -> int:
    """What the product needs besides: the general kernel's sums, or rows in the plan's order."""
    if a.general or w.shape[-1] % 128 or w.shape[-1] > 1 << 24 or desc.data % 32 or desc.scales % 4 or (a.experts and a.x_rows != ROWS_PLAN):
        return _lib.lib().b200_scaled_linear_scratch(ctypes.byref(desc), ctypes.byref(a))
    return 0


def _product(x, w, y, rows, bias, activation, gated, residual=None, plan=None, x_rows=0, general=False):
    """Launches one product of checked operands into y."""
    codes, scales, keep = x._pointers()
    if type(y) is BlockScaled:
        y_ptr, ys_ptr, _ = y._pointers()
        y_dtype = _RESULTS[_E4M3]
    else:
        y_ptr, ys_ptr, y_dtype = y.data_ptr(), None, _REAL[y.dtype]
    a = _args(codes, scales, rows, y_ptr, ys_ptr, y_dtype, bias, activation, gated, residual, plan, x_rows, ROWS_PAIRS, general)
    desc = w.desc()
    size = _scratch_bytes(desc, a, w)
    if size:
        scratch = torch.empty(size, dtype=torch.uint8, device=x.device)
        a.scratch = scratch.data_ptr()
    _call("b200_scaled_linear", x.device, ctypes.byref(desc), ctypes.byref(a))


def scaled_linear(x: BlockScaled, w: PackedTensor, bias: torch.Tensor | None = None, activation: str | None = None,
                  gated: bool = False, residual: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
                  _general: bool = False):
    """``act(x W^T + bias) + residual``: products of 8-bit rows with packed weights and what follows them.

    x (..., K); ``w`` (N, K) FP4 or FP6 with E8M0 scales in blocks of 32 (K a multiple of 32; of 128, with data on a
    32-byte boundary, for the tensor cores: other calls, K = 2880 among them, take a general kernel of some 0.1 TFLOP/s). Both are multiplied
    as stored, sums are fp32. ``activation``: None, "relu", "silu", "gelu" or "gelu_tanh". ``gated``: w's rows are
    [gate; up], N / 2 each, and the result is act(gate) * up. ``bias`` (N,). ``residual`` (..., columns of the
    result) is added behind the activation. ``dtype``: float16, bfloat16 or float32, rounded once, or float8_e4m3fn for
    ``BlockScaled`` rows quantised from fp32 (columns a multiple of 32). No gradients."""
    _check_weights(w, 2, "scaled_linear")
    cols = _check_product(x, w, activation, gated, dtype, "scaled_linear")
    device = x.device
    bias = _check_bias(bias, w.shape[:1], device)
    shape = (*x.shape[:-1], cols)
    rows = math.prod(x.shape[:-1])
    if residual is not None:
        if residual.dtype not in _REAL or tuple(residual.shape) != shape:
            raise ValueError(f"residual must be float16, bfloat16 or float32 of shape {shape}")
        if residual.device != device:
            raise _elsewhere("residual", residual, device)
        residual = _flat(residual, rows, cols)
    y = BlockScaled._empty(shape, device) if dtype == _E4M3 else torch.empty(shape, dtype=dtype, device=device)
    if rows and cols:
        _product(x, w, y, rows, bias, activation, gated, residual, general=_general)
    return y
