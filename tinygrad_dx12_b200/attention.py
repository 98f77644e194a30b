"""Attention over a packed key/value cache: rotary positions, the cache, decode and shared prefixes.

tinygrad-dx12 has no counterpart: its packed path ends at one matmul (``src/tinygrad_dx12/codegen/
linalg.py:136-223``). These are the operators between the packed projections of a decoder layer:

    q, k   = rotary(q), rotary(k)                      ``rotary``, or fused into ``cache_write``
    cache <- quantised k, v of the new tokens          ``cache_write`` (``cache_read`` gives them back)
    out    = softmax(scale * q K^T) V                  ``cache_attention``, with or without a prefix
                                                       that the whole batch shares

Everything runs in the library's kernels on the current stream; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib
from . import dtypes as D
from .packed import _require_cuda, stream_ptr

CACHE_FORMATS = {"int8": 0, "fp8e4m3": 1, "int4": 2, "fp4_e2m1": 3}
CACHE_BITS = {"int8": 8, "fp8e4m3": 8, "int4": 4, "fp4_e2m1": 4}
HEAD_DIMS = (64, 128, 256)
_REAL = {torch.float16: _lib.DT["float16"], torch.bfloat16: _lib.DT["bfloat16"], torch.float32: _lib.DT["float32"]}
_INDEX = {torch.int32: _lib.DT["int32"], torch.int64: _lib.DT["int64"]}
_SCALES = {torch.bfloat16: _lib.DT["bfloat16"], torch.float8_e8m0fnu: _lib.DT["e8m0"]}
_I64x3 = ctypes.c_int64 * 3


class RotaryDesc(ctypes.Structure):
    """``b200_rotary_desc``."""

    _fields_ = [("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("rotary_dim", ctypes.c_int32), ("interleaved", ctypes.c_int32)]


class CacheDesc(ctypes.Structure):
    """``b200_cache_desc``."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page_size", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("block_size", ctypes.c_int32),
                ("format", ctypes.c_int32), ("scale_dtype", ctypes.c_int32), ("strides", ctypes.c_int64 * 3),
                ("scale_strides", ctypes.c_int64 * 3)]


class AttentionArgs(ctypes.Structure):
    """``b200_attention_args``."""

    _fields_ = [("q", ctypes.c_void_p), ("q_strides", ctypes.c_int64 * 3), ("tables", ctypes.c_void_p),
                ("lengths", ctypes.c_void_p), ("prefix", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("scratch", ctypes.c_void_p), ("batch", ctypes.c_int64),
                ("queries", ctypes.c_int64), ("table_stride", ctypes.c_int64), ("max_pages", ctypes.c_int64),
                ("prefix_pages", ctypes.c_int64), ("prefix_length", ctypes.c_int64), ("q_dtype", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


_FN: dict = {}  # library functions by name


def _call(name: str, device: torch.device, *args) -> None:
    """A library call on the current stream of the operands' device, which is made current."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_lib.lib(), name)
    if device.index is None or device.index == torch.cuda.current_device():
        status = fn(*args, stream_ptr(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream_ptr(device))
    if status < 0:
        _lib.check(status, name)


def _elsewhere(name: str, t, device: torch.device) -> ValueError:
    return ValueError(f"{name} must be on {device}, not {t.device}")


# ---- rotary positions -------------------------------------------------------------------------
class RotaryTable:
    """Cosines and sines of ``rotary_dim / 2`` pairs at positions 0 .. rows - 1, and how heads pair up.

    ``layout`` "half" pairs value i with i + rotary_dim / 2, "interleaved" 2i with 2i + 1. Values of
    a head behind ``rotary_dim`` are left alone. ``RotaryTable(cos, sin, layout)`` takes fp32 CUDA
    tensors of shape (rows, rotary_dim / 2); ``RotaryTable.build`` computes them."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, layout: str = "half"):
        if layout not in ("half", "interleaved"):
            raise ValueError(f"unknown rotary layout {layout!r}")
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
            raise ValueError("rotary tables must be float32 of one shape (rows, rotary_dim / 2)")
        if cos.shape[1] < 1:
            raise ValueError("rotary tables need at least one pair")
        _require_cuda(cos, "rotary tables")
        if sin.device != cos.device:
            raise _elsewhere("sin", sin, cos.device)
        self.cos, self.sin, self.layout = cos.contiguous(), sin.contiguous(), layout
        self.rotary_dim, self.rows, self.device = 2 * cos.shape[1], cos.shape[0], cos.device
        self.desc = RotaryDesc(self.cos.data_ptr(), self.sin.data_ptr(), self.rows, self.rotary_dim,
                               int(layout == "interleaved"))
        self._ref = ctypes.byref(self.desc)

    @classmethod
    def build(cls, rotary_dim: int, rows: int, base: float = 10000.0, layout: str = "half",
              scaling: str | None = None, factor: float = 1.0, original: int | None = None,
              beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda") -> "RotaryTable":
        """Angles position * base^(-2i / rotary_dim), computed in float64, rounded once.

        ``scaling`` stretches them to contexts ``factor`` times longer than ``original`` (rows /
        factor when not given): "linear" divides every position by the factor; "base" raises the
        base to base * factor^(rotary_dim / (rotary_dim - 2)); "by_parts" keeps pairs that turn more
        than ``beta_fast`` times within the original length, slows those that turn less than
        ``beta_slow`` times by the factor, ramps between, and multiplies cosine and sine by
        0.1 ln(factor) + 1."""
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError("rotary_dim must be even and positive")
        if rows < 1 or base <= 0 or factor <= 0:
            raise ValueError("rotary tables need rows, a positive base and a positive factor")
        if scaling not in (None, "linear", "base", "by_parts"):
            raise ValueError(f"unknown rotary scaling {scaling!r}")
        i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
        gain = 1.0
        if scaling == "base":
            if rotary_dim == 2:
                raise ValueError("base scaling needs rotary_dim > 2")
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        freq = base ** (-2.0 * i / rotary_dim)
        if scaling == "linear":
            freq = freq / factor
        elif scaling == "by_parts" and factor != 1.0:
            n = original if original is not None else rows / factor
            pair = lambda beta: rotary_dim * math.log(n / (beta * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rotary_dim - 1)
            ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            freq = freq * (1 - ramp) + freq / factor * ramp
            gain = 0.1 * math.log(factor) + 1.0
        a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * freq
        return cls((a.cos() * gain).float(), (a.sin() * gain).float(), layout)


def _index(t: torch.Tensor, name: str, shape, device) -> torch.Tensor:
    if t.dtype not in _INDEX:
        raise ValueError(f"{name} must be int32 or int64")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.device != device:
        raise _elsewhere(name, t, device)
    return t if t.is_contiguous() else t.contiguous()


def _turned(x, table, positions, transpose, out=None):
    """``rotary`` of operands that have been checked, but for ``out``."""
    device = x.device
    xs = x.stride()
    if xs[-1] != 1:
        x = x.contiguous()
        xs = x.stride()
    if out is None:
        out = torch.empty_like(x)  # x's own order of axes where that is dense
        if out.stride(-1) != 1:
            out = torch.empty(x.shape, dtype=x.dtype, device=device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != device:
        raise ValueError("out must have x's shape, type and device")
    ys = out.stride()
    if ys[-1] != 1:
        raise ValueError("out must have contiguous heads")
    shape = x.shape
    if len(shape) == 4:
        b, t, xb, yb = shape[0], shape[1], xs[0], ys[0]
    else:
        b, t, xb, yb = 1, shape[0], 0, 0
    _call("b200_rotary", device, x.data_ptr(), _REAL[x.dtype], b, t, shape[-2], shape[-1], xb, xs[-3], xs[-2],
          out.data_ptr(), yb, ys[-3], ys[-2], table._ref, positions.data_ptr(), _INDEX[positions.dtype], int(transpose))
    return out


_transforms = torch._C._are_functorch_transforms_active


def _tracked(x: torch.Tensor) -> bool:
    """Whether a gradient, a forward-mode tangent or a transform of torch.func goes through x (which may wrap
    the tensor there: only autograd's own call takes it out)."""
    if (x.requires_grad and torch.is_grad_enabled()) or _transforms():
        return True
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


class _Turn:
    """The linear map that rotary() applies: what autograd carries beside x, closed to torch.func's wrapping."""

    __slots__ = ("table", "positions", "version", "transpose")

    def __init__(self, table, positions, transpose):
        self.table, self.positions, self.transpose = table, positions, transpose
        self.version = None if positions.is_inference() else positions._version

    def of(self, x: torch.Tensor, back: bool) -> torch.Tensor:
        if self.version is not None and self.positions._version != self.version:
            raise RuntimeError("the positions of a rotary() were changed in place before its gradient was computed")
        transpose = self.transpose != back
        if _tracked(x):
            return _apply(x, _Turn(self.table, self.positions, transpose))
        return _turned(x, self.table, self.positions, transpose)


class _Rotary(torch.autograd.Function):
    # the map is linear: its gradient is the transposed map, a tangent goes through the map itself
    @staticmethod
    def forward(ctx, x, turn):
        ctx.turn = turn
        return _turned(x, turn.table, turn.positions, turn.transpose)

    @staticmethod
    def backward(ctx, dy):
        return ctx.turn.of(dy, back=True), None

    @staticmethod
    def jvp(ctx, tangent, _):
        return ctx.turn.of(tangent, back=False)


class _RotaryTransformed(_Rotary):
    """The form that torch.func's transforms take; elsewhere a training step's call is 115 us in it, 87 in the other."""

    @staticmethod
    def forward(x, turn):
        return _turned(x, turn.table, turn.positions, turn.transpose)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.turn = inputs[1]


def _apply(x, turn):
    return (_RotaryTransformed if _transforms() else _Rotary).apply(x, turn)


def rotary(x: torch.Tensor, table: RotaryTable, positions: torch.Tensor, transpose: bool = False,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """``x`` (..., tokens, heads, head_dim) with each pair turned by its token's position.

    Pair (a, b) becomes (a cos - b sin, b cos + a sin), computed in fp32 and rounded once to x's
    type (float16, bfloat16 or float32); ``transpose`` applies the transposed map, which is the
    gradient's. x has three or four axes of any strides (a copy is made when head_dim is not
    contiguous); ``positions`` (int32 or int64) has x's shape without the last two. ``out`` may be x
    itself. A position outside the table gives NaN and sets bit 1 of the device status.
    Differentiable in x, any number of times, in reverse and in forward mode."""
    if x.dim() not in (3, 4):
        raise ValueError("rotary takes (tokens, heads, head_dim) or (batch, tokens, heads, head_dim)")
    if x.dtype not in _REAL:
        raise ValueError(f"rotary takes float16, bfloat16 or float32, not {x.dtype}")
    if table.rotary_dim > x.shape[-1]:
        raise ValueError(f"a table of {table.rotary_dim} rotary dimensions does not fit heads of {x.shape[-1]}")
    device = x.device
    if device.type != "cuda":
        _require_cuda(x, "rotary input")
    if table.device != device:
        raise _elsewhere("table", table, device)
    positions = _index(positions, "positions", x.shape[:-2], device)
    if _tracked(x):
        if out is not None:
            raise ValueError("rotary with a gradient cannot write into out")
        return _apply(x, _Turn(table, positions, bool(transpose)))
    return _turned(x, table, positions, transpose, out)


# ---- the cache ----------------------------------------------------------------------------------
@dataclass(frozen=True, eq=False)  # a cache equals itself: comparing storage would read the device
class PackedCache:
    """Keys and values of cached tokens as low-bit codes with block scales, in pages.

    ``k`` and ``v``: uint8 (pages, kv_heads, page_size, head_dim * bits / 8), codes of ``format``
    (``CACHE_FORMATS``: int8, fp8e4m3, int4, fp4_e2m1) back to back, lowest bits first.
    ``k_scales`` and ``v_scales``: bfloat16 or ``torch.float8_e8m0fnu`` (pages, kv_heads, page_size,
    head_dim / block_size), a scale per 32 values or per head. Both may be views of any strides
    whose rows are contiguous, so that a page may hold heads before tokens or tokens before heads.
    Cell (page, offset) is slot ``page * page_size + offset``. ``PackedCache.empty`` allocates one."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    format: str
    head_dim: int
    block_size: int

    def __post_init__(self) -> None:
        if self.format not in CACHE_FORMATS:
            raise ValueError(f"unknown cache format {self.format!r}")
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"cache head_dim must be one of {HEAD_DIMS}, not {self.head_dim}")
        if self.block_size not in (32, self.head_dim):
            raise ValueError("cache block_size must be 32 or head_dim")
        if self.k.dim() != 4 or self.k.dtype != torch.uint8 or self.v.dtype != torch.uint8 or self.k.shape != self.v.shape:
            raise ValueError("cache codes must be two uint8 tensors (pages, kv_heads, page_size, bytes)")
        pages, heads, size, row = self.k.shape
        if row != self.head_dim * CACHE_BITS[self.format] // 8:
            raise ValueError(f"a {self.format} row of {self.head_dim} values is not {row} bytes")
        if size < 16 or size & (size - 1) or size > 1 << 20:
            raise ValueError("cache page_size must be a power of two from 16")
        if heads < 1:
            raise ValueError("a cache needs at least one key head")
        if self.k_scales.dtype not in _SCALES or self.v_scales.dtype != self.k_scales.dtype:
            raise ValueError("cache scales must be bfloat16 or float8_e8m0fnu")
        expected = (pages, heads, size, self.head_dim // self.block_size)
        if tuple(self.k_scales.shape) != expected or tuple(self.v_scales.shape) != expected:
            raise ValueError(f"cache scales must have shape {expected}")
        if self.k.stride() != self.v.stride() or self.k_scales.stride() != self.v_scales.stride():
            raise ValueError("keys and values of a cache must have the same strides")
        if self.k.stride(3) != 1 or any(s % 16 for s in self.k.stride()[:3]):
            raise ValueError("rows of a cache's codes must be contiguous and start on 16-byte boundaries")
        if self.k_scales.stride(3) != 1 and self.k_scales.shape[3] > 1:
            raise ValueError("rows of a cache's scales must be contiguous")
        if any(getattr(self, name).device != self.k.device for name in ("v", "k_scales", "v_scales")):
            raise ValueError("the cache's tensors must be on one device")

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, format: str = "int8",
              block_size: int | None = None, scale_dtype: torch.dtype = torch.bfloat16, device="cuda",
              order: str = "heads") -> "PackedCache":
        """A cache of ``pages`` pages of zeros; ``block_size`` defaults to the whole head. ``order``: what
        comes first within a page in memory, "heads" (a head's tokens lie side by side) or "tokens"."""
        if order not in ("heads", "tokens"):
            raise ValueError(f"unknown cache order {order!r}")
        if format not in CACHE_FORMATS:
            raise ValueError(f"unknown cache format {format!r}")
        if scale_dtype not in _SCALES:
            raise ValueError("cache scales must be bfloat16 or float8_e8m0fnu")
        block_size = head_dim if block_size is None else block_size
        if block_size < 1 or pages < 0:
            raise ValueError("a cache needs pages >= 0 and block_size >= 1")
        raw = torch.uint8 if scale_dtype == torch.float8_e8m0fnu else scale_dtype

        def zeros(row, dtype):
            if order == "heads":
                return torch.zeros((pages, kv_heads, page_size, row), dtype=dtype, device=device)
            return torch.zeros((pages, page_size, kv_heads, row), dtype=dtype, device=device).transpose(1, 2)

        codes = [zeros(head_dim * CACHE_BITS[format] // 8, torch.uint8) for _ in "kv"]
        scales = [zeros(head_dim // block_size, raw).view(scale_dtype) for _ in "kv"]
        return cls(*codes, *scales, format, head_dim, block_size)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def token_bytes(self) -> int:
        """Bytes of codes and scales that one token takes (keys and values, all heads)."""
        row = self.k.shape[3] + self.k_scales.shape[3] * self.k_scales.element_size()
        return 2 * self.kv_heads * row

    def desc(self):
        """Reference to the C-ABI descriptor (cached: the storage does not move)."""
        cached = self.__dict__.get("_desc")
        if cached is None:
            _require_cuda(self.k, "the cache")
            d = CacheDesc(self.k.data_ptr(), self.v.data_ptr(), self.k_scales.data_ptr(), self.v_scales.data_ptr(),
                          self.pages, self.page_size, self.kv_heads, self.head_dim, self.block_size,
                          CACHE_FORMATS[self.format], _SCALES[self.k_scales.dtype], _I64x3(*self.k.stride()[:3]),
                          _I64x3(*self.k_scales.stride()[:3]))
            cached = (d, ctypes.byref(d))
            object.__setattr__(self, "_desc", cached)
        return cached[1]


def _rows(t: torch.Tensor, name: str, heads: int | None, cache: PackedCache) -> torch.Tensor:
    if t.dim() != 3 or t.shape[2] != cache.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must have shape (tokens, {'heads' if heads is None else heads}, {cache.head_dim})")
    return t if t.stride(2) == 1 else t.contiguous()


def cache_write(cache: PackedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                table: RotaryTable | None = None, positions: torch.Tensor | None = None,
                q: torch.Tensor | None = None) -> torch.Tensor | None:
    """Quantise the keys and values (tokens, kv_heads, head_dim) of new tokens into the cells ``slots``.

    With ``table`` and ``positions`` keys are turned first (in fp32, not rounded in between), and
    ``q`` (tokens, heads, head_dim), when given, comes back turned like ``rotary``'s: one launch for
    all three. k, v and q share one type (float16, bfloat16 or float32) and may be views into one
    projection's rows. ``slots`` (int32 or int64): a negative one stores nothing; one beyond the
    cache stores nothing and sets bit 1 of the device status; no two tokens of a call may share one.
    A NaN makes its block NaN; magnitudes over QMAX * 2^100 are held at that. No gradients."""
    k, v = _rows(k, "k", cache.kv_heads, cache), _rows(v, "v", cache.kv_heads, cache)
    n = k.shape[0]
    if v.shape[0] != n:
        raise ValueError("k and v must hold the same tokens")
    if k.dtype not in _REAL or v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("k, v and q must share a type: float16, bfloat16 or float32")
    if (table is None) != (positions is None):
        raise ValueError("table and positions go together")
    device = cache.k.device
    if device.type != "cuda":
        _require_cuda(cache.k, "the cache")
    if k.device != device or v.device != device:
        raise _elsewhere("k and v", k if k.device != device else v, device)
    slots = _index(slots, "slots", k.shape[:1], device)
    out, q_ptr, out_ptr, heads, qt, qh = None, None, None, 0, 0, 0
    if table is not None:
        if table.device != device:
            raise _elsewhere("table", table, device)
        if table.rotary_dim > cache.head_dim:
            raise ValueError(f"a table of {table.rotary_dim} rotary dimensions does not fit heads of {cache.head_dim}")
        positions = _index(positions, "positions", k.shape[:1], device)
    if q is not None:
        if table is None:
            raise ValueError("q needs table and positions")
        q = _rows(q, "q", None, cache)
        if q.shape[0] != n:
            raise ValueError("q and k must hold the same tokens")
        if q.device != device:
            raise _elsewhere("q", q, device)
        heads = q.shape[1]
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        if heads:
            qt, qh = q.stride()[:2]
            q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
    ks, vs = k.stride(), v.stride()
    if table is None:
        _call("b200_cache_write", device, cache.desc(), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              _REAL[k.dtype], n, slots.data_ptr(), _INDEX[slots.dtype], None, None, 0, None, 0, 0, 0, None)
    else:
        _call("b200_cache_write", device, cache.desc(), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              _REAL[k.dtype], n, slots.data_ptr(), _INDEX[slots.dtype], table._ref, positions.data_ptr(),
              _INDEX[positions.dtype], q_ptr, heads, qt, qh, out_ptr)
    return out


def cache_read(cache: PackedCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """The keys and values (tokens, kv_heads, head_dim) that the cells ``slots`` hold, as ``dtype``.

    Codes times scales in fp32, rounded once. A negative slot reads zeros; one beyond the cache too,
    and sets bit 1 of the device status."""
    if dtype not in _REAL:
        raise ValueError(f"cache_read gives float16, bfloat16 or float32, not {dtype}")
    device = cache.k.device
    if device.type != "cuda":
        _require_cuda(cache.k, "the cache")
    if slots.dim() != 1:
        raise ValueError("slots must be one-dimensional")
    slots = _index(slots, "slots", slots.shape, device)
    n = slots.shape[0]
    both = torch.empty((2, n, cache.k.shape[1], cache.head_dim), dtype=dtype, device=device)
    k, v = both.unbind(0)
    _call("b200_cache_read", device, cache.desc(), slots.data_ptr(), _INDEX[slots.dtype], n, k.data_ptr(), v.data_ptr(),
          _REAL[dtype])
    return k, v


# ---- attention ----------------------------------------------------------------------------------
def cache_attention(q: torch.Tensor, cache: PackedCache, tables: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, prefix: torch.Tensor | None = None, prefix_length: int = 0,
                    return_lse: bool = False, out: torch.Tensor | None = None):
    """Softmax attention of new tokens over what the cache holds of their requests.

    ``q`` (batch, heads, head_dim), one token a request, or (batch, queries, heads, head_dim);
    float16 or bfloat16, any strides with contiguous heads. Head h reads key head
    h // (heads / kv_heads). ``tables`` int32 (batch, max_pages) names each request's pages and
    ``lengths`` int32 (batch) how many tokens they hold, the new ones included: query j of n sees
    keys 0 .. length - n + j. ``scale`` defaults to 1 / sqrt(head_dim).

    ``prefix`` int32 pages and ``prefix_length`` add keys before every request's own that the whole
    batch shares: they are read once and multiplied with all requests' queries together.

    A query that sees no key gives zeros, with a logarithm of -inf. ``return_lse`` also returns the
    natural logarithms of the softmax sums, float32 of q's shape without head_dim; with over 64 query
    rows of a key head over int8 or fp8e4m3 codes with a bfloat16 scale a row, bfloat16 results then
    differ in their last bits from those without (keys' scales stay in fp32). Lengths beyond the
    table count as the table's; a page outside the cache counts as no keys and sets bit 1 of the
    device status. The launch does not depend on the lengths, so it can be recorded in a
    ``GraphStep``. At most 262144 query rows of a key head (queries, or batch * queries for the prefix,
    times heads / kv_heads), 32768 for a head_dim of 256: longer prompts are called in parts. No
    gradients."""
    single = q.dim() == 3
    if q.dim() not in (3, 4) or q.shape[-1] != cache.head_dim:
        raise ValueError(f"q must have shape (batch, [queries,] heads, {cache.head_dim})")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"cache_attention takes float16 or bfloat16 queries, not {q.dtype}")
    batch, queries, heads = q.shape[0], 1 if single else q.shape[1], q.shape[-2]
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"{heads} heads do not share {cache.kv_heads} key heads evenly")
    device = cache.k.device
    if device.type != "cuda":
        _require_cuda(cache.k, "the cache")
    if q.device != device:
        raise _elsewhere("q", q, device)
    if tables.device != device or lengths.device != device:
        raise _elsewhere("tables and lengths", tables if tables.device != device else lengths, device)
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.shape[0] != batch:
        raise ValueError("tables must be int32 (batch, max_pages)")
    if lengths.dtype != torch.int32 or lengths.shape != q.shape[:1]:
        raise ValueError("lengths must be int32 (batch,)")
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    if tables.stride(1) != 1 and tables.shape[1] > 1:
        tables = tables.contiguous()
    if prefix_length < 0 or (prefix_length > 0 and prefix is None):
        raise ValueError("prefix_length needs the prefix's pages")
    if prefix is not None:
        if prefix.device != device:
            raise _elsewhere("prefix", prefix, device)
        if prefix.dtype != torch.int32 or prefix.dim() != 1 or prefix_length > prefix.shape[0] * cache.page_size:
            raise ValueError("prefix must be int32 pages that hold prefix_length tokens")
        if not prefix.is_contiguous():
            prefix = prefix.contiguous()
    if q.stride(-1) != 1:
        q = q.contiguous()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape, type and device")
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=device) if return_lse else None
    if out.numel():
        a = AttentionArgs()
        a.q, a.out, a.tables, a.lengths = q.data_ptr(), out.data_ptr(), tables.data_ptr(), lengths.data_ptr()
        s = q.stride()
        a.q_strides[0], a.q_strides[1], a.q_strides[2] = s[0], 0 if single else s[1], s[-2]
        a.batch, a.queries, a.heads, a.q_dtype = batch, queries, heads, _REAL[q.dtype]
        a.table_stride, a.max_pages = tables.stride(0), tables.shape[1]
        a.scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
        if lse is not None:
            a.lse = lse.data_ptr()
        if prefix_length > 0:
            size = _lib.lib().b200_cache_attention_scratch(batch, queries, heads, cache.head_dim, prefix_length)
            scratch = torch.empty(size, dtype=torch.uint8, device=device)
            a.prefix, a.prefix_pages, a.prefix_length, a.scratch = (prefix.data_ptr(), prefix.shape[0], prefix_length,
                                                                    scratch.data_ptr())
        _call("b200_cache_attention", device, cache.desc(), ctypes.byref(a))
    return (out, lse) if return_lse else out
