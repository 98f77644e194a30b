"""Experts over packed weights: routing of tokens, and the products of 8-bit activations with the weights of
the experts that each token goes to.

    routing = route_experts(logits, k)                              which experts, with what weights
    out     = expert_mlp(x8, gate_up, down, routing, residual=h)    sum of what they give

tinygrad-dx12 has no counterpart: its packed path ends at one matmul (``src/tinygrad_dx12/codegen/
linalg.py:136-223``). Nothing here reads the routing back to the host, so a step with experts can be recorded in a
``GraphStep`` and replayed for any routing. There is no CPU path. No gradients.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _REAL, _call, _elsewhere
from .packed import PackedTensor, _require_cuda
from .scaled import (_E4M3, _RESULTS, BLOCK, ROWS_PAIRS, ROWS_PLAN, ROWS_TOKENS, BlockScaled, _args, _check_bias, _check_product,
                     _check_weights, _flat, _product, _scratch_bytes)

MAX_EXPERTS, MAX_K, MAX_GROUPS = 1024, 32, 32


class RouteArgs(ctypes.Structure):
    """``b200_route_args``."""

    _fields_ = [("logits", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("live", ctypes.c_void_p),
                ("indices", ctypes.c_void_p), ("weights", ctypes.c_void_p), ("offsets", ctypes.c_void_p),
                ("order", ctypes.c_void_p), ("scratch", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("stride", ctypes.c_int64), ("dtype", ctypes.c_int32), ("experts", ctypes.c_int32),
                ("k", ctypes.c_int32), ("sigmoid", ctypes.c_int32), ("groups", ctypes.c_int32),
                ("top_groups", ctypes.c_int32), ("group_best", ctypes.c_int32), ("renormalize", ctypes.c_int32),
                ("scale", ctypes.c_float)]


class CombineArgs(ctypes.Structure):
    """``b200_combine_args``."""

    _fields_ = [("y", ctypes.c_void_p), ("weights", ctypes.c_void_p), ("indices", ctypes.c_void_p), ("residual", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("tokens", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("residual_stride", ctypes.c_int64), ("y_dtype", ctypes.c_int32), ("residual_dtype", ctypes.c_int32),
                ("out_dtype", ctypes.c_int32), ("first", ctypes.c_int32), ("experts", ctypes.c_int32), ("fan", ctypes.c_int32)]


class Routing:
    """Which experts each token goes to, and the order in which the experts read them; ``route_experts`` and
    ``plan_experts`` make them.

    ``indices`` int32 and ``weights`` float32 (tokens, k): a token's experts and what multiplies their results; an
    index outside ``first`` .. ``first + experts - 1`` (such as -1) stands for no expert here. ``rows`` int32
    (tokens * k): pairs token * k + j in the order of their experts, those of expert first + e at
    ``offsets[e]`` .. ``offsets[e + 1]`` (int32, experts + 1 of them). The kernels go by offsets and rows as they find them."""

    __slots__ = ("indices", "weights", "offsets", "rows", "experts", "first")

    def __init__(self):
        raise TypeError("route_experts and plan_experts make routings")

    @classmethod
    def _made(cls, indices, weights, offsets, rows, experts, first=0) -> "Routing":
        r = object.__new__(cls)
        r.indices, r.weights, r.offsets, r.rows, r.experts, r.first = indices, weights, offsets, rows, experts, first
        return r

    @property
    def device(self) -> torch.device:
        return self.indices.device

    @property
    def tokens(self) -> int:
        return self.indices.shape[0]

    @property
    def k(self) -> int:
        return self.indices.shape[1]


def _scratch(pairs: int, experts: int, device):
    """Memory for the plan's counts; None where one CTA makes it."""
    if pairs <= 4096:
        return None
    return torch.empty(_lib.lib().b200_expert_plan_scratch(pairs, experts), dtype=torch.uint8, device=device)


def route_experts(logits: torch.Tensor, k: int, scores: str = "softmax", bias: torch.Tensor | None = None,
                  groups: int = 1, top_groups: int = 1, group_best: int = 1, renormalize: bool = True,
                  scale: float = 1.0, live: torch.Tensor | None = None) -> Routing:
    """The k experts of each token by its ``logits`` (tokens, experts): float16, bfloat16 or float32.

    ``scores``: "softmax" over a token's experts, or "sigmoid" of each logit. Experts are chosen by score + ``bias``
    (float32 (experts,), which balances them and does not reach the weights), best first, ties to the lowest index.
    With ``groups`` > 1 experts fall into that many groups of neighbours; groups are ranked by their best choice,
    or the sum of their best two (``group_best`` 2), and only experts of the ``top_groups`` best can be chosen.
    Scores that decide are compared in 64 bits; without a bias or a sum the logits themselves decide.
    ``weights``: the chosen experts' scores, divided by their sum with ``renormalize``, times ``scale``.

    A logit (or bias) of -inf or NaN keeps its expert from being chosen, larger ones count as the largest finite
    value. Where fewer than k experts can be chosen, and for tokens from ``live`` on (int32 of one element on the
    device, for padded batches), indices are -1 and weights 0. At most 1024 experts, 32 of a token, 32 groups."""
    if logits.dim() != 2 or logits.dtype not in _REAL:
        raise ValueError("logits must be float16, bfloat16 or float32 (tokens, experts)")
    if scores not in ("softmax", "sigmoid"):
        raise ValueError(f"unknown scores {scores!r}")
    tokens, experts = logits.shape
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= k <= min(MAX_K, experts):
        raise ValueError(f"route_experts chooses up to {MAX_K} of up to {MAX_EXPERTS} experts, not {k} of {experts}")
    if not 1 <= groups <= MAX_GROUPS or experts % groups or not 1 <= top_groups <= groups or group_best not in (1, 2):
        raise ValueError(f"{groups} groups, {top_groups} of them by their best {group_best}, do not fit {experts} experts")
    if k > experts // groups * top_groups:
        raise ValueError(f"{top_groups} groups of {experts // groups} experts do not hold {k}")
    device = logits.device
    if device.type != "cuda":
        _require_cuda(logits, "logits")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (experts,):
            raise ValueError(f"bias must be float32 ({experts},)")
        if bias.device != device:
            raise _elsewhere("bias", bias, device)
        bias = bias.contiguous()
    if live is not None:
        if live.dtype != torch.int32 or live.numel() != 1:
            raise ValueError("live must be one int32")
        if live.device != device:
            raise _elsewhere("live", live, device)
    if logits.stride(1) != 1 and experts > 1:
        logits = logits.contiguous()
    indices = torch.empty((tokens, k), dtype=torch.int32, device=device)
    weights = torch.empty((tokens, k), dtype=torch.float32, device=device)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    rows = torch.empty(tokens * k, dtype=torch.int32, device=device)
    scratch = _scratch(tokens * k, experts, device)
    a = RouteArgs(logits.data_ptr(), None if bias is None else bias.data_ptr(), None if live is None else live.data_ptr(),
                  indices.data_ptr(), weights.data_ptr(), offsets.data_ptr(), rows.data_ptr(),
                  None if scratch is None else scratch.data_ptr(), tokens, logits.stride(0), _REAL[logits.dtype], experts, k,
                  int(scores == "sigmoid"), groups, top_groups, group_best, int(renormalize), scale)
    _call("b200_route_experts", device, ctypes.byref(a))
    return Routing._made(indices, weights, offsets, rows, experts)


def plan_experts(indices: torch.Tensor, weights: torch.Tensor, experts: int, first: int = 0) -> Routing:
    """The ``Routing`` of given ``indices`` int32 and ``weights`` float32 (tokens, k), for the experts ``first`` ..
    ``first + experts - 1``: all of a model's, or those that this rank holds. Others' indices stand for no expert here."""
    if indices.dim() != 2 or indices.dtype != torch.int32 or indices.shape[1] < 1:
        raise ValueError("indices must be int32 (tokens, k), k at least 1")
    if weights.shape != indices.shape or weights.dtype != torch.float32:
        raise ValueError("weights must be float32 of indices' shape")
    if not 1 <= experts <= MAX_EXPERTS or first < 0 or first + experts > 1 << 30:
        raise ValueError(f"a plan is of 1 to {MAX_EXPERTS} experts")
    device = indices.device
    if device.type != "cuda":
        _require_cuda(indices, "indices")
    if weights.device != device:
        raise _elsewhere("weights", weights, device)
    indices, weights = indices.contiguous(), weights.contiguous()
    pairs = indices.numel()
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=device)
    rows = torch.empty(pairs, dtype=torch.int32, device=device)
    scratch = _scratch(pairs, experts, device)
    _call("b200_expert_plan", device, indices.data_ptr(), pairs, first, experts, offsets.data_ptr(), rows.data_ptr(),
          None if scratch is None else scratch.data_ptr())
    return Routing._made(indices, weights, offsets, rows, experts, first)


def _check_routing(w: PackedTensor, routing: Routing, what: str) -> None:
    _check_weights(w, 3, what)
    if w.shape[0] != routing.experts:
        raise ValueError(f"weights of {w.shape[0]} experts do not fit a routing over {routing.experts}")
    if routing.indices.device != w.device:
        raise _elsewhere("routing", routing, w.device)


def expert_linear(x: BlockScaled, w: PackedTensor, routing: Routing, bias: torch.Tensor | None = None,
                  activation: str | None = None, gated: bool = False, dtype: torch.dtype = torch.bfloat16,
                  _general: bool = False):
    """``scaled_linear`` of each token with the weights ``w`` (experts, N, K) of each of its experts.

    x (tokens, K), or (tokens * k, K), a row for each pair token * k + j. ``bias`` (experts, N). Gives (tokens * k,
    columns) in the order of the pairs; rows of pairs without an expert are zeros."""
    _check_routing(w, routing, "expert_linear")
    cols = _check_product(x, w, activation, gated, dtype, "expert_linear")
    pairs = routing.indices.numel()
    if len(x.shape) != 2 or x.shape[0] not in (routing.tokens, pairs):
        raise ValueError(f"activations must have {routing.tokens} rows, one a token, or {pairs}, one a pair")
    bias = _check_bias(bias, w.shape[:2], x.device)
    y = BlockScaled._empty((pairs, cols), x.device) if dtype == _E4M3 else torch.empty((pairs, cols), dtype=dtype, device=x.device)
    if pairs and cols:
        _product(x, w, y, pairs, bias, activation, gated, None, routing, ROWS_TOKENS if x.shape[0] == routing.tokens else ROWS_PAIRS,
                 _general)
    return y


def expert_mlp(x: BlockScaled, up: PackedTensor, down: PackedTensor, routing: Routing, activation: str | None = "silu",
               gated: bool = True, up_bias: torch.Tensor | None = None, down_bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16, _general: bool = False) -> torch.Tensor:
    """The weighted sum of what each token's experts give, added to ``residual``:

        out[t] = residual[t] + sum_j weights[t, j] * (act(x[t] Up_e^T) quantised) Down_e^T,   e = indices[t, j]

    x (tokens, K); ``up`` (experts, N, K), with ``gated`` [gate; up] rows; ``down`` (experts, columns, N or N / 2).
    What lies between the two products is held in 8 bits (``quantize``; its width a multiple of 32), their results and the
    sum in fp32 (in the order of a token's experts: the same bits every time). Tokens without an expert give the
    residual, or zeros. ``dtype``: float16, bfloat16 or float32."""
    _check_routing(up, routing, "expert_mlp")
    _check_routing(down, routing, "expert_mlp")
    inner = _check_product(x, up, activation, gated, _E4M3, "expert_mlp")
    tokens, pairs, device = routing.tokens, routing.indices.numel(), x.device
    if tuple(x.shape[:-1]) != (tokens,):
        raise ValueError(f"activations must have {tokens} rows, one a token")
    if down.cols != inner or inner == 0:
        raise ValueError(f"down weights of {down.cols} columns do not fit {inner} values between the products")
    if dtype not in _REAL:
        raise ValueError(f"expert_mlp gives float16, bfloat16 or float32, not {dtype}")
    cols = down.shape[1]
    up_bias = _check_bias(up_bias, up.shape[:2], device, "up_bias")
    down_bias = _check_bias(down_bias, down.shape[:2], device, "down_bias")
    if residual is not None:
        if residual.dtype not in _REAL or tuple(residual.shape) != (tokens, cols):
            raise ValueError(f"residual must be float16, bfloat16 or float32 of shape {(tokens, cols)}")
        if residual.device != device:
            raise _elsewhere("residual", residual, device)
        residual = _flat(residual, tokens, cols)
    out = torch.empty((tokens, cols), dtype=dtype, device=device)
    if not out.numel():
        return out
    # what lies between, in one allocation: the first product's codes and scales, the pairs' results, scratch
    codes, scales, keep = x._pointers()
    f32 = _REAL[torch.float32]
    first = _args(codes, scales, pairs, 0, 0, _RESULTS[_E4M3], up_bias, activation, gated, None, routing, ROWS_TOKENS, ROWS_PLAN, _general)
    second = _args(16, 4, pairs, 0, None, f32, down_bias, None, False, None, routing, ROWS_PLAN, ROWS_PAIRS, _general)
    up_desc, down_desc = up.desc(), down.desc()
    scratch = max(_scratch_bytes(up_desc, first, up), _scratch_bytes(down_desc, second, down))
    at, sizes = 0, (pairs * inner, pairs * inner // BLOCK, pairs * cols * 4, scratch)
    places = []
    for size in sizes:
        places.append(at)
        at += -(-size // 256) * 256
    work = torch.empty(at, dtype=torch.uint8, device=device)
    h, hs, y, spare = (work.data_ptr() + place for place in places)
    first.y, first.y_scales, first.scratch = h, hs, spare
    second.x, second.x_scales, second.y, second.scratch = h, hs, y, spare
    r = residual
    combine = CombineArgs(y, routing.weights.data_ptr(), routing.indices.data_ptr(), None if r is None else r.data_ptr(), out.data_ptr(),
                          tokens, cols, 0 if r is None else r.stride(0), f32, 0 if r is None else _REAL[r.dtype], _REAL[dtype],
                          routing.first, routing.experts, routing.k)
    _call("b200_expert_mlp", device, ctypes.byref(up_desc), ctypes.byref(first), ctypes.byref(down_desc), ctypes.byref(second),
          ctypes.byref(combine))
    return out
