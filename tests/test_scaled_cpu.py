"""8-bit activations and experts without a GPU: what the host side refuses, and the C entries' checks."""

import ctypes

import pytest
import torch

import tinygrad_dx12_b200 as tg
from tinygrad_dx12_b200 import _lib, experts as E, scaled as SC

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def rows(*shape):
    return tg.BlockScaled(torch.zeros(shape, dtype=torch.uint8).view(E4M3),
                          torch.full((*shape[:-1], shape[-1] // 32), 127, dtype=torch.uint8).view(E8M0))


def weights(*shape, fmt="fp4_e2m1", scales=E8M0, block=32):
    n = 1
    for s in shape:
        n *= s
    s = torch.ones((*shape[:-1], -(-shape[-1] // block)))
    s = None if scales is None else torch.full(s.shape, 127, dtype=torch.uint8).view(E8M0) if scales == E8M0 else s.to(scales)
    return tg.PackedTensor(torch.zeros(n * SC_BITS[fmt] // 8, dtype=torch.uint8), fmt, shape, s, block)


SC_BITS = {"fp4_e2m1": 4, "fp6_e2m3": 6, "fp6_e3m2": 6, "int4": 4}


def test_block_scaled_shapes():
    x = rows(3, 64)
    assert x.shape == (3, 64) and x.device.type == "cpu" and "3, 64" in repr(x)
    x = tg.BlockScaled._empty((2, 5, 96), "cpu")
    assert x.codes.shape == (2, 5, 96) and x.codes.dtype == E4M3 and x.scales.shape == (2, 5, 3) and x.scales.dtype == E8M0
    assert x.scales.data_ptr() == x.codes.data_ptr() + 2 * 5 * 96
    assert tg.BlockScaled._empty((0, 64), "cpu").scales.shape == (0, 2)


@pytest.mark.parametrize("codes,scales,msg", [
    (torch.zeros(2, 64), torch.zeros(2, 2), "float8"),
    (torch.zeros(2, 48, dtype=torch.uint8).view(E4M3), torch.zeros(2, 1, dtype=torch.uint8).view(E8M0), "blocks"),
    (torch.zeros(2, 64, dtype=torch.uint8).view(E4M3), torch.zeros(2, 3, dtype=torch.uint8).view(E8M0), "shape"),
])
def test_block_scaled_refusals(codes, scales, msg):
    with pytest.raises(ValueError, match=msg):
        tg.BlockScaled(codes, scales)


def test_no_cpu_path():
    for call in (lambda: tg.quantize(torch.zeros(2, 64)), lambda: tg.rms_norm(torch.zeros(2, 64)), lambda: rows(2, 64).values(),
                 lambda: tg.scaled_linear(rows(2, 128), weights(4, 128)), lambda: tg.route_experts(torch.zeros(2, 8), 2),
                 lambda: tg.plan_experts(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2), 4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("call,msg", [
    (lambda: tg.quantize(torch.zeros(2, 64, dtype=torch.int32)), "float16"),
    (lambda: tg.quantize(torch.zeros(2, 40)), "blocks"),
    (lambda: tg.rms_norm(torch.zeros(2, 40), dtype=E4M3), "blocks"),
    (lambda: tg.rms_norm(torch.zeros(2, 64), dtype=torch.float64), "rms_norm gives"),
    (lambda: tg.rms_norm(torch.zeros(2, 64, dtype=torch.float64)), "rms_norm takes"),
    (lambda: rows(2, 64).values(torch.int8), "values are"),
    (lambda: tg.route_experts(torch.zeros(8), 2), "tokens, experts"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 9), "chooses up to"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 0), "chooses up to"),
    (lambda: tg.route_experts(torch.zeros(2, 64), 33), "chooses up to"),
    (lambda: tg.route_experts(torch.zeros(2, 2048), 2), "chooses up to"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 2, scores="relu"), "unknown scores"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 2, groups=3), "groups"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 2, groups=4, top_groups=5), "groups"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 2, groups=4, group_best=3), "groups"),
    (lambda: tg.route_experts(torch.zeros(2, 8), 3, groups=4, top_groups=1), "do not hold"),
    (lambda: tg.plan_experts(torch.zeros(4, dtype=torch.int32), torch.zeros(4), 4), "tokens, k"),
    (lambda: tg.plan_experts(torch.zeros(4, 0, dtype=torch.int32), torch.zeros(4, 0), 4), "at least 1"),
    (lambda: tg.plan_experts(torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1), 4), "int32"),
    (lambda: tg.plan_experts(torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 2), 4), "weights"),
    (lambda: tg.plan_experts(torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1), 0), "1 to"),
    (lambda: tg.plan_experts(torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, 1), 4, first=-1), "1 to"),
])
def test_refusals(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()


def test_routings_are_made_by_their_functions():
    with pytest.raises(TypeError, match="plan_experts"):
        tg.Routing()


@pytest.mark.parametrize("w,msg", [
    (lambda: weights(4, 128, fmt="int4"), "FP4 or FP6"),
    (lambda: weights(4, 128, scales=None), "scales"),
    (lambda: weights(4, 128, scales=torch.float16), "scales"),
    (lambda: weights(4, 128, block=64), "scales"),
    (lambda: weights(2, 4, 128), "2 dimensions"),
])
def test_weight_refusals(w, msg):
    with pytest.raises(ValueError, match=msg):
        SC._check_weights(w(), 2, "scaled_linear")


@pytest.mark.parametrize("kw,msg", [
    (dict(x=torch.zeros(2, 128)), "BlockScaled"),
    (dict(x=rows(2, 64)), "do not fit"),
    (dict(activation="tanh"), "unknown activation"),
    (dict(dtype=torch.float64), "gives"),
    (dict(w=weights(5, 128), gated=True), "as many gate rows"),
    (dict(w=weights(48, 128), dtype=E4M3), "blocks"),
    (dict(w=weights(96, 128), gated=True, dtype=E4M3), "blocks"),
])
def test_product_refusals(kw, msg):
    a = {**dict(x=rows(2, 128), w=weights(64, 128), activation=None, gated=False, dtype=torch.bfloat16), **kw}
    with pytest.raises(ValueError, match=msg):
        SC._check_product(a["x"], a["w"], a["activation"], a["gated"], a["dtype"], "scaled_linear")


def test_bias_refusals():
    for bias in (torch.zeros(3), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="bias"):
            SC._check_bias(bias, (4,), torch.device("cpu"))
    assert SC._check_bias(torch.zeros(4, 2)[:, 0], (4,), torch.device("cpu")).is_contiguous()


def desc(**kw):
    d = _lib.PackedDesc()
    d.data, d.data_bytes, d.format, d.scale_dtype, d.rows, d.cols, d.block_size, d.scales = 4096, 1 << 20, 2, 16, 64, 128, 32, 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def args(**kw):
    a = SC.ScaledArgs(4096, 4096, 2, None, None, 0, 4096, 4096, None, None, None, 0, 0, 0, 0, 0, 0, _lib.DT["bfloat16"], 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("d,a,code,msg", [
    ({}, dict(rows=-1), _lib.ERR_INVALID, "out of range"),
    ({}, dict(experts=3), _lib.ERR_INVALID, "equal rows"),
    ({}, dict(experts=2, fan=0), _lib.ERR_INVALID, "fan"),
    ({}, dict(experts=2, fan=1, residual=4096), _lib.ERR_INVALID, "no residual"),
    ({}, dict(experts=2, fan=1, x_rows=3), _lib.ERR_INVALID, "kind of rows"),
    ({}, dict(experts=2, fan=1, y_rows=0), _lib.ERR_INVALID, "kind of rows"),
    ({}, dict(experts=2048, fan=1), _lib.ERR_INVALID, "out of range"),
    ({}, dict(activation=9), _lib.ERR_INVALID, "activation"),
    (dict(rows=63), dict(gated=1), _lib.ERR_INVALID, "odd"),
    ({}, dict(y_dtype=_lib.DT["float64"]), _lib.ERR_INVALID, "float16"),
    (dict(rows=48), dict(y_dtype=_lib.DT["fp8e4m3"]), _lib.ERR_INVALID, "whole blocks"),
    ({}, dict(x=None), _lib.ERR_INVALID, "null"),
    ({}, dict(y=4097), _lib.ERR_INVALID, "boundary"),
    ({}, dict(bias=4097, bias_dtype=_lib.DT["float32"]), _lib.ERR_INVALID, "boundary"),
    ({}, dict(general=1), _lib.ERR_INVALID, "scratch"),
    (dict(format=0), {}, _lib.ERR_UNSUPPORTED, "FP4 or FP6"),
    (dict(block_size=64), {}, _lib.ERR_UNSUPPORTED, "blocks of 32"),
    (dict(scale_dtype=12), {}, _lib.ERR_UNSUPPORTED, "E8M0"),
    (dict(data_bytes=9), {}, _lib.ERR_INVALID, "smaller"),
])
def test_c_checks_of_products(d, a, code, msg):
    rc = _lib.lib().b200_scaled_linear(ctypes.byref(desc(**d)), ctypes.byref(args(**a)), None)
    assert rc == code and msg in _lib.last_error()


def test_c_scratch():
    size = lambda d, a: _lib.lib().b200_scaled_linear_scratch(ctypes.byref(d), ctypes.byref(a))  # noqa: E731
    assert size(desc(), args()) == 0 and size(desc(), args(general=1)) == 2 * 64 * 4
    assert size(desc(cols=96), args()) == 2 * 64 * 4 and size(desc(data=4112), args()) == 2 * 64 * 4
    assert size(desc(), args(experts=2, fan=1, x_rows=0, y_rows=1)) == 2 * 128  # two tokens' rows in the plan's order
    assert size(desc(), args(experts=2, fan=2, x_rows=0, y_rows=1)) == 0        # one token's
    assert size(desc(), args(experts=2, fan=1, x_rows=2, y_rows=1)) == 0
    assert _lib.lib().b200_expert_plan_scratch(100, 8) == 0 and _lib.lib().b200_expert_plan_scratch(100000, 8) > 0


def test_c_checks_of_routing_and_norms():
    lib = _lib.lib()
    assert lib.b200_route_experts(None, None) == _lib.ERR_INVALID
    a = E.RouteArgs(4096, None, None, 4096, 4096, 4096, 4096, None, 2, 8, _lib.DT["float32"], 8, 2, 0, 1, 1, 1, 1, 1.0)
    for k, v in (("experts", 2000), ("k", 0), ("k", 9), ("groups", 3), ("top_groups", 2), ("group_best", 3), ("dtype", 9), ("rows", -1)):
        b = E.RouteArgs.from_buffer_copy(a)
        setattr(b, k, v)
        assert lib.b200_route_experts(ctypes.byref(b), None) == _lib.ERR_INVALID, k
    assert lib.b200_expert_plan(4096, 4, 0, 2000, 4096, 4096, None, None) == _lib.ERR_INVALID
    assert lib.b200_expert_plan(4096, 1 << 20, 0, 8, 4096, 4096, None, None) == _lib.ERR_INVALID  # without scratch
    n = SC.NormArgs(4096, None, None, None, 4096, 4096, 2, 40, 40, 0, 0, _lib.DT["float32"], 0, 0, _lib.DT["fp8e4m3"], 1, 1e-6)
    assert lib.b200_rms_norm(ctypes.byref(n), None) == _lib.ERR_INVALID and "blocks of 32" in _lib.last_error()
    assert lib.b200_scaled_values(4096, 4096, 2, 40, 4096, _lib.DT["float32"], None) == _lib.ERR_INVALID
    assert lib.b200_expert_combine(None, None) == _lib.ERR_INVALID


def test_injected_failures_reach_the_new_entries():
    lib = _lib.lib()
    for call in (lambda: lib.b200_scaled_linear(None, None, None), lambda: lib.b200_rms_norm(None, None), lambda: lib.b200_route_experts(None, None)):
        lib.b200_inject_failure(1, _lib.ERR_INJECTED)
        assert call() == _lib.ERR_INJECTED
    lib.b200_inject_failure(0, 0)
