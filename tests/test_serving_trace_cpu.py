"""The serving operators under tracing, without a GPU: fake tensors get shapes
and types and never reach the launch code, and the schemas say what is written."""

from __future__ import annotations

import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import tensorshrink_b200 as ts
from tensorshrink_b200 import _C, fp4

DEVICE = "cuda"


@pytest.fixture
def fake():
    """Fake CUDA tensors; a kernel that touches their memory warns, which is an error here."""
    with warnings.catch_warnings(), FakeTensorMode() as mode:
        warnings.simplefilter("error")
        yield mode


def weight(n, k, fmt, device=DEVICE):
    g = torch.ones(1, device=device) if fmt == "nvfp4" else None
    codes = torch.empty(n, fp4.padded_cols(k) // 2, dtype=torch.uint8, device=device)
    scales = torch.empty(fp4.scales_nbytes(n, k, fmt), dtype=torch.uint8, device=device)
    return ts.Fp4Tensor(codes, scales, g, n, k, fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 64), (129, 200), (300, 4099)])
def test_quantise_and_back(fake, fmt, rows, cols):
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEVICE)
    t = ts.fp4_quantize(x, fmt)
    assert t.codes.shape == (rows, fp4.padded_cols(cols) // 2) and t.codes.dtype == torch.uint8
    assert t.scales.shape == (fp4.scales_nbytes(rows, cols, fmt),)
    assert (t.global_scale is not None) == (fmt == "nvfp4")
    y = ts.fp4_dequantize(t, torch.float16)
    assert y.shape == x.shape and y.dtype == torch.float16 and y.device.type == "cuda"
    if fmt == "nvfp4":
        g = torch.ones(1, device=DEVICE)
        assert ts.fp4_quantize(x, fmt, global_scale=g).global_scale is g


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_products(fake, fmt):
    w = weight(300, 520, fmt)
    for shape in ((520,), (1, 520), (40, 520), (2, 5, 520)):
        x = torch.empty(shape, dtype=torch.float16, device=DEVICE)
        y = ts.fp4_linear(x, w, bias=torch.empty(300, device=DEVICE))
        assert y.shape == (*shape[:-1], 300) and y.dtype == torch.float16 and y.device.type == "cuda"
        assert ts.fp4_linear(x, w, out_dtype=torch.float32).dtype == torch.float32
    a = weight(7, 520, fmt)
    y = ts.fp4_matmul(a, w)
    assert y.shape == (7, 300) and y.dtype == torch.bfloat16
    with pytest.raises(ValueError):
        ts.fp4_linear(torch.empty(4, 519, device=DEVICE), w)


def test_module_traces_to_one_operator(fake):
    from torch.fx.experimental.proxy_tensor import make_fx
    layer = ts.Fp4Linear(weight(128, 256, "nvfp4"), torch.empty(128, device=DEVICE))
    graph = make_fx(layer)(torch.empty(3, 256, dtype=torch.bfloat16, device=DEVICE))
    calls = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    assert calls == [torch.ops.tensorshrink.fp4_linear.default]


def test_dynamic_token_counts():
    from torch.fx.experimental.proxy_tensor import make_fx
    w = weight(128, 256, "mxfp4", "meta")
    x = torch.empty(9, 256, dtype=torch.bfloat16, device="meta")
    graph = make_fx(lambda x: ts.fp4_linear(x, w), tracing_mode="symbolic", _allow_non_fake_inputs=True)(x)
    out = next(n for n in graph.graph.nodes if n.op == "output").args[0]
    assert not isinstance(out.meta["val"].shape[0], int) and out.meta["val"].shape[1] == 128


@pytest.mark.parametrize("track", [False, True])
def test_cache(fake, track):
    c = ts.PagedKVCache.allocate(3, 2, 64, 100, 16, device=DEVICE, track=track)
    pos = torch.zeros(3, dtype=torch.int64, device=DEVICE)
    cos, sin = torch.empty(200, 32, device=DEVICE), torch.empty(200, 32, device=DEVICE)
    kv = torch.empty(3, 9, 2, 64, dtype=torch.bfloat16, device=DEVICE)
    assert ts.paged_append(kv, kv, c, pos, cos, sin) is None
    qkv = torch.empty(3, 12 * 64, dtype=torch.bfloat16, device=DEVICE)
    y = ts.paged_decode_attention(qkv, 8, c, pos, cos, sin, accumulate=track)
    assert y.shape == (3, 8 * 64) and y.dtype == torch.bfloat16 and y.device.type == "cuda"
    out = torch.empty(3, 8 * 64, dtype=torch.bfloat16, device=DEVICE)
    assert ts.paged_decode_attention(qkv, 8, c, pos, cos, sin, out=out) is out
    if track:
        assert ts.paged_evict(c, 50, 4) is None
    else:
        with pytest.raises(ValueError):
            ts.paged_evict(c, 50, 4)


def test_schemas_name_what_is_written_and_returned():
    ops = _C.serving_ops()

    def written(overload):
        return {a.name for a in overload._schema.arguments if a.alias_info is not None and a.alias_info.is_write}
    pool = {"k_pages", "v_pages", "scores", "slot_pos"}
    assert written(ops.paged_append.default) == pool
    assert written(ops.paged_decode_attention.default) == pool
    assert written(ops.paged_decode_attention.out) == pool | {"out"}
    assert written(ops.paged_evict.default) == pool | {"seq_lens"}
    assert ops.paged_decode_attention.out._schema.returns[0].alias_info.is_write
    for op in (ops.fp4_quantize, ops.fp4_dequantize, ops.fp4_matmul, ops.fp4_linear, ops.paged_decode_attention):
        assert all(r.alias_info is None for r in op.default._schema.returns)


def test_the_cpu_is_refused_by_name():
    x = torch.randn(4, 64)
    for call in (lambda: ts.fp4_quantize(x), lambda: _C.serving_ops().paged_evict(
            torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, dtype=torch.int32),
            torch.zeros(1, dtype=torch.int32), None, None, 4, 0)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def differentiable():
    """Calls on tensors without memory whose results depend on something that wants a gradient."""
    x = torch.randn(4, 256, device="meta", requires_grad=True)
    bias = torch.randn(128, device="meta", requires_grad=True)
    w, g = weight(128, 256, "nvfp4", "meta"), torch.ones(1, device="meta", requires_grad=True)
    a = ts.Fp4Tensor(w.codes, w.scales, g, 128, 256, "nvfp4")
    c = ts.PagedKVCache.allocate(2, 2, 64, 32, 16, device="meta", dtype=torch.float16)
    qkv = torch.randn(2, 8 * 64, device="meta", dtype=torch.float16, requires_grad=True)
    return {"x": lambda: ts.fp4_linear(x, w), "bias": lambda: ts.fp4_linear(x.detach(), w, bias=bias),
            "input_scale": lambda: ts.fp4_linear(x.detach(), w, input_scale=g), "matmul": lambda: ts.fp4_matmul(a, w),
            "dequantize": lambda: ts.fp4_dequantize(a), "attention": lambda: ts.paged_decode_attention(qkv, 4, c)}


@pytest.mark.parametrize("name", ["x", "bias", "input_scale", "matmul", "dequantize", "attention"])
def test_a_backward_pass_is_refused(name):
    call = differentiable()[name]
    with torch.no_grad():
        assert not call().requires_grad
    with pytest.raises(RuntimeError, match="derivative for tensorshrink::.* is not implemented"):
        call().sum().backward()


def test_nothing_else_gets_a_history():
    x = torch.randn(4, 256, device="meta", requires_grad=True)
    t = ts.fp4_quantize(x)
    assert not t.global_scale.requires_grad and not ts.fp4_dequantize(t).requires_grad
    assert not ts.fp4_linear(x.detach(), t).requires_grad
    c = ts.PagedKVCache.allocate(2, 2, 64, 32, 16, device="meta", dtype=torch.float16)
    kv = torch.randn(2, 3, 2, 64, device="meta", dtype=torch.float16, requires_grad=True)
    ts.paged_append(kv, kv, c)
    qkv = torch.randn(2, 8 * 64, device="meta", dtype=torch.float16, requires_grad=True)
    out = torch.empty(2, 256, device="meta", dtype=torch.float16)
    ts.paged_decode_attention(qkv, 4, c, out=out)
    assert not (c.k_pages.requires_grad or c.v_pages.requires_grad or out.requires_grad)


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: torch.nn.Sequential(m).to(torch.float16)[0],
                                  lambda m: m.bfloat16().float()])
def test_a_cast_module_keeps_its_scales(cast):
    """Values that bf16 and fp16 would round."""
    w = weight(128, 256, "nvfp4", "meta")
    with torch.device("meta"):
        layer = ts.Fp4Linear(w, torch.randn(128))
    layer.global_scale, layer.input_scale = torch.full((1,), 1.0001e-9), torch.full((1,), 0.0100001)
    want = [layer.global_scale.clone(), layer.input_scale.clone()]
    layer = cast(layer)
    assert torch.equal(layer.global_scale, want[0]) and torch.equal(layer.input_scale, want[1])
    assert layer.codes.dtype == torch.uint8 and layer.scales.dtype == torch.uint8
    assert {"global_scale", "input_scale"} <= set(layer.state_dict())


def test_a_cast_module_runs_and_moves(fake):
    layer = ts.Fp4Linear(weight(128, 256, "nvfp4"), torch.empty(128, device=DEVICE)).to(torch.bfloat16)
    x = torch.empty(3, 256, dtype=torch.bfloat16, device=DEVICE)
    assert layer(x).shape == (3, 128) and layer.bias.dtype == torch.bfloat16
    moved = layer.to("cpu", torch.float16)
    assert moved.global_scale.device.type == "cpu" and moved.global_scale.dtype == torch.float32
    mx = ts.Fp4Linear(weight(128, 256, "mxfp4")).half()
    assert mx.global_scale is None and mx(x).shape == (3, 128)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_calibration_takes_finite_samples(bad):
    layer = ts.Fp4Linear(weight(128, 256, "nvfp4", "meta"))
    layer.input_scale = torch.ones(1)
    x = torch.linspace(-3, 2, 512).view(2, 256)
    x[0, 5] = bad
    layer.calibrate(x)
    assert layer.input_scale.item() == (torch.tensor(3.0) / 2688.0).item()
    layer.calibrate(torch.full((1, 256), bad))
    assert layer.input_scale.item() == 2.0 ** -100
