"""Gradients that the serving operators do not compute, on tensors without memory."""

from __future__ import annotations

import pytest
import torch

import tensorshrink_b200 as ts


def meta(*shape, dtype=torch.float16):
    return torch.randn(*shape, device="meta").to(dtype)


def cache8():
    i = {"dtype": torch.int32, "device": "meta"}
    pages = torch.empty(8, 2, 32, 64, device="meta", dtype=torch.int8)
    # (without memory there is nothing to check the pages by)
    c = ts.PagedKVCache8.__new__(ts.PagedKVCache8)
    c.k_pages, c.v_pages, c.k_scales, c.v_scales = pages, pages.clone(), meta(8, 2, 2, dtype=torch.float32), \
        meta(8, 2, 2, dtype=torch.float32)
    c.page_table, c.seq_lens = torch.empty(2, 4, **i), torch.empty(2, **i)
    return c


def outputs():
    """Calls that write into a given result: name -> (call, its result's columns)."""
    q, qkv, c16 = meta(2, 4 * 64), meta(2, 8 * 64), ts.PagedKVCache.allocate(2, 2, 64, 32, 16, device="meta", dtype=torch.float16)
    slots = torch.zeros(2, dtype=torch.int64, device="meta")
    return {"attention": (lambda out: ts.paged_attention(q, cache8(), out=out), 256),
            "decode 8": (lambda out: ts.paged_decode_attention(qkv, 4, cache8(), out=out), 256),
            "decode 16": (lambda out: ts.paged_decode_attention(qkv, 4, c16, out=out), 256),
            "norm": (lambda out: ts.qk_norm_rope(qkv, 4, 2, out=out), 512),
            "norm and store": (lambda out: ts.qk_norm_rope(qkv, 4, 2, out=out, cache=c16, slots=slots), 512)}


@pytest.mark.parametrize("name", ["attention", "decode 8", "decode 16", "norm", "norm and store"])
def test_a_given_result_that_wants_a_gradient_is_refused(name):
    call, width = outputs()[name]
    leaf = meta(2, width).requires_grad_()
    with pytest.raises(RuntimeError, match="wants a gradient"):
        call(leaf)
    with torch.no_grad():
        assert call(leaf) is leaf
    assert not call(meta(2, width)).requires_grad


def differentiable(of):
    """Calls whose results depend on something that has a derivative, made by `of` from a tensor without memory."""
    x, qkv, q = meta(4, 256), meta(2, 8 * 64), meta(2, 4 * 64)
    codes, scales, bias = torch.empty(32, 256, device="meta", dtype=torch.int8), meta(32, dtype=torch.float32), meta(32)
    i = {"dtype": torch.uint8, "device": "meta"}
    c16 = ts.PagedKVCache.allocate(2, 2, 64, 32, 16, device="meta", dtype=torch.float16)
    f4 = ts.Fp4Tensor(torch.empty(128, 128, **i), torch.empty(128 * 16, **i), None, 128, 256, "nvfp4")
    norm = meta(64, dtype=torch.float32)
    slots = torch.zeros(2, dtype=torch.int64, device="meta")

    def int8(s):
        t = ts.Int8Tensor.__new__(ts.Int8Tensor)
        t.codes, t.scales, t.cols = codes, s, 256
        return t
    return {"int8_linear": lambda: ts.int8_linear(of(x), int8(scales)), "int8 scales": lambda: ts.int8_linear(x, int8(of(scales))),
            "int8 bias": lambda: ts.int8_linear(x, int8(scales), of(bias)),
            "int8_matmul": lambda: ts.int8_matmul(int8(scales), int8(of(scales))),
            "int8_dequantize": lambda: ts.int8_dequantize(int8(of(scales))),
            "norm": lambda: ts.qk_norm_rope(of(qkv), 4, 2), "norm's weight": lambda: ts.qk_norm_rope(qkv, 4, 2, of(norm), norm),
            "norm and store": lambda: ts.qk_norm_rope(of(qkv), 4, 2, cache=c16, slots=slots),
            "attention 8": lambda: ts.paged_attention(of(q), cache8()),
            "decode 8": lambda: ts.paged_decode_attention(of(qkv), 4, cache8()),
            "decode 16": lambda: ts.paged_decode_attention(of(qkv), 4, c16), "fp4_linear": lambda: ts.fp4_linear(of(x), f4)}


NAMES = list(differentiable(lambda t: t))


@pytest.mark.parametrize("name", NAMES)
def test_a_derivative_in_forward_mode_is_refused(name):
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        call = differentiable(lambda t: fwd.make_dual(t, torch.ones_like(t)))[name]
        with pytest.raises(NotImplementedError, match="forward mode"):
            call()
        with pytest.raises(NotImplementedError, match="forward mode"), torch.no_grad():
            call()
        with fwd._set_fwd_grad_enabled(False):
            call()
        differentiable(lambda t: t)[name]()
    out = {"attention 8": 256, "decode 8": 256, "decode 16": 256, "norm": 512, "norm and store": 512}.get(name)
    if out is not None:
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
            outputs()[name.replace("attention 8", "attention")][0](fwd.make_dual(meta(2, out), meta(2, out)))


@pytest.mark.parametrize("name", NAMES)
def test_a_backward_pass_is_refused(name):
    call = differentiable(lambda t: t.requires_grad_())[name]
    with torch.no_grad():
        assert not call().requires_grad
    with pytest.raises(RuntimeError, match="derivative for tensorshrink::.* is not implemented"):
        call().float().sum().backward()


def test_a_quantised_tensor_has_no_history():
    t = ts.int8_quantize(meta(4, 256).requires_grad_())
    assert not t.scales.requires_grad and not ts.int8_dequantize(t).requires_grad
