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
