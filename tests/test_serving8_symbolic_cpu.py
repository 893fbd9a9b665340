"""The 8-bit serving operators traced with sizes that change, without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv, StatelessSymbolicContext

import tensorshrink_b200 as ts


@pytest.fixture
def traced():
    """A fake mode, and what makes its tensors: with a changing first size, or of fixed sizes."""
    mode = FakeTensorMode(shape_env=ShapeEnv())

    def changing(t):
        sizes = [DimDynamic.DYNAMIC] + [DimDynamic.STATIC] * (t.dim() - 1)
        return mode.from_tensor(t, symbolic_context=StatelessSymbolicContext(dynamic_sizes=sizes))

    def fixed(*shape, dtype):
        with mode:
            return torch.empty(*shape, dtype=dtype, device="cuda")
    return mode, changing, fixed


def symbolic(n):
    return isinstance(n, torch.SymInt) and n.node.maybe_as_int() is None


def test_tokens_of_a_step(traced):
    """A serving loop's packed tokens: their number goes through reserve, norms, append and product."""
    mode, changing, fixed = traced
    n = changing(torch.empty(37, device="meta")).shape[0]
    assert symbolic(n)
    qkv = fixed(n, 6 * 64, dtype=torch.bfloat16)
    i = lambda *s: fixed(*s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: fixed(*s, dtype=torch.float32)  # noqa: E731
    with mode:
        pages = torch.empty(9, 2, 32, 64, dtype=torch.int8, device="cuda")
        c = ts.PagedKVCache8(pages, pages.clone(), f(9, 2, 2), f(9, 2, 2), i(3, 4), i(3))
        got = ts.paged_reserve(ts.PagePool(i(9), i(1)), c, i(3), n)
        for t in (got.slots, got.positions, got.sequences):
            assert symbolic(t.shape[0]) and t.shape[0].node.expr == n.node.expr
        assert got.granted.shape == (3,) and got.offsets.shape == (4,)
        y = ts.qk_norm_rope(qkv, 2, 2)
        assert y.shape[0].node.expr == n.node.expr
        k, v = y.view(-1, 6, 64).split([2, 2, 2], dim=1)[1:]
        ts.paged_append(k, v, c, offsets=got.offsets)
        w = ts.int8_quantize(fixed(30, 6 * 64, dtype=torch.bfloat16))
        assert ts.int8_linear(y, w).shape[0].node.expr == n.node.expr
    # nothing has pinned the number
    assert not any(type(g.expr).__name__ == "Equality" for g in mode.shape_env.guards), mode.shape_env.guards


def test_bad_numbers_are_refused_when_they_are_known(traced):
    mode, _, fixed = traced
    i = lambda *s: fixed(*s, dtype=torch.int32)  # noqa: E731
    with mode, pytest.raises(ValueError):
        pages = torch.empty(9, 2, 32, 64, dtype=torch.bfloat16, device="cuda")
        c = ts.PagedKVCache(pages, pages.clone(), i(3, 4), i(3))
        ts.paged_reserve(ts.PagePool(i(9), i(1)), c, i(3), -1)
