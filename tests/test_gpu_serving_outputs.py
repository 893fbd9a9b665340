"""Given outputs of the serving operators: which memory they may share with the inputs."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


def rows(n, width, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, width, generator=g, device="cuda").bfloat16()


def shared(buf, n, width, x0, w):
    """Outputs of w columns next to the input buf[:n, x0:x0 + width]: (name, out, allowed)."""
    step, at = buf.stride(0), buf.storage_offset() + x0
    return [("the next rows", buf[1:n + 1, x0:x0 + w], False), ("columns on", buf[:n, x0 + 8:x0 + 8 + w], False),
            ("the columns' end", buf.as_strided((n, w), (step, 1), at + width - 8), False),
            ("the next row's first columns", buf.as_strided((n, w), (step, 1), at + step - w + 8), False),
            ("another stride", buf.as_strided((n, w), (step + 64, 1), at), False),
            ("rows of no distance", buf[n:n + 1, :w].expand(n, w), False),
            ("rows that overlap", buf[n:].as_strided((n, w), (w - 8, 1)), False),
            ("the input's own columns", buf[:n, x0:x0 + w], True)]


def test_norm_outputs(ts):
    n, w = 64, 4 * 128
    pos = torch.arange(n, device="cuda")
    inv = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, device="cuda") / 128))
    ang = torch.outer(torch.arange(n, device="cuda").float(), inv)
    qw, rest = rows(1, 128, 1)[0], (pos, ang.cos(), ang.sin())
    want = ts.qk_norm_rope(rows(n, w), 2, 1, qw, qw, *rest)
    for wide in (w + 64, 2 * w + 64):
        for i in range(8):
            buf = torch.zeros(2 * n + 8, wide, device="cuda", dtype=torch.bfloat16)
            x = buf[:n, 8:8 + w]
            x.copy_(rows(n, w))
            name, out, ok = shared(buf, n, w, 8, w)[i]
            before = buf.clone()
            if ok:
                assert torch.equal(ts.qk_norm_rope(x, 2, 1, qw, qw, *rest, out=out), want), name
            else:
                with pytest.raises((RuntimeError, ValueError), match="overlap"):
                    ts.qk_norm_rope(x, 2, 1, qw, qw, *rest, out=out)
                assert torch.equal(buf, before), name
    # beside the input, in its rows or in later ones
    for first in (0, 1):
        buf = torch.zeros(n + 1, 2 * w + 16, device="cuda", dtype=torch.bfloat16)
        x, out = buf[:n, 8:8 + w], buf[first:first + n, 16 + w:16 + 2 * w]
        x.copy_(rows(n, w))
        ts.qk_norm_rope(x, 2, 1, qw, qw, *rest, out=out)
        assert torch.equal(out, want) and torch.equal(x, rows(n, w))


def caches(ts, n):
    """Filled caches of both widths, the same each time."""
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(n, 300, 2, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    out = [ts.PagedKVCache8.allocate(n, 2, 64, 320), ts.PagedKVCache.allocate(n, 2, 64, 320)]
    for c in out:
        ts.paged_append(k, v, c)
        c.advance(300)
    return out


@pytest.mark.parametrize("kind", ["attention", "decode 8", "decode 16"])
def test_attention_outputs(ts, kind):
    n, w = 8, 8 * 64
    width = w if kind == "attention" else w + 4 * 64
    cache = caches(ts, n)[kind == "decode 16"]

    def call(x, out=None):
        # (the same token again: it goes to the same slot, whose block has room for it)
        if kind == "attention":
            return ts.paged_attention(x, cache, out=out)
        return ts.paged_decode_attention(x, 8, cache, out=out)
    x0 = rows(n, width, 5)
    call(x0)
    want = call(x0)
    for wide in (width + 64, 2 * width + 64):
        for i in range(8):
            buf = torch.zeros(2 * n + 8, wide, device="cuda", dtype=torch.bfloat16)
            x = buf[:n, 8:8 + width]
            x.copy_(x0)
            name, out, ok = shared(buf, n, width, 8, w)[i]
            before = buf.clone()
            if ok:
                assert torch.equal(call(x, out), want), name
                assert torch.equal(x[:, w:], x0[:, w:])
            else:
                with pytest.raises((RuntimeError, ValueError), match="overlap"):
                    call(x, out)
                assert torch.equal(buf, before), name
    if kind != "attention":                              # the new token's keys and values are input too
        buf = x0.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            call(buf, buf[:, width - w:])
    buf = torch.zeros(n + 1, width + w + 16, device="cuda", dtype=torch.bfloat16)
    x, out = buf[:n, 8:8 + width], buf[1:, 16 + width:]
    x.copy_(x0)
    call(x, out)
    assert torch.equal(out, want) and torch.equal(x, x0)
    one = torch.zeros(2 * width, device="cuda", dtype=torch.bfloat16)     # one sequence: a row, whatever its stride
    c1 = [ts.PagedKVCache8.allocate(1, 2, 64, 64), ts.PagedKVCache.allocate(1, 2, 64, 64)][kind == "decode 16"]
    cache = c1
    with pytest.raises(RuntimeError, match="overlap"):
        call(one[:width].view(1, -1), one[8:8 + w].view(1, -1))
    call(one[:width].view(1, -1), one[width:width + w].view(1, -1))


@pytest.mark.parametrize("kind", ["attention", "decode 8", "decode 16"])
def test_a_result_that_wants_a_gradient_is_refused(ts, kind):
    cache = caches(ts, 2)[kind == "decode 16"]
    x = rows(2, 8 * 64 if kind == "attention" else 12 * 64)

    def call(out):
        return ts.paged_attention(x, cache, out=out) if kind == "attention" else ts.paged_decode_attention(x, 8, cache, out=out)
    leaf = torch.full((2, 8 * 64), 3.0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="wants a gradient"):
        call(leaf)
    assert (leaf == 3).all()
    with torch.no_grad():
        call(leaf)
        assert not (leaf == 3).any() and torch.equal(leaf, call(None))


@pytest.mark.parametrize("kind", ["attention", "decode 8", "decode 16", "norm and store", "product"])
def test_derivatives_in_forward_mode_are_refused(ts, kind):
    import torch.autograd.forward_ad as fwd
    cache = caches(ts, 2)[kind in ("decode 16", "norm and store")]
    before = [t.clone() for t in cache._args() if t is not None]
    x = rows(2, 8 * 64 if kind == "attention" else 12 * 64)
    w = ts.int8_quantize(rows(16, 12 * 64, 1))
    calls = {"attention": lambda y: ts.paged_attention(y, cache), "product": lambda y: ts.int8_linear(y, w),
             "norm and store": lambda y: ts.qk_norm_rope(y, 8, 2, cache=cache, slots=torch.arange(2, device="cuda"))}
    call = calls.get(kind, lambda y: ts.paged_decode_attention(y, 8, cache))
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        call(fwd.make_dual(x, torch.ones_like(x)))
    assert all(torch.equal(a, b) for a, b in zip(before, [t for t in cache._args() if t is not None]))
