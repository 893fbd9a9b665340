"""Norms of queries and keys with their rotation, against 64 bits.

Tolerance of a value y = a c - b s (or a s + b c) in type T: the rounding to T
is half a step, eps / 2 |y| (and half of T's smallest step); the norm's sum of up to 256
squares (a chain of 16, then a tree of 4), its root and the products are fp32, 2^-20
of |a| + |b| together. Values (and everything without norm and rotation) are copied exactly.
"""

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


def tables(n, d):
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
    ang = torch.outer(torch.arange(n, device="cuda", dtype=torch.float32), inv)
    return ang.cos().contiguous(), ang.sin().contiguous()


def make(tokens, n_q, n_kv, d, dtype, seed, wdtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, n_q + 2 * n_kv, d, generator=g, device="cuda")
    x *= torch.exp(torch.randn(1, n_q + 2 * n_kv, 1, generator=g, device="cuda"))
    w = (1 + 0.3 * torch.randn(2, d, generator=g, device="cuda")).to(wdtype)
    return x.to(dtype).view(tokens, -1), w[0].clone(), w[1].clone(), torch.randint(0, 50, (tokens,), generator=g, device="cuda")


def expected(x, n_q, n_kv, qw, kw, pos, cos, sin, eps):
    """(values, tolerance) in 64 bits."""
    t = x.shape[0]
    y = x.double().view(t, n_q + 2 * n_kv, -1).clone()
    d = y.shape[-1]
    for lo, hi, w in ((0, n_q, qw), (n_q, n_q + n_kv, kw)):
        if w is not None:
            y[:, lo:hi] = y[:, lo:hi] / torch.sqrt(y[:, lo:hi].square().mean(-1, keepdim=True) + eps) * w.double()
    tol = torch.zeros_like(y)
    qk = y[:, :n_q + n_kv]
    if cos is not None:
        a, b = qk[..., :d // 2].clone(), qk[..., d // 2:].clone()
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        size = (a.abs() + b.abs()) * 2.0 ** -20
        y[:, :n_q + n_kv] = torch.cat([a * c - b * s, a * s + b * c], -1)
        tol[:, :n_q + n_kv] = torch.cat([size, size], -1)
    else:
        tol[:, :n_q + n_kv] = qk.abs() * 2.0 ** -20
    if qw is None and cos is None:
        tol[:, :n_q] = 0
    if kw is None and cos is None:
        tol[:, n_q:n_q + n_kv] = 0
    fi = torch.finfo(x.dtype)
    tol[:, :n_q + n_kv] += (tol[:, :n_q + n_kv] > 0) * (y[:, :n_q + n_kv].abs() * (fi.eps / 2) + fi.smallest_normal * fi.eps / 2)
    return y.view(t, -1), tol.view(t, -1)


def close(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,n_q,n_kv,d", [(1, 32, 8, 128), (1, 1, 1, 16), (3, 7, 1, 96), (5, 4, 2, 64), (33, 6, 3, 80), (9, 5, 5, 32),
                                               (2, 16, 2, 256), (700, 32, 8, 128), (2049, 14, 2, 64), (257, 3, 3, 160)])
def test_norm_and_rotation(ts, tokens, n_q, n_kv, d, dtype):
    x, qw, kw, pos = make(tokens, n_q, n_kv, d, dtype, tokens)
    cos, sin = tables(50, d)
    for a, b in ((qw, kw), (qw, None), (None, kw), (None, None)):
        for turn in (True, False):
            args = (pos, cos, sin) if turn else (None, None, None)
            got = ts.qk_norm_rope(x, n_q, n_kv, a, b, *args, eps=1e-5)
            want, tol = expected(x, n_q, n_kv, a, b, *args, 1e-5)
            close(got, want, tol)
            assert torch.equal(got[:, (n_q + n_kv) * d:], x[:, (n_q + n_kv) * d:])
            y = x.clone()                                        # the same in place
            assert ts.qk_norm_rope(y, n_q, n_kv, a, b, *args, eps=1e-5, out=y) is y
            assert torch.equal(y, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_of_the_same_type_and_strided_rows(ts, dtype):
    n_q, n_kv, d = 4, 2, 64
    x, qw, kw, pos = make(21, n_q, n_kv, d, dtype, 3, wdtype=dtype)
    cos, sin = tables(50, d)
    wide = torch.zeros(21, x.shape[1] + 24, dtype=dtype, device="cuda")
    for at in (8, 3):                                            # rows on 16 bytes, and not
        v = wide[:, at:at + x.shape[1]]
        v.copy_(x)
        got = ts.qk_norm_rope(v, n_q, n_kv, qw, kw, pos, cos, sin)
        close(got, *expected(x, n_q, n_kv, qw, kw, pos, cos, sin, 1e-6))
    out = torch.full_like(wide, 5.0)
    ts.qk_norm_rope(x, n_q, n_kv, qw, kw, pos, cos, sin, out=out[:, 16:16 + x.shape[1]])
    assert torch.equal(out[:, 16:16 + x.shape[1]], got) and (out[:, :16] == 5).all() and (out[:, 16 + x.shape[1]:] == 5).all()


def test_rotation_alone_equals_that_of_the_cache(ts):
    x, _, _, pos = make(40, 4, 2, 128, torch.bfloat16, 7)
    cos, sin = tables(50, 128)
    got = ts.qk_norm_rope(x, 4, 2, None, None, pos, cos, sin)
    k = x.view(40, 8, 128)[:, 4:6]
    a, b = k.float().chunk(2, -1)
    c, s = cos[pos][:, None], sin[pos][:, None]
    assert torch.equal(got.view(40, 8, 128)[:, 4:6], torch.cat([a * c - b * s, a * s + b * c], -1).to(torch.bfloat16))


@pytest.mark.parametrize("page,track", [(16, False), (64, True), (24, True)])
def test_store(ts, page, track):
    n_q, n_kv, d, tokens = 6, 2, 96, 300
    x, qw, kw, pos = make(tokens, n_q, n_kv, d, torch.float16, 9)
    cos, sin = tables(50, d)
    pages = tokens // page + 4
    for layout in ("heads", "tokens"):
        shape = (pages, n_kv, page, d) if layout == "heads" else (pages, page, n_kv, d)
        k, v = torch.randn(2, *shape, device="cuda").half().unbind(0)
        if layout == "tokens":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        scores = torch.rand(pages, n_kv, page, device="cuda") if track else None
        sp = torch.zeros(pages, n_kv, page, dtype=torch.int32, device="cuda") if track else None
        cache = ts.PagedKVCache(k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                torch.zeros(1, dtype=torch.int32, device="cuda"), scores, sp)
        slots = torch.randperm(pages * page, device="cuda")[:tokens]
        slots[5], slots[6], slots[7] = -1, pages * page, 1 << 40  # none, behind the pool, far behind it
        pos2 = pos.clone()
        pos2[9] = 50                                             # no rotary row: zeros, not stored
        wk, wv = k.clone(), v.clone()
        wsc, wsp = (scores.clone(), sp.clone()) if track else (None, None)
        got = ts.qk_norm_rope(x, n_q, n_kv, qw, kw, pos2, cos, sin, cache=cache, slots=slots)
        assert (got[9] == 0).all()
        plain = ts.qk_norm_rope(x, n_q, n_kv, qw, kw, pos2, cos, sin)
        assert torch.equal(got, plain)
        rows = got.view(tokens, -1, d)
        for t in range(tokens):
            if t in (5, 6, 7, 9):
                continue
            p, o = int(slots[t]) // page, int(slots[t]) % page
            wk[p, :, o], wv[p, :, o] = rows[t, n_q:n_q + n_kv], rows[t, n_q + n_kv:]
            if track:
                wsc[p, :, o], wsp[p, :, o] = 0.0, int(pos2[t])
        assert torch.equal(k, wk) and torch.equal(v, wv)
        if track:
            assert torch.equal(scores, wsc) and torch.equal(sp, wsp)
        y = x.clone()                                            # in place, values only to the pages
        ts.qk_norm_rope(y, n_q, n_kv, qw, kw, pos2, cos, sin, out=y, cache=cache, slots=slots)
        assert torch.equal(y, got) and torch.equal(k, wk) and torch.equal(v, wv)


def test_numbers_that_are_none(ts):
    x, qw, kw, _ = make(4, 2, 1, 64, torch.bfloat16, 1)
    x[0, 3], x[1, 64 * 2 + 5] = float("nan"), float("inf")
    x[2] = 0
    y = ts.qk_norm_rope(x, 2, 1, qw, kw).view(4, 4, 64)
    assert y[0, 0].isnan().all() and y[0, 1:].isfinite().all()
    assert y[1, 2, 5].isnan() and y[1, :2].isfinite().all()
    assert (y[2] == 0).all() and y[3].isfinite().all()


def test_few_and_no_tokens_captured(ts):
    x, qw, kw, pos = make(2, 8, 2, 128, torch.bfloat16, 4)
    cos, sin = tables(50, 128)
    assert ts.qk_norm_rope(x[:0], 8, 2, qw, kw, pos[:0], cos, sin).shape == (0, x.shape[1])
    g = torch.cuda.CUDAGraph()
    buf = x.clone()
    with torch.cuda.graph(g):
        y = ts.qk_norm_rope(buf, 8, 2, qw, kw, pos, cos, sin)
    buf.copy_(x * 2)
    g.replay()
    assert torch.equal(y, ts.qk_norm_rope(x * 2, 8, 2, qw, kw, pos, cos, sin))


def test_refusals(ts):
    x, qw, kw, pos = make(4, 2, 1, 64, torch.bfloat16, 1)
    cos, sin = tables(50, 64)
    f = ts.qk_norm_rope
    with pytest.raises(ValueError):
        f(x, 3, 1, qw, kw)                                       # heads that do not fill the row
    with pytest.raises(ValueError):
        f(x, 2, 1, qw[:32], kw)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, None, cos, sin)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, pos, cos, None)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, pos[:3], cos, sin)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, pos.int(), cos, sin)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw.half())
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, eps=-1.0)
    with pytest.raises(NotImplementedError):
        f(x.float(), 2, 1, qw, kw)
    with pytest.raises(NotImplementedError):
        f(x[:, :4 * 8].contiguous(), 2, 1)                       # heads of 8
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, out=x[:, :128])
    cache = ts.PagedKVCache.allocate(1, 1, 64, 64)
    with pytest.raises(ValueError):
        f(x, 2, 1, qw, kw, cache=cache)
    with pytest.raises(ValueError):
        f(x, 0, 2, None, kw, cache=cache, slots=torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(NotImplementedError):
        f(x, 2, 1, cache=ts.PagedKVCache8.allocate(1, 1, 64, 64), slots=torch.zeros(4, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError):
        f(x.cpu(), 2, 1)
    y = f(x.clone().requires_grad_(), 2, 1, qw, kw)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()
    z = x.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        f(z, 2, 1, qw, kw, out=z)
    with torch.no_grad():
        f(z, 2, 1, qw, kw, out=z)
    buf = torch.zeros(5, 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        f(buf[:4], 2, 1, qw, kw, out=buf[1:])                    # rows of the one are rows of the other
