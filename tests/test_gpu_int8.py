"""8-bit integers with a scale per row on the GPU, against their definition.

Everything here is exact: the codes and scales follow from fp32 operations
that torch rounds the same way, the sums of products are integers, and the
result is the sum as fp32, times the smaller and the larger scale, plus the
bias, each rounded once, and rounded to its type.
"""

from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


def rows_of(x):
    """Codes and scales of x's rows by the formula."""
    f = x.float()
    s = (f.abs().amax(dim=1) * (1.0 / 127.0)).clamp(min=2.0 ** -100)
    q = torch.round(f * (1.0 / s)[:, None]).to(torch.int8)
    bad = ~f.isfinite().all(dim=1)
    return torch.where(bad[:, None], torch.zeros_like(q), q), torch.where(bad, torch.full_like(s, float("nan")), s)


def product(a, sa, b, sb, bias, dtype):
    """The result of codes a, b (any width) with their scales."""
    sums = a.double() @ b.double().t()                        # exact: below 2^53
    y = (sums.float() * torch.minimum(sa[:, None], sb)) * torch.maximum(sa[:, None], sb)
    return (y if bias is None else y + bias.float()).to(dtype)


def matrix(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(dtype)


def same(x, y):
    assert x.shape == y.shape and x.dtype == y.dtype
    assert torch.equal(x.isnan(), y.isnan())
    assert torch.equal(x.nan_to_num(nan=7.0), y.nan_to_num(nan=7.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (2, 1024), (2, 1025), (9, 4095), (131, 4096), (4, 8200),
                                       (3, 14330), (2, 28672), (2, 33001)])
def test_quantize(ts, rows, cols, dtype):
    x = matrix(rows, cols, dtype, cols)
    x[-1, cols // 2] = 0.0
    t = ts.int8_quantize(x)
    q, s = rows_of(x)
    assert t.shape == (rows, cols) and t.codes.shape[1] % 16 == 0
    assert torch.equal(t.codes[:, :cols], q) and torch.equal(t.scales, s)
    assert not t.codes[:, cols:].any()
    for out in DTYPES:
        assert torch.equal(ts.int8_dequantize(t, out), (q.float() * s[:, None]).to(out))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strided_rows(ts, dtype):
    base = matrix(40, 4200, dtype, 1)
    for x in (base[:, 1:4098], base[::3, 3:], base[:, 8:4104], base.t()[:50], base[5:6]):
        t = ts.int8_quantize(x)
        q, s = rows_of(x)
        assert torch.equal(t.codes[:, :x.shape[1]], q) and torch.equal(t.scales, s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_rows(ts, dtype):
    x = matrix(8, 300, dtype, 2)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 299] = float("nan")
    x[3, 0] = -float("inf")
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).tiny
    x[6] = x[6] * 0 + 0.5                                       # every code 127
    t = ts.int8_quantize(x)
    q, s = rows_of(x)
    assert torch.equal(t.codes[:, :300], q)
    same(t.scales, s)
    back = ts.int8_dequantize(t)
    assert back[1:4].isnan().all() and back[[0, 4, 5, 6, 7]].isfinite().all()
    w = ts.int8_quantize(matrix(20, 300, torch.float32, 3))
    y = ts.int8_matmul(t, w, out_dtype=torch.float32)
    assert y[1:4].isnan().all() and (y[0] == 0).all()
    same(y, product(q, s, w.codes[:, :300], w.scales, None, torch.float32))


SHAPES = [(1, 1, 1), (1, 128, 16), (2, 7, 31), (1, 14336, 4096), (5, 1000, 100), (16, 129, 4096), (17, 4096, 128), (33, 4096, 14336),
          (64, 257, 129), (65, 128, 8192), (128, 1025, 4095), (129, 256, 32), (129, 300, 14330), (200, 4096, 33),
          (255, 1000, 1000), (256, 256, 128), (257, 513, 384), (300, 4097, 1024), (513, 2048, 4100), (1025, 1030, 513),
          (2047, 4096, 4096)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(ts, m, n, k):
    a, b = ts.int8_quantize(matrix(m, k, torch.float32, m)), ts.int8_quantize(matrix(n, k, torch.float32, n + 1))
    bias = matrix(1, n, torch.float32, 5)[0]
    for dtype in DTYPES:
        for z in (None, bias.to(dtype)):
            assert torch.equal(ts.int8_matmul(a, b, z, dtype),
                               product(a.codes[:, :k], a.scales, b.codes[:, :k], b.scales, z, dtype)), (dtype, z is None)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (1, 130, 1), (1, 1000, 16384), (1, 200, 16385), (2, 4000, 8192), (2, 77, 333),
                                   (3, 512, 4096), (8, 300, 1000), (40, 1024, 4096), (300, 520, 777)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_is_quantize_then_matmul(ts, m, n, k, dtype):
    x, w = matrix(m, k, dtype, 3), ts.int8_quantize(matrix(n, k, torch.float32, 4))
    bias = matrix(1, n, dtype, 6)[0]
    y = ts.int8_linear(x, w, bias)
    t = ts.int8_quantize(x)
    assert torch.equal(y, ts.int8_matmul(t, w, bias, dtype))
    assert torch.equal(y, product(t.codes[:, :k], t.scales, w.codes[:, :k], w.scales, bias, dtype))
    for _ in range(3):                                          # sums do not depend on who adds first
        assert torch.equal(ts.int8_linear(x, w, bias), y)
    assert torch.equal(ts.int8_linear(x, w, bias, out_dtype=torch.float32),
                       product(t.codes[:, :k], t.scales, w.codes[:, :k], w.scales, bias, torch.float32))


def test_largest_codes_fill_the_sums(ts):
    # every product 127^2 over the longest rows allowed: sums close to 2^31, of either sign
    k = 131072
    a = torch.full((130, k), 127, dtype=torch.int8, device="cuda")
    b = torch.full((300, k), 127, dtype=torch.int8, device="cuda")
    b[::2] = -127
    one = torch.ones(300, device="cuda")
    for m in (1, 130):
        y = ts.int8_matmul(ts.Int8Tensor(a[:m], one[:m]), ts.Int8Tensor(b, one), out_dtype=torch.float32)
        assert torch.equal(y, torch.where(torch.arange(300, device="cuda") % 2 == 0, -1.0, 1.0).float().mul(127.0 * 127 * k).expand(m, 300))


def test_scales_at_the_ends_of_the_range(ts):
    k = 64
    a = torch.randint(-127, 128, (4, k), dtype=torch.int8, device="cuda")
    b = torch.randint(-127, 128, (6, k), dtype=torch.int8, device="cuda")
    sa = torch.tensor([2.0 ** -100, 2.0 ** 100, 1.0, 2.0 ** 121], device="cuda")
    sb = torch.tensor([2.0 ** 100, 2.0 ** -100, 2.0 ** -100, 1.0, 2.0 ** 60, float("nan")], device="cuda")
    y = ts.int8_matmul(ts.Int8Tensor(a, sa), ts.Int8Tensor(b, sb), out_dtype=torch.float32)
    exact = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    assert y[:, 5].isnan().all()
    for i in range(4):
        for j in range(5):
            e = exact[i, j].float()                             # a product with a power of two rounds once at most
            assert y[i, j] == e or (e.abs() < 2.0 ** -126 and (y[i, j] - e).abs() <= 2.0 ** -149)


def test_padding_of_the_codes_does_not_count(ts):
    k = 100
    a, b = ts.int8_quantize(matrix(3, k, torch.float32, 1)), ts.int8_quantize(matrix(200, k, torch.float32, 2))
    y = ts.int8_matmul(a, b)
    for t in (a, b):
        t.codes[:, k:] = 99
    assert torch.equal(ts.int8_matmul(a, b), y)
    wide = torch.full((200, 256), 77, dtype=torch.int8, device="cuda")
    wide[:, :k] = b.codes[:, :k]
    assert torch.equal(ts.int8_matmul(a, ts.Int8Tensor(wide[:, :112], b.scales, k)), y)


def test_shapes_and_module(ts):
    layer = torch.nn.Linear(200, 72).cuda().half()
    m = ts.Int8Linear.from_linear(layer)
    x = matrix(6, 200, torch.float16, 8)
    y = m(x)
    assert torch.equal(m(x.view(2, 3, 200)).view(6, 72), y) and torch.equal(m(x[0]), y[0])
    assert m(x[:0]).shape == (0, 72)
    m = m.bfloat16()
    assert m.scales.dtype == torch.float32 and m.bias.dtype == torch.bfloat16
    assert ts.int8_quantize(x[:0]).codes.shape == (0, 208)
    assert ts.int8_linear(x, ts.int8_quantize(x[:0])).shape == (6, 0)
    big = matrix(6, 401, torch.float16, 8)
    assert torch.equal(m.half()(big[:, 1:201]), m(big[:, 1:201].contiguous()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_and_two_tokens_as_they_come(ts, dtype):
    # rows that start anywhere, of any size and content, through the kernel that quantises them itself
    w = ts.int8_quantize(matrix(300, 515, torch.float32, 4))
    base = matrix(6, 1200, dtype, 5)
    base[4] = 0
    base[5, 530] = float("nan")
    for rows in (slice(0, 1), slice(1, 3), slice(4, 5), slice(4, 6)):
        for at in (0, 1, 3, 8):
            x = base[rows, at:at + 515]
            q, s = rows_of(x)
            same(ts.int8_linear(x, w), product(q, s, w.codes[:, :515], w.scales, None, dtype))


def test_refusals(ts):
    x = matrix(4, 64, torch.bfloat16, 1)
    w = ts.int8_quantize(x)
    with pytest.raises(ValueError):
        ts.int8_quantize(x[0])
    with pytest.raises(NotImplementedError):
        ts.int8_quantize(x.double())
    with pytest.raises(ValueError):
        ts.int8_linear(x[:, :32], w)
    with pytest.raises(ValueError):
        ts.int8_linear(x, w, torch.zeros(3, device="cuda"))
    with pytest.raises(NotImplementedError):
        ts.int8_linear(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ts.Int8Tensor(w.codes, w.scales[:2])
    with pytest.raises(ValueError):
        ts.Int8Tensor(w.codes[:, :40], w.scales, 40)           # not padded to 16
    with pytest.raises(ValueError):
        ts.Int8Tensor(w.codes.float(), w.scales)
    with pytest.raises(ValueError):
        ts.int8_matmul(w, ts.int8_quantize(x[:, :32]))
    with pytest.raises(RuntimeError):
        ts.int8_linear(x.cpu(), w)
    long = torch.zeros(1, 131088, dtype=torch.int8, device="cuda")
    t = ts.Int8Tensor(long, torch.ones(1, device="cuda"))
    with pytest.raises(NotImplementedError):
        ts.int8_matmul(t, t)
    y = ts.int8_linear(x.float().requires_grad_(), w)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_captured_and_on_other_streams(ts):
    w = ts.int8_quantize(matrix(4096, 4096, torch.float32, 1))
    x = matrix(3, 4096, torch.bfloat16, 2)
    want = [ts.int8_linear(x + i, w) for i in range(3)]
    buf = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ts.int8_linear(buf, w)
        z = ts.int8_linear(buf, w)
    for i in range(3):
        buf.copy_(x + i)
        g.replay()
        assert torch.equal(y, want[i]) and torch.equal(z, want[i])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = [[] for _ in streams]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                outs[i].append(ts.int8_linear(x + i, w))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(3):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("m", [2, 300])
def test_a_wait_that_runs_out_is_reported(ts, m):
    from tensorshrink_b200 import _C
    w = ts.int8_quantize(matrix(1024, 2048, torch.float32, 1))
    x = matrix(m, 2048, torch.bfloat16, 2)
    y = ts.int8_linear(x, w)
    torch.cuda.synchronize()
    _C.load().ts_test_inject_stall(20_000_000)                  # 20 ms
    ts.int8_linear(x, w)
    with pytest.raises(RuntimeError, match="ts_int8_status"):
        _C.serving_ops().serving_status(0)
    _C.serving_ops().serving_status(0)
    assert torch.equal(ts.int8_linear(x, w), y)
