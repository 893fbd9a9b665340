"""Microscaled 4-bit floating point on the GPU: codes and scales bit for bit
against the formulas, the product and the linear layer against 64-bit
arithmetic on the values that the codes stand for.

Tolerance of a product: the operands' values are exact in 64 bits, so only the
sum can differ. The tensor cores add 64 products per instruction to an fp32
sum: K / 64 additions, each off by at most 2^-22 of what it adds up to, bounded by
S = sum |a b|; 8 more for the scales, the bias and the pieces of a split sum.
An output in 16 bits adds half a unit in the last place.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
HALF_ULP = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12, torch.float32: 2.0 ** -25}


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


def nearest_e2m1(y):
    """Index of the nearest E2M1 magnitude, ties to the even index."""
    grid = torch.tensor(GRID, dtype=torch.float64, device=y.device)
    a = y.abs().double().clamp(max=6.0)
    d = (a[..., None] - grid).abs()
    best = d.amin(-1, keepdim=True)
    tied = d == best
    even = tied & (torch.arange(8, device=y.device) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, tied)
    return pick.to(torch.uint8).argmax(-1)


def formula(x, fmt, g):
    """(codes, scale bytes [rows, blocks], g) in fp32 steps, from the definition."""
    blk = 16 if fmt == "nvfp4" else 32
    rows, cols = x.shape
    xp = torch.zeros(rows, -(-cols // 64) * 64, device=x.device)
    xp[:, :cols] = x.float()
    xb = xp.view(rows, -1, blk)
    fine = xb.isfinite().all(-1)
    xb = torch.where(fine[..., None], xb, torch.zeros_like(xb))
    amax = xb.abs().amax(-1)
    if fmt == "nvfp4":
        if g is None:
            f = x.float()
            g = (torch.where(f.isfinite(), f, torch.zeros_like(f)).abs().max() / 2688).clamp(min=2.0 ** -100)
        else:
            g = torch.nan_to_num(g.reshape(()), nan=0.0).clamp(2.0 ** -100, 2.0 ** 118)
        s = (amax * (1 / (6 * g))).clamp(max=448).to(torch.float8_e4m3fn)
        sf = s.float()
        r = torch.where(sf > 0, 1 / (sf * g), torch.zeros_like(sf))
        raw = torch.where(fine, s.view(torch.uint8), torch.full_like(s.view(torch.uint8), 0x7F))
    else:
        e = torch.frexp(amax.double()).exponent - 1                      # floor(log2)
        e = torch.where(amax > 0, (e - 2).clamp(min=-127), torch.full_like(e, -127))
        r = torch.exp2(-e.double()).float()
        raw = torch.where(fine, (e + 127).to(torch.uint8), torch.full_like(e, 0xFF, dtype=torch.uint8))
    y = xb * r[..., None]
    codes = nearest_e2m1(y).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    codes = torch.where(fine[..., None], codes, torch.zeros_like(codes))
    return codes.reshape(rows, -1), raw, g


def unpack(t):
    c = t.codes
    return torch.stack((c & 15, c >> 4), -1).reshape(t.rows, -1)


def scale_bytes(t):
    blk = 16 if t.format == "nvfp4" else 32
    nb = -(-t.cols // 64) * 64 // blk
    kt = -(-nb // 4)
    r = torch.arange(t.rows, device=t.device)[:, None]
    j = torch.arange(nb, device=t.device)[None, :]
    return t.scales[((r // 128) * kt + j // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4]


def values64(t):
    """What the bytes of t stand for, in 64 bits."""
    code = unpack(t).long()
    mag = torch.tensor(GRID, dtype=torch.float64, device=t.device)[code & 7]
    v = torch.where(code >= 8, -mag, mag)
    raw = scale_bytes(t)
    if t.format == "nvfp4":
        s = raw.contiguous().view(torch.float8_e4m3fn).double()
        s = s * (1.0 if t.global_scale is None else t.global_scale.double())
        blk = 16
    else:
        s = torch.where(raw == 255, torch.full_like(raw, 0).double() * float("nan"), torch.exp2(raw.double() - 127))
        blk = 32
    return (v.view(t.rows, -1, blk) * s[..., None]).reshape(t.rows, -1)[:, :t.cols]


def data(rows, cols, dtype, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device=device) * torch.exp(torch.randn(rows, 1, generator=g, device=device))
    return x.to(dtype)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 64), (3, 17), (2, 96), (130, 200), (257, 513), (33, 1056), (5, 4099)])
def test_codes_and_scales_are_the_formulas(ts, fmt, dtype, rows, cols):
    x = data(rows, cols, dtype, rows * 1000 + cols)
    for given in ([None, torch.full((1,), 0.011, device="cuda")] if fmt == "nvfp4" else [None]):
        t = ts.fp4_quantize(x, fmt, global_scale=given)
        codes, raw, g = formula(x, fmt, given)
        assert torch.equal(scale_bytes(t), raw)
        assert torch.equal(unpack(t), codes)
        if fmt == "nvfp4":
            assert t.global_scale.item() == g.item()
        back = ts.fp4_dequantize(t, torch.float32)
        v = torch.tensor(GRID, device="cuda")[codes.long() & 7] * (1 - 2 * (codes >= 8).float())
        s = raw.contiguous().view(torch.float8_e4m3fn).float() * g if fmt == "nvfp4" else torch.exp2(raw.double() - 127).float()
        want = (v.view(rows, -1, 16 if fmt == "nvfp4" else 32) * s[..., None]).reshape(rows, -1)[:, :cols]
        assert torch.equal(back, want)
        for dt in (torch.bfloat16, torch.float16):
            assert torch.equal(ts.fp4_dequantize(t, dt), want.to(dt))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_strided_and_unaligned_rows(ts, fmt):
    base = data(40, 700, torch.bfloat16, 5)
    for x in (base[:, 3:259], base[::2, :256], base[1:, 1:130].contiguous(), base.t()[:64]):
        a, b = ts.fp4_quantize(x, fmt), ts.fp4_quantize(x.contiguous().clone(), fmt)
        assert torch.equal(a.codes, b.codes) and torch.equal(scale_bytes(a), scale_bytes(b))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_extreme_values(ts, fmt, dtype):
    fi = torch.finfo(dtype)
    x = torch.zeros(12, 128, dtype=dtype, device="cuda")
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    x[3, 41] = -float("inf")
    x[4] = fi.max
    x[5] = -fi.max
    x[6] = fi.tiny
    x[7, ::3] = fi.smallest_normal / 4                       # below the normal range
    x[8] = torch.linspace(-6, 6, 128).to(dtype)              # ties of the grid
    x[9] = -0.0
    x[10, :16] = fi.max
    x[10, 16:] = 1.0
    for sub in (x, x[4:6], x[6:8], x[8:10], x[:1]):
        t = ts.fp4_quantize(sub, fmt)
        codes, raw, g = formula(sub, fmt, None)
        assert torch.equal(scale_bytes(t), raw) and torch.equal(unpack(t), codes)
        back = ts.fp4_dequantize(t)
        blk = 16 if fmt == "nvfp4" else 32
        bad = ~sub.float().isfinite().reshape(sub.shape[0], -1, blk).all(-1)
        assert torch.equal(back.reshape(sub.shape[0], -1, blk).isnan().all(-1), bad)
        assert not back.isinf().any()


@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf"), 1e-38])
def test_given_scale_out_of_range_is_clamped(ts, g):
    x = data(4, 64, torch.float32, 1)
    t = ts.fp4_quantize(x, "nvfp4", global_scale=torch.full((1,), g, device="cuda"))
    codes, raw, _ = formula(x, "nvfp4", torch.full((1,), g, device="cuda"))
    assert torch.equal(scale_bytes(t), raw) and torch.equal(unpack(t), codes)
    assert ts.fp4_dequantize(t).isfinite().all()


def check_product(y, a, b, bias, k):
    want = a @ b.t()
    mag = a.abs() @ b.abs().t()
    if bias is not None:
        want = want + bias.double()
        mag = mag + bias.double().abs()
    tol = (k / 64 + 8) * 2.0 ** -22 * mag + HALF_ULP[y.dtype] * 2 * want.abs() + 1e-30
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -24
    err = (y.double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.3g} tolerances"


SHAPES = [(1, 128, 64), (1, 1, 256), (3, 200, 300), (16, 256, 1024), (17, 129, 4096), (33, 1000, 2112), (64, 384, 640),
          (65, 500, 832), (128, 256, 512), (129, 300, 4160), (255, 640, 1280), (300, 1025, 704), (513, 130, 64)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(ts, fmt, m, n, k):
    a = ts.fp4_quantize(data(m, k, torch.bfloat16, m + k), fmt)
    b = ts.fp4_quantize(data(n, k, torch.float32, n), fmt)
    bias = torch.randn(n, device="cuda")
    va, vb = values64(a), values64(b)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        check_product(ts.fp4_matmul(a, b, out_dtype=dt), va, vb, None, k)
    check_product(ts.fp4_matmul(a, b, bias=bias.to(torch.bfloat16), out_dtype=torch.float32), va, vb,
                  bias.to(torch.bfloat16), k)


# few tiles of many columns: tiles split over CTAs, as whole parts and as equal shares, few and many of them
SPLITS = [(1, 128, 14336), (100, 120, 9000), (40, 10300, 4160), (3, 1023, 4160), (33, 640, 9000), (128, 257, 12173),
          (7, 3136, 2000), (64, 9000, 3000), (190, 700, 6000), (16, 2300, 1100), (1, 18800, 8192)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SPLITS)
def test_product_split_along_its_columns(ts, fmt, m, n, k):
    a = ts.fp4_quantize(data(m, k, torch.bfloat16, m + k), fmt)
    b = ts.fp4_quantize(data(n, k, torch.bfloat16, n), fmt)
    bias = torch.randn(n, device="cuda").to(torch.bfloat16)
    va, vb = values64(a), values64(b)
    first = {}
    for _ in range(2):
        for dt in (torch.float32, torch.bfloat16):
            y = ts.fp4_matmul(a, b, bias=bias, out_dtype=dt)
            check_product(y, va, vb, bias, k)
            assert torch.equal(y, first.setdefault(dt, y))


# enough tiles for CTA pairs, with edges in every direction
PAIRS = [(200, 9500, 320), (257, 5000, 1088), (1000, 2561, 576), (129, 19000, 64), (600, 3200, 2000),
         (130, 16576, 256), (512, 8288, 640), (400, 8100, 1344), (256, 16500, 832)]


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", PAIRS)
def test_product_on_pairs(ts, fmt, m, n, k):
    a = ts.fp4_quantize(data(m, k, torch.bfloat16, m + k), fmt)
    b = ts.fp4_quantize(data(n, k, torch.float32, n), fmt)
    bias = torch.randn(n, device="cuda").to(torch.float16)
    va, vb = values64(a), values64(b)
    for dt in (torch.float32, torch.bfloat16):
        check_product(ts.fp4_matmul(a, b, out_dtype=dt), va, vb, None, k)
    check_product(ts.fp4_matmul(a, b, bias=bias, out_dtype=torch.float16), va, vb, bias, k)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 14336), (2048, 1024, 4096), (2047, 14336, 4096), (2048, 4096, 14336)])
def test_product_of_large_shapes(ts, m, n, k):
    a, b = ts.fp4_quantize(data(m, k, torch.bfloat16, 1)), ts.fp4_quantize(data(n, k, torch.bfloat16, 2))
    check_product(ts.fp4_matmul(a, b, out_dtype=torch.float32), values64(a), values64(b), None, k)


@pytest.mark.parametrize("m", [3, 40, 2000])
@pytest.mark.parametrize("ga,gb", [(-70, -65), (-100, -40), (118, -100), (-90, 118), (100, 21), (61, 60), (-3, 5)])
def test_product_of_extreme_tensor_scales(ts, m, ga, gb):
    """Scales whose product leaves fp32's normal range on the way to sums that do not."""
    n, k = (300, 500) if m < 100 else (4800, 500)
    def tensor(rows, seed, e):
        t = ts.fp4_quantize(data(rows, k, torch.bfloat16, seed), "nvfp4")
        return ts.Fp4Tensor(t.codes, t.scales, torch.full((1,), 2.0 ** e, device="cuda"), rows, k, "nvfp4")
    a, b = tensor(m, 1, ga), tensor(n, 2, gb)
    if ga + gb > 90:                                     # sums of up to 2^39 would leave the range
        for t in (a, b):
            t.scales.copy_(torch.where(t.scales > 8, t.scales // 16, t.scales))
    a.codes[0] = 0
    va, vb = values64(a), values64(b)
    y = ts.fp4_matmul(a, b, out_dtype=torch.float32).double()
    want, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    assert mag.max() < 2.0 ** 127 and (y[0] == 0).all()
    assert ((y - want).abs() <= (k / 64 + 8) * 2.0 ** -22 * mag + 2.0 ** -149).all()


def test_nan_blocks_reach_their_rows_only(ts):
    x, w = data(20, 256, torch.bfloat16, 3), data(140, 256, torch.bfloat16, 4)
    x[7, 100] = float("nan")
    w[133, 5] = float("inf")
    for fmt in ("nvfp4", "mxfp4"):
        y = ts.fp4_matmul(ts.fp4_quantize(x, fmt), ts.fp4_quantize(w, fmt), out_dtype=torch.float32)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[7] = True
        bad[:, 133] = True
        assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("shape,n,k", [((1, 256), 384, 256), ((2, 5, 320), 200, 320), ((150, 1000), 129, 1000), ((0, 128), 64, 128)])
def test_linear_is_quantise_then_product(ts, fmt, shape, n, k):
    x = data(max(1, torch.Size(shape).numel() // k), k, torch.bfloat16, 9)[:torch.Size(shape).numel() // k].reshape(shape)
    w = ts.fp4_quantize(data(n, k, torch.bfloat16, 10), fmt)
    g = torch.full((1,), 0.02, device="cuda") if fmt == "nvfp4" else None
    bias = torch.randn(n, device="cuda").to(torch.float16)
    y = ts.fp4_linear(x, w, bias=bias, input_scale=g)
    assert y.shape == (*shape[:-1], n) and y.dtype == x.dtype
    if x.numel():
        a = ts.fp4_quantize(x.reshape(-1, k), fmt, global_scale=g)
        assert torch.equal(y.reshape(-1, n), ts.fp4_matmul(a, w, bias=bias, out_dtype=x.dtype))
        check_product(y.reshape(-1, n), values64(a), values64(w), bias, k)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 130, 17), (2, 300, 64), (3, 128, 250), (5, 1000, 5001), (8, 4096, 4096), (8, 200, 8200),
                                   (9, 130, 515)])
def test_linear_of_few_tokens(ts, fmt, dtype, m, n, k):
    """Tokens that the product may quantise itself: the bits of a quantisation
    in front, for any stride and alignment, with blocks that are not finite."""
    w = ts.fp4_quantize(data(n, k, torch.bfloat16, 20), fmt)
    wide = data(m, k + 21, dtype, 21)
    g = torch.full((1,), 0.01, device="cuda") if fmt == "nvfp4" else None
    for x in (wide[:, :k].contiguous(), wide[:, 8:8 + k], wide[:, 1:1 + k], wide[:1, 3:3 + k].expand(m, k)):
        y = ts.fp4_linear(x, w, input_scale=g, out_dtype=torch.float32)
        assert torch.equal(y, ts.fp4_matmul(ts.fp4_quantize(x, fmt, g), w, out_dtype=torch.float32))
    x = wide[:, :k].clone()
    x[0, k // 2] = float("inf")
    x[m - 1, 0] = float("nan")
    x[m // 2, k - 1] = 0.0
    y = ts.fp4_linear(x, w, input_scale=g, out_dtype=torch.float32)
    want = ts.fp4_matmul(ts.fp4_quantize(x, fmt, g), w, out_dtype=torch.float32)
    assert torch.equal(y.nan_to_num(), want.nan_to_num()) and torch.equal(y.isnan(), want.isnan())
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[0] = bad[m - 1] = True
    assert torch.equal(y.isnan().all(1), bad)


def test_results_repeat_and_do_not_depend_on_earlier_calls(ts):
    """Split sums are added in a fixed order, and a call leaves the workspace
    as the next one of another shape needs it."""
    calls = []
    for m, n, k in [(1, 2000, 8192), (40, 300, 4096), (100, 512, 2048), (1, 129, 64), (700, 512, 512)]:
        a, b = ts.fp4_quantize(data(m, k, torch.bfloat16, m)), ts.fp4_quantize(data(n, k, torch.bfloat16, n))
        calls.append((a, b, ts.fp4_matmul(a, b, out_dtype=torch.float32)))
    for _ in range(3):
        for a, b, y in reversed(calls):
            assert torch.equal(ts.fp4_matmul(a, b, out_dtype=torch.float32), y)


def test_side_stream_and_graph(ts):
    x, w = data(8, 512, torch.bfloat16, 1), ts.fp4_quantize(data(640, 512, torch.bfloat16, 2))
    want = ts.fp4_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ts.fp4_linear(x, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        ts.fp4_linear(buf, w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        out = ts.fp4_linear(buf, w)
    buf.copy_(x * 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ts.fp4_linear(x * 2, w))


def test_module(ts):
    layer = torch.nn.Linear(320, 200, device="cuda", dtype=torch.bfloat16)
    x = data(12, 320, torch.bfloat16, 6)
    for fmt in ("nvfp4", "mxfp4"):
        q = ts.Fp4Linear.from_linear(layer, fmt)
        q.calibrate(x)
        y = q(x)
        a = ts.fp4_quantize(x, fmt, global_scale=q.input_scale)
        check_product(y, values64(a), values64(q.weight()), layer.bias.detach(), 320)
        # 4-bit operands: the layer's own result to within the formats' coarseness
        ref = layer(x).float()
        assert (y.float() - ref).norm() / ref.norm() < 0.25
        again = ts.Fp4Linear.from_linear(torch.nn.Linear(320, 200, device="cuda", dtype=torch.bfloat16), fmt)
        again.load_state_dict(q.state_dict())
        assert torch.equal(again(x), y)


def test_refusals(ts):
    x = data(4, 64, torch.bfloat16, 1)
    w = ts.fp4_quantize(data(8, 64, torch.bfloat16, 2))
    one = torch.ones(1, device="cuda")
    for bad, err in [(lambda: ts.fp4_quantize(x, "fp4"), NotImplementedError),
                     (lambda: ts.fp4_quantize(x.int()), NotImplementedError),
                     (lambda: ts.fp4_quantize(x[0]), ValueError),
                     (lambda: ts.fp4_quantize(x[:, :0]), ValueError),
                     (lambda: ts.fp4_quantize(x, "mxfp4", global_scale=one), ValueError),
                     (lambda: ts.fp4_quantize(x, global_scale=one.double()), ValueError),
                     (lambda: ts.fp4_quantize(x.cpu()), RuntimeError),
                     (lambda: ts.fp4_matmul(ts.fp4_quantize(x, "mxfp4"), w), ValueError),
                     (lambda: ts.fp4_linear(x[:, :32], w), ValueError),
                     (lambda: ts.fp4_linear(x, w, bias=torch.zeros(9, device="cuda")), ValueError),
                     (lambda: ts.fp4_linear(x, w, out_dtype=torch.int32), NotImplementedError),
                     (lambda: ts.fp4_dequantize(w, torch.float64), NotImplementedError),
                     (lambda: ts.Fp4Tensor(w.codes[:, :16], w.scales, None, 8, 64, "nvfp4"), ValueError),
                     (lambda: ts.Fp4Tensor(w.codes, w.scales[:16], None, 8, 64, "nvfp4"), ValueError),
                     (lambda: ts.Fp4Tensor(w.codes, w.scales, one, 8, 64, "mxfp4"), ValueError)]:
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("m", [1, 200])
def test_stalled_product_reports_and_recovers(ts, m):
    """A launch whose producer issues nothing: its waits run out, the status
    says so, and the same workspace serves the next call."""
    from tensorshrink_b200 import _C, kernels
    a, b = ts.fp4_quantize(data(m, 1024, torch.bfloat16, 1)), ts.fp4_quantize(data(9500, 1024, torch.bfloat16, 2))
    want = ts.fp4_matmul(a, b)
    kernels.device_status()
    assert _C.load().ts_test_inject_stall(1_000_000) == 0
    ts.fp4_matmul(a, b)
    with pytest.raises(RuntimeError, match="ts_fp4_status"):
        kernels.device_status()
    kernels.device_status()
    assert torch.equal(ts.fp4_matmul(a, b), want)
