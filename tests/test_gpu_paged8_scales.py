"""Scales of any sign in the 8-bit cache: a code stands for code * scale, whoever wrote the two.

Attention over scales (and codes) of other signs is the same sums, so that it is the same bits as over the values' own
signs; appended tokens and the earlier ones of their block keep their values but for roundings: half a step of the
scale each (e4m3: 2^-4 of the value, or 2^-10 of the scale where the code is subnormal), and fp32's 2^-20.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


def filled(ts, held, d, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ts.PagedKVCache8.allocate(3, 2, d, 256, page_size=32, dtype=held)
    for pages in (c.k_pages, c.v_pages):
        pages.copy_((torch.randn(pages.shape, generator=g, device="cuda") * 30).round().clamp(-127, 127).to(held))
    for s in (c.k_scales, c.v_scales):
        s.copy_(torch.exp2(torch.randn(s.shape, generator=g, device="cuda")) / 64)
    c.seq_lens.copy_(torch.tensor(n, dtype=torch.int32))
    return c, g


def flipped(ts, c, g):
    """The same values, by other codes and scales."""
    args = []
    for pages, scales in ((c.k_pages, c.k_scales), (c.v_pages, c.v_scales)):
        sign = torch.where(torch.rand(scales.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
        args.append(((pages.float() * sign.repeat_interleave(16, 2)[..., None]).to(pages.dtype), scales * sign))
    (k, ks), (v, vs) = args
    return ts.PagedKVCache8(k, v, ks, vs, c.page_table.clone(), c.seq_lens.clone())


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(128, 4), (64, 12), (256, 2)])
def test_attention(ts, held, dtype, d, group):
    c, g = filled(ts, held, d, [250, 17, 100], 1)
    other = flipped(ts, c, g)
    q = torch.randn(3, 2 * group * d, generator=g, device="cuda").to(dtype)
    assert (other.v_scales < 0).any() and (other.k_scales < 0).any()
    for a, b in zip(ts.paged_dequantize(c, torch.float32), ts.paged_dequantize(other, torch.float32)):
        assert torch.equal(a, b)
    assert torch.equal(ts.paged_attention(q, other), ts.paged_attention(q, c))
    other.v_scales.neg_()                                # not a positive one among them, or the other way round
    torch.testing.assert_close(ts.paged_attention(q, other), -ts.paged_attention(q, c), rtol=0, atol=0)
    other.v_scales.copy_(-other.v_scales.abs())
    c.v_scales.copy_(other.v_scales.abs())
    c.v_pages.copy_(other.v_pages)
    assert torch.equal(ts.paged_attention(q, other), -ts.paged_attention(q, c))


@pytest.mark.parametrize("held", [INT8, E4M3])
def test_append(ts, held):
    n = [5, 16, 40]
    c, g = filled(ts, held, 64, n, 2)
    c = flipped(ts, c, g)
    for loud in (0.1, 4.0, 60.0):                        # fits the block, or makes its scale grow
        was = ts.paged_dequantize(c, torch.float32)
        k, v = (torch.randn(3, 3, 2, 64, generator=g, device="cuda") * loud).bfloat16(), \
            (torch.randn(3, 3, 2, 64, generator=g, device="cuda") * loud).bfloat16()
        ts.paged_append(k, v, c)
        now = ts.paged_dequantize(c, torch.float32)
        for x, before, after, scales in ((k, was[0], now[0], c.k_scales), (v, was[1], now[1], c.v_scales)):
            for b in range(3):
                for slot in range(n[b] // 16 * 16, n[b] + 3):
                    p, o = int(c.page_table[b, slot // 32]), slot % 32
                    want = before[p, :, o] if slot < n[b] else x[b, slot - n[b]].float()
                    s = scales[p, :, o // 16].abs()[:, None]
                    tol = 0.5 * s if held == INT8 else torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * s)
                    assert ((after[p, :, o] - want).abs() <= tol + 2.0 ** -20 * (want.abs() + s)).all()
        c.seq_lens.add_(3)
        n = [i + 3 for i in n]
