"""The softmax weights of the 8-bit attention, where the values cancel.

Every second value is the negative of the one before it, and the scores are close
together, so that a result is small beside the values it is made of and shows what the
weights lost. Scores are at most 2^-3, the sums of at most 256 products of that size, whose
additions in fp32 (cut off, not rounded, by the tensor cores) err by 256 * 2^-23 * 2^-3 =
2^-18; integers of the queries by 2^-22 of the largest, under 2^-20 in a score. The
exponential, two terms of a weight, the sums of 32 of them and the division add 2^-19 at most.
So |err| <= eps / 2 |o| + 2^-17 sum p |v| for results of either type.
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


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group,batch", [(128, 4, 40), (128, 16, 10), (64, 8, 20), (96, 1, 80), (256, 3, 10), (128, 8, 200)])
def test_weights_keep_their_bits(ts, d, group, batch, dtype, held):
    n_kv, g = 2, torch.Generator(device="cuda").manual_seed(d + group)
    c = ts.PagedKVCache8.allocate(batch, n_kv, d, 32, page_size=32, dtype=held)
    k, v = (torch.randn(batch, n_kv, 32, d, generator=g, device="cuda") for _ in range(2))
    v[:, :, 1::2] = -v[:, :, ::2]
    for pages, x in ((c.k_pages, k), (c.v_pages, v)):
        pages.copy_((x * 20).round().clamp(-127, 127).to(held))
    c.v_scales.uniform_(0.7, 1.9, generator=g)
    c.seq_lens.copy_(torch.tensor([2, 32, 14, 2, 16] * (batch // 5), dtype=torch.int32))
    q = torch.randn(batch, n_kv * group * d, generator=g, device="cuda").to(dtype)
    x, kk, vv = q.double().view(batch, n_kv, group, d), c.k_pages.double(), c.v_pages.double()
    kk, vv = (y * s.double().repeat_interleave(16, 2)[..., None] for y, s in ((kk, c.k_scales), (vv, c.v_scales)))
    scale = 2.0 ** -3 / float((x.abs() @ kk.abs().transpose(2, 3)).max())
    s = x @ kk.transpose(2, 3) * scale
    s.masked_fill_(torch.arange(32, device="cuda") >= c.seq_lens.view(-1, 1, 1, 1), float("-inf"))
    p = torch.softmax(s, -1)
    want, size = (p @ vv).view(batch, -1), (p @ vv.abs()).view(batch, -1)
    got = ts.paged_attention(q, c, scale=scale)
    err = (got.double() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -17 * size
    assert (err <= tol).all(), (float((err / size).max()), int((err > tol).sum()))
