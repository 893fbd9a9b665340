"""How far codes drift while the scale of their block grows.

A token that does not fit its block's scale makes it grow by a quarter at least, and the earlier codes are
rounded anew. With s the last scale and m the growths since a token x came:

int8: every rounding is off by half a step, 1/2 of the scale of its time, and each scale is at most 0.8 of the next:
|x' - x| <= s / 2 (1 + 0.8 + 0.64 + ...) = 2.5 s. (The products in front of the roundings are fp32:
127 * 2^-22 of a step more each time, under 2^-10 in all.)

e4m3: a rounding is off by 2^-4 of the value, or by 2^-10 of the scale where the code is subnormal. Values do not shrink with
the growing scale, so the first kind adds up: |x' - x| <= ((1 + 2^-4)^(m + 1) - 1) |x| + 2^-10 s
(1 + 1.0625 / 1.25 + ...) <= ((1 + 2^-4)^(m + 1) - 1) |x| + 6.7 * 2^-10 s, and fp32 as above. Beside the block's largest
value, 448 s, that is no more than max over m of ((1 + 2^-4)^(m + 1) - 1) / 1.25^m = 0.146 (m = 4: 0.1457), as x was at most
448 times its own scale, and the subnormal term.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
INT8, E4M3 = torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("growth", [1.01, 1.26, 1.5, "drawn"])
def test_drift_of_growing_blocks(held, block, growth):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as ts
    g = torch.Generator(device="cuda").manual_seed(block)
    n_kv, d = 4, 128
    c = ts.PagedKVCache8.allocate(1, n_kv, d, block, page_size=block, block=block, dtype=held)
    rows, scales, loud = [], [], 1.0
    for t in range(block):
        x = torch.randn(1, 1, n_kv, d, generator=g, device="cuda")
        x = (x / x.abs().amax(-1, keepdim=True) * loud).bfloat16()
        ts.paged_append(x, x, c)
        c.advance()
        rows.append(x[0, 0].double())
        scales.append(c.k_scales[0, :, 0].double())
        loud *= float(torch.rand((), generator=g, device="cuda")) * 0.3 + 1.25 if growth == "drawn" else growth
    x, s = torch.stack(rows, 1), torch.stack(scales, 1)              # [n_kv, block, d], [n_kv, block]
    grew = (s[:, 1:] > s[:, :-1]).sum(1)
    if growth != 1.01:
        assert (grew == block - 1).all()                             # with every token
    assert (s[:, 1:] >= s[:, :-1]).all()
    assert ((s[:, 1:] >= 1.25 * s[:, :-1] * (1 - 2.0 ** -20)) | (s[:, 1:] == s[:, :-1])).all()
    last = s[:, -1, None, None]
    since = torch.stack([(s[:, t + 1:] > s[:, t:-1]).sum(1) for t in range(block)], 1)[..., None]
    for got, scale in zip(ts.paged_dequantize(c, torch.float32), (c.k_scales, c.v_scales)):
        err = (got[0].double() - x).abs()
        if held == INT8:
            assert (err <= (2.5 + 2.0 ** -10) * last).all(), float((err / last).max())
        else:
            own = (1 + 2.0 ** -4) ** (since + 1) - 1
            assert (err <= (own * x.abs() + 6.7 * 2.0 ** -10 * last) * (1 + 2.0 ** -10)).all()
            assert (err <= (0.146 * 448 + 6.7 * 2.0 ** -10) * last * (1 + 2.0 ** -10)).all()


def worst_growths(tokens):
    """Loudness of `tokens` tokens that makes an e4m3 code of the first drift upwards, found step by step by the
    formulas: (loudness, the value's place among the first token's, its drift in the end)."""
    start = torch.arange(128, 256, dtype=torch.float32) / 256                  # the first token: 0.5 to 1
    inv = torch.tensor(1.0 / 448.0, dtype=torch.float32)
    loud, scale = [1.0], inv.clone()
    codes = (start * (1 / scale)).to(E4M3).float()
    at = int((codes * scale / start).argmax())                                 # the value that starts off highest
    code = codes[at]
    for _ in range(tokens - 1):
        steps = torch.arange(1.25, 1.56, 1 / 128)
        more = (loud[-1] * steps).bfloat16().float()
        more = more[more * inv >= 1.25 * scale]
        new = more * inv
        got = (code * (scale / new)).to(E4M3).float()
        best = int((got * new).argmax())
        loud.append(float(more[best]))
        scale, code = new[best], got[best]
    return loud, at, float(code * scale / start[at]) - 1


def test_codes_of_floating_point_drift_with_every_growth():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as ts
    for tokens in (4, 8, 16):
        loud, at, drift = worst_growths(tokens)
        c = ts.PagedKVCache8.allocate(1, 1, 128, 16, page_size=16, dtype=E4M3)
        first = (torch.arange(128, 256, device="cuda") / 256).bfloat16()
        for t, a in enumerate(loud):
            x = torch.zeros(1, 1, 1, 128, device="cuda", dtype=torch.bfloat16)
            x[..., 0] = a
            if t == 0:
                x = first.clone().view(1, 1, 1, 128)
                x[..., 0 if at != 0 else 1] = 1.0
            ts.paged_append(x, x, c)
            c.advance()
        got = float(ts.paged_dequantize(c, torch.float32)[0][0, 0, 0, at]) / float(first[at]) - 1
        assert abs(got - drift) <= 2.0 ** -20
        assert got <= (1 + 2.0 ** -4) ** tokens - 1
        # five half steps, what integers can drift at most, are less than this
        assert tokens < 16 or got > 5 * 2.0 ** -4
