"""The 8-bit decode attention at its largest batches: a call that is refused stores nothing.

A block has 227 KB: 64 bytes for the kernel's own variables, 1024 to align, 196608 + 96 + 4224 + 32 for stages, barriers, queries and
their powers of 256 columns, 8 for a sequence and 4 more: room for 3799 sequences.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_refused_step_stores_nothing(held, dtype):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as ts
    n, d = 3900, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    c = ts.PagedKVCache8.allocate(n, 1, d, 16, page_size=16, dtype=held)
    first = torch.randn(n, 3, 1, d, generator=g, device="cuda").to(dtype)
    ts.paged_append(first, first, c)
    c.advance(3)
    before = [t.clone() for t in c._args()]
    qkv = torch.randn(n, 3 * d, generator=g, device="cuda").to(dtype) * 20          # (scales would grow)
    out = torch.full((n, d), 3.0, device="cuda", dtype=dtype)
    with pytest.raises(NotImplementedError, match="batch too large"):
        ts.paged_decode_attention(qkv, 1, c, out=out)
    assert (out == 3).all() and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, c._args()))
    # as many as there is room for: the same as in two halves
    n = 3700
    parts = [ts.PagedKVCache8(*(t.clone() for t in c._args()[:4]), c.page_table[s], c.seq_lens[s])
             for s in (slice(0, n), slice(0, n // 2), slice(n // 2, n))]
    whole = ts.paged_decode_attention(qkv[:n], 1, parts[0])
    halves = [ts.paged_decode_attention(qkv[s], 1, p) for s, p in zip((slice(0, n // 2), slice(n // 2, n)), parts[1:])]
    assert torch.equal(whole, torch.cat(halves))
    assert torch.equal(parts[0].k_scales[:n // 2], parts[1].k_scales[:n // 2]) and (parts[0].k_scales[:n] > before[2][:n]).all()
