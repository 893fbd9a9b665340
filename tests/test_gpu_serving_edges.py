"""The serving operators where calls meet: kernels of one call, threads of one
program, streams of one device, sequences that take no part."""

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


def filled_cache(ts, lens, n_kv=2, d=64, page=16, room=8, seed=1, track=True):
    """A cache of random content, its pages dealt out in order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ts.PagedKVCache.allocate(len(lens), n_kv, d, max(max(lens), 0) + room, page, track=track)
    c.k_pages.copy_(torch.randn(c.k_pages.shape, generator=g, device="cuda"))
    c.v_pages.copy_(torch.randn(c.v_pages.shape, generator=g, device="cuda"))
    c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    if track:
        c.scores.copy_(torch.rand(c.scores.shape, generator=g, device="cuda"))
        c.slot_pos.copy_(torch.randint(0, 1000, c.slot_pos.shape, generator=g, device="cuda"))
    return c


@pytest.mark.parametrize("lens", [[-1], [-1] * 70, [24, 24], [-1, 24, -5]])
def test_zeros_of_sequences_that_take_no_part_are_there_for_the_next_kernel(ts, lens):
    """Nobody takes part (marked, or full: the capacity is 24 or 32 slots): the
    kernel that adds up weights has nothing to do, and what follows it still
    finds the attention's zeros."""
    c = filled_cache(ts, [max(n, 0) for n in lens], page=8, room=0 if max(lens) > 0 else 24)
    c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    nq, n = 64, len(lens)
    qkv = torch.randn(n, (nq + 4) * 64, device="cuda").to(torch.bfloat16)
    pos = torch.zeros(n, dtype=torch.int64, device="cuda")
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.scores, c.slot_pos)]
    seen = []
    out = torch.empty(n, nq * 64, dtype=torch.bfloat16, device="cuda")
    for _ in range(50):
        out.fill_(1.0)
        ts.paged_decode_attention(qkv, nq, c, pos, accumulate=True, out=out)
        seen.append(out.clone())
    assert all((o == 0).all() for o in seen)
    assert all(torch.equal(x, y) for x, y in zip(before, (c.k_pages, c.v_pages, c.scores, c.slot_pos)))
