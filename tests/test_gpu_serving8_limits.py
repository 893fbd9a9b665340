"""Steps that nobody counts, of sequences past their last rotary row, with norms of queries and keys."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(batch=3, **kw):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tensorshrink_b200.decoder import DecoderConfig
    from tensorshrink_b200.serving import PagedDecoder
    cfg = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=512, vocab=500, seed=3)
    return PagedDecoder(cfg, "cuda", max_batch=batch, page_size=16, qk_norm=True, **kw)


def cached(m, b, tokens):
    """What sequence b's first `tokens` slots hold, in all layers."""
    out = []
    for c in m.caches:
        slot = torch.arange(tokens, device="cuda")
        page, off = c.page_table[b, slot // 16].long(), slot % 16
        for name in ("k_pages", "v_pages", "scores", "slot_pos"):
            t = getattr(c, name, None)
            if t is not None:
                out.append(t[page, :, off].clone().view(torch.uint8))
        for name in ("k_scales", "v_scales"):
            if hasattr(c, name):
                out.append(getattr(c, name)[page].clone())
        out.append(c.seq_lens.clone()[b])
    return out


@pytest.mark.parametrize("kw", [dict(max_len=64, budget=16, recent=4, max_position=40), dict(max_len=96, max_position=40),
                                dict(max_len=96, max_position=40, cache_dtype=torch.int8),
                                dict(max_len=96, max_position=40, cache_dtype=torch.int8, pages=14)])
def test_a_sequence_past_its_limit_keeps_its_cache(kw):
    g = torch.Generator().manual_seed(1)
    m = build(**kw)
    token = m.prefill([torch.randint(0, 500, (n,), generator=g) for n in (38, 5, 30)])
    for _ in range(2):
        token = m.decode_step(token)
    assert m.positions.tolist() == [40, 7, 32]
    lens = m.caches[0].seq_lens.tolist()
    before = cached(m, 0, lens[0])
    for step in range(4):
        m._tokens = [0] * 3                          # (as replays of a captured step go by)
        token = m.decode_step(token)
    assert m.caches[0].seq_lens.tolist() == [lens[0], min(lens[1] + 4, 16 if "budget" in kw else 99), min(lens[2] + 4, 16 if "budget" in kw else 99)]
    assert all(torch.equal(x, y) for x, y in zip(before, cached(m, 0, lens[0])))
