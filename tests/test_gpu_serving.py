"""The paged decoder over 4-bit floating-point projections: ragged prompts,
decode steps against prefill, a bounded cache, and a captured step."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

PROMPTS = [5, 33, 12, 1]


def build(budget=None, recent=0, fmt="nvfp4"):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tensorshrink_b200.decoder import DecoderConfig
    from tensorshrink_b200.serving import PagedDecoder
    cfg = DecoderConfig(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, intermediate=1024, vocab=1000, seed=5)
    return PagedDecoder(cfg, "cuda", format=fmt, max_batch=len(PROMPTS), max_len=80, page_size=16, budget=budget,
                        recent=recent, max_position=200)


def prompts(extra=0, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n + extra,), generator=g) for n in PROMPTS]


def first_layer(m, b, n):
    """Keys and values of sequence b's first n tokens in the first layer."""
    c = m.caches[0]
    t = torch.arange(n, device="cuda")
    page, off = c.page_table[b, t // 16].long(), t % 16
    return c.k_pages[page, :, off].double(), c.v_pages[page, :, off].double()


def same_tokens(x, y):
    """The first layer sees the embeddings alone, so both runs project the same
    4-bit codes; only the order of fp32 sums may differ, and with it a bf16
    result by one unit (2^-7 of its size). Rotated halves mix: a pair is off by
    at most 2^-7 (|x1| + |x2|), and another 2^-8 of each from rounding again, in all
    below 2^-5.5 of the pair's norm."""
    k, v = x
    k2, v2 = y
    half = k.shape[-1] // 2
    norm = (k[..., :half].square() + k[..., half:].square()).sqrt().repeat(1, 1, 2)
    assert ((k - k2).abs() <= 2.0 ** -5.5 * norm).all()
    assert ((v - v2).abs() <= 2.0 ** -7 * v.abs()).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_ragged_prompts_are_cached_as_prompts_alone(fmt):
    m = build(fmt=fmt)
    ps = prompts()
    m.prefill(ps)
    assert m.positions.tolist() == PROMPTS and m.caches[1].seq_lens.tolist() == PROMPTS
    together = [first_layer(m, i, n) for i, n in enumerate(PROMPTS)]
    for i, n in enumerate(PROMPTS):
        m.prefill([ps[i]] * len(ps))
        same_tokens(first_layer(m, 2, n), together[i])
    assert m.positions.tolist() == [PROMPTS[-1]] * len(PROMPTS)


def test_decode_steps_cache_what_prefill_does():
    m, other = build(), build()
    full = prompts(extra=3)
    m.prefill([p[:-3] for p in full])
    for t in (3, 2, 1):
        m.decode_step(torch.stack([p[-t] for p in full]).cuda())
    other.prefill(full)
    assert m.caches[0].seq_lens.tolist() == [n + 3 for n in PROMPTS]
    assert m.positions.tolist() == other.positions.tolist()
    for i, n in enumerate(PROMPTS):
        same_tokens(first_layer(m, i, n + 3), first_layer(other, i, n + 3))


def test_bounded_cache():
    m = build(budget=24, recent=8)
    token = m.prefill(prompts())
    assert m.caches[0].seq_lens.tolist() == [min(n, 24) for n in PROMPTS]
    for step in range(1, 40):
        token = m.decode_step(token)
        assert m.caches[1].seq_lens.tolist() == [min(n + step, 24) for n in PROMPTS]
    assert (token >= 0).all() and (token < 1000).all()
    # the newest positions are all there, each once
    cache = m.caches[0]
    for b, n in enumerate(PROMPTS):
        s = torch.arange(24, device="cuda")
        pos = cache.slot_pos[cache.page_table[b, s // 16].long(), :, s % 16]
        for h in range(2):
            have = pos[:, h].tolist()
            assert len(set(have)) == 24 and set(range(n + 39 - 8, n + 39)) <= set(have)


def test_a_budget_that_holds_everything_changes_nothing():
    a, b = build(), build(budget=70, recent=3)
    ta, tb = a.prefill(prompts(), return_logits=True), b.prefill(prompts(), return_logits=True)
    assert torch.equal(ta, tb)
    tok = ta.argmax(-1)
    for _ in range(4):
        la, lb = a.decode_step(tok, return_logits=True), b.decode_step(tok, return_logits=True)
        assert torch.equal(la, lb)
        tok = la.argmax(-1)


def test_captured_step_equals_eager():
    eager, graphed = build(budget=30, recent=4), build(budget=30, recent=4)
    t0 = eager.prefill(prompts())
    assert torch.equal(graphed.prefill(prompts()), t0)
    tok = t0.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graphed.decode_step(tok)
    torch.cuda.synchronize()
    graphed.prefill(prompts())                      # the warm-up moved the caches on
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        tok.copy_(graphed.decode_step(tok))
    want = t0
    for _ in range(12):
        want = eager.decode_step(want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, want)


def test_refusals():
    m = build()
    with pytest.raises(ValueError):
        m.prefill(prompts()[:2])
    with pytest.raises(ValueError):
        m.prefill([torch.zeros(0, dtype=torch.long)] * 4)
    with pytest.raises(ValueError):
        build(budget=80)
    with pytest.raises(ValueError):
        build(budget=10, recent=11)
