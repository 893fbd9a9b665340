"""The paged decoder at the ends of its tables and caches."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def build(batch=2, **kw):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tensorshrink_b200.decoder import DecoderConfig
    from tensorshrink_b200.serving import PagedDecoder
    cfg = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, intermediate=512, vocab=500, seed=3)
    return PagedDecoder(cfg, "cuda", max_batch=batch, page_size=16, **kw)


def prompts(lens, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 500, (n,), generator=g) for n in lens]


def state(m):
    return [t.clone() for c in m.caches for t in (c.k_pages, c.v_pages, c.seq_lens, c.scores, c.slot_pos) if t is not None]


def test_a_full_cache_raises():
    m = build(max_len=32)
    token = m.prefill(prompts([7, 30]))
    assert m.steps_left == 2
    for _ in range(2):
        token = m.decode_step(token)
    before = state(m)
    with pytest.raises(RuntimeError, match="32 of 32 tokens"):
        m.decode_step(token)
    assert all(torch.equal(x, y) for x, y in zip(before, state(m)))
    assert m.positions.tolist() == [9, 32]
    m.prefill(prompts([7, 9]))                               # a new prompt starts anew
    assert m.steps_left == 23


def test_the_last_rotary_row_raises():
    m = build(max_len=64, budget=16, recent=4, max_position=40)
    token = m.prefill(prompts([38, 5]))
    assert m.steps_left == 2
    m.decode_step(m.decode_step(token))
    with pytest.raises(RuntimeError, match="40 of 40 tokens"):
        m.decode_step(token)
    with pytest.raises(ValueError, match="1 to 40 tokens"):
        m.prefill(prompts([41, 5]))


def test_a_budget_goes_on_beyond_max_len_by_default():
    """Every kept slot is a token's own: positions are distinct and the newest are among them."""
    a, b = build(max_len=48, budget=24, recent=8), build(max_len=48, budget=24, recent=8, max_position=300)
    x, y = a.prefill(prompts([20, 40])), b.prefill(prompts([20, 40]))
    for step in range(100):
        x, y = a.decode_step(x), b.decode_step(y)
        assert torch.equal(x, y), step
    assert a.positions.tolist() == [120, 140] and a.steps_left == a.LONG - 140
    for c in a.caches:
        s = torch.arange(24, device="cuda")
        for i, last in enumerate((120, 140)):
            pos = c.slot_pos[c.page_table[i, s // 16].long(), :, s % 16]
            for h in range(2):
                have = set(pos[:, h].tolist())
                assert len(have) == 24 and set(range(last - 8, last)) <= have and max(have) == last - 1


@pytest.mark.parametrize("kw", [dict(max_len=32), dict(max_len=64, budget=16, recent=4, max_position=32)])
def test_replays_past_the_end_leave_the_cache(kw):
    m = build(**kw)
    m.prefill(prompts([10, 29]))
    tok = torch.zeros(2, dtype=torch.long, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.decode_step(tok)
    assert m.steps_left == 3                                 # the capture ran nothing
    lens = []
    for _ in range(3):
        m.count_steps()
        graph.replay()
    assert m.steps_left == 0
    with pytest.raises(RuntimeError):
        m.count_steps()
    own = m.caches[1].page_table[1].long()
    kept = [t[own].clone() for t in (m.caches[1].k_pages, m.caches[1].v_pages)]
    lens = [c.seq_lens[1].item() for c in m.caches]
    for _ in range(5):                                       # uncounted
        graph.replay()
    torch.cuda.synchronize()
    assert [c.seq_lens[1].item() for c in m.caches] == lens
    assert all(torch.equal(x, t[own]) for x, t in zip(kept, (m.caches[1].k_pages, m.caches[1].v_pages)))
    assert m.caches[0].seq_lens[0].item() == (18 if m.budget is None else 16)


def test_a_dropped_sequence_lets_the_others_go_on():
    m, alone = build(max_len=32), build(max_len=32)
    ps = prompts([7, 31])
    a, b = m.prefill(ps, return_logits=True), alone.prefill([ps[0], ps[0]], return_logits=True)
    m.decode_step(a.argmax(-1))
    alone.decode_step(a.argmax(-1)[:1].repeat(2))
    with pytest.raises(RuntimeError, match="drop"):
        m.decode_step(a.argmax(-1))
    m.drop(1)
    assert m.steps_left == 24
    before = m.caches[0].k_pages[m.caches[0].page_table[1].long()].clone()
    tok = torch.tensor([3, 4], device="cuda")
    for _ in range(24):
        x, y = m.decode_step(tok, return_logits=True), alone.decode_step(tok[:1].repeat(2), return_logits=True)
        assert torch.equal(x[0], y[0])
    assert m.steps_left == 0 and [c.seq_lens.tolist() for c in m.caches] == [[32, -1]] * 2
    assert torch.equal(before, m.caches[0].k_pages[m.caches[0].page_table[1].long()])
    m.prefill(ps)
    assert m.steps_left == 1 and m.caches[0].seq_lens.tolist() == [7, 31]
