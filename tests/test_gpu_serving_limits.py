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


def prompt_weights64(q, k):
    """Weight that each key of one prompt draws, [tokens, n_kv] in 64 bits, and
    a bound on the error that fp32 scores make of it, as a part of the weight:
    a score is off by (D + 2) 2^-24 of sum |q||k| at most, a weight by twice
    that (numerator and denominator), and 2^-18 more from exponentials and sums."""
    n, heads, d = q.shape
    n_kv = k.shape[1]
    q = q.double().view(n, n_kv, heads // n_kv, d)
    s = torch.einsum("ihgd,jhd->hgij", q, k.double()) * d ** -0.5
    size = torch.einsum("ihgd,jhd->hgij", q.abs(), k.double().abs()).max().item() * d ** -0.5
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -float("inf"))
    return s.softmax(-1).sum((1, 2)).t(), 2 * (d + 2) * 2.0 ** -24 * size + 2.0 ** -18


@pytest.mark.parametrize("most", [None, 4000])
def test_prompts_are_cut_back_to_the_tokens_that_drew_attention(monkeypatch, most):
    """Against column sums in 64 bits of the first layer's own queries and keys."""
    import tensorshrink_b200.serving as serving
    if most is not None:                                     # many blocks of queries
        whole = serving._prompt_weights
        monkeypatch.setattr(serving, "_prompt_weights", lambda q, k, n: whole(q, k, n, most))
    lens, budget, recent = [90, 5, 41, 64], 40, 8
    m, full = build(batch=4, max_len=96, budget=budget, recent=recent), build(batch=4, max_len=96)
    for x in (m, full):                                      # six times the queries and keys: a few tokens draw most of it
        x.layers[0].qkv.global_scale.mul_(6)
    seen = []
    hook = full.layers[0].qkv.register_forward_hook(lambda _, x, y: seen.append(y))
    ps = prompts(lens, seed=9)
    m.prefill(ps)
    full.prefill(ps)
    hook.remove()
    qkv = seen[0].view(4, max(lens), 8, 64)
    c, f = m.caches[0], full.caches[0]
    middle = 0
    for b, n in enumerate(lens):
        cos, sin = full.rope_cos[:n, None], full.rope_sin[:n, None]
        x1, x2 = qkv[b, :n, :4].float().chunk(2, dim=-1)
        q = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1).to(qkv.dtype)
        t = torch.arange(n, device="cuda")
        k = f.k_pages[f.page_table[b, t // 16].long(), :, t % 16]
        want, off = prompt_weights64(q, k)
        s = torch.arange(min(n, budget), device="cuda")
        page = c.page_table[b, s // 16].long()
        pos, have = c.slot_pos[page, :, s % 16].long(), c.scores[page, :, s % 16].double()
        for h in range(2):
            kept = pos[:, h]
            assert len(set(kept.tolist())) == len(s)
            assert ((have[:, h] - want[kept, h]).abs() <= off * want[kept, h]).all()
            if n <= budget:
                continue
            gone = torch.ones(n, dtype=torch.bool, device="cuda")
            gone[kept] = False
            assert not gone[n - recent:].any()
            least = want[kept[kept < n - recent], h].min()
            assert least >= want[gone, h].max() * (1 - 2 * off)
            middle += int(((kept >= budget) & (kept < n - recent)).sum())
    assert middle > 0                                        # the first slots alone would not have done


def test_decoding_starts_from_the_prompts_weights():
    """A step adds its weights to the prompt's: kept scores sum up to one per
    query, of the prompt and of the step, and per query head of the kv head."""
    m = build(batch=2, max_len=96, budget=80, recent=4)
    token = m.prefill(prompts([30, 50]))
    for step in range(1, 4):
        token = m.decode_step(token)
        for c in m.caches:
            for b, n in enumerate((30 + step, 50 + step)):
                s = torch.arange(n, device="cuda")
                total = c.scores[c.page_table[b, s // 16].long(), :, s % 16].double().sum(0)
                assert ((total - 2 * n).abs() <= 2.0 ** -16 * 2 * n).all()


def projection_inputs(m, ps):
    """What each projection is given by a prefill, without the padding, and the prefill's logits."""
    seen, n = {}, [len(p) for p in ps]
    keep = (torch.arange(max(n)) < torch.tensor(n)[:, None]).cuda()
    names = {p: f"{i}.{name}" for i, layer in enumerate(m.layers) for name, p in zip(("qkv", "o", "gate_up", "down"),
                                                                                     layer.projections())}
    hooks = [p.register_forward_pre_hook(lambda p, args: seen.update({names[p]: (p, args[0][keep].clone())})) for p in names]
    logits = m.prefill(ps, return_logits=True)
    for h in hooks:
        h.remove()
    return seen, logits


def test_calibrated_scales_are_those_of_the_samples():
    """Each projection's scale is max|x| / 2688 of what a prefill of the samples
    gives it, and with it 4 bits hold the small activations behind the attention
    better than with 1, where block scales fall below E4M3's normal range."""
    import tensorshrink_b200 as ts
    m = build(max_len=64)
    ps = prompts([30, 17])
    before, _ = projection_inputs(m, ps)
    m.calibrate(ps)
    assert m.positions.tolist() == [30, 17] and m.caches[0].seq_lens.tolist() == [30, 17]
    after, logits = projection_inputs(m, ps)
    assert len(after) == 8
    for name, (proj, x) in after.items():
        assert proj.input_scale.item() == (x.float().abs().max() / 2688.0).item(), name

    one, small = torch.ones(1, device="cuda"), 0
    for name, (proj, x) in before.items():
        own = (x.float().abs().max() / 2688.0).reshape(1)
        blocks = x.float().reshape(x.shape[0], -1, 16)
        low = (blocks.abs().amax(-1) < 6 * 2.0 ** -7) & (blocks.abs().amax(-1) > 0)
        small += int(low.sum())

        def off(g):
            y = ts.fp4_dequantize(ts.fp4_quantize(x, "nvfp4", global_scale=g)).reshape(blocks.shape)
            return (y - blocks)[low].norm()
        assert low.sum() == 0 or off(own) < off(one), name
    assert small > 0
    again = m.prefill(ps, return_logits=True)
    assert torch.equal(again, logits)


def test_calibration_of_mxfp4_and_of_bad_samples():
    m = build(max_len=64, format="mxfp4")
    ps = prompts([30, 17])
    want = m.prefill(ps, return_logits=True)
    m.calibrate(ps)
    assert torch.equal(m.prefill(ps, return_logits=True), want)
    with pytest.raises(ValueError):
        m.calibrate(ps[:1])
    with pytest.raises(ValueError):
        m.calibrate([])
    assert not any(p._forward_pre_hooks for layer in m.layers for p in layer.projections())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_a_decode_step_is_its_parts(fmt):
    """A step retraced from what its projections got and gave: every part but the
    attention bit for bit, the attention against 64 bits over the cache that the
    step leaves. Its bound: rounding to the 8 bits of bf16, 2^-8 of the result;
    weights in two terms of bf16, 2^-8 of 2^-8 of each, and fp32 arithmetic on scores
    of this size, 2^-16: 2^-15 of sum p |v|. (A result left out, or of another layer,
    would be off by about 1 of the same; weights rounded once, by up to 2^-8.)"""
    import torch.nn.functional as F
    from tensorshrink_b200.decoder import _rms_norm
    m = build(batch=3, max_len=300, format=fmt)
    lens = [130, 1, 259]
    m.prefill(prompts(lens))
    names = {p: (i, name) for i, layer in enumerate(m.layers) for name, p in zip(("qkv", "o", "gate_up", "down"),
                                                                                 layer.projections())}
    seen = {}
    for p in names:
        p.register_forward_hook(lambda p, x, y: seen.update({names[p]: (x[0].clone(), y.clone())}))
    tokens = torch.tensor([7, 77, 377], device="cuda")
    logits = m.decode_step(tokens, return_logits=True)
    h = m.embed[tokens].float()
    for i, (layer, c) in enumerate(zip(m.layers, m.caches)):
        assert torch.equal(seen[i, "qkv"][0], _rms_norm(h, layer.input_norm, m.cfg.rms_eps))
        assert c.seq_lens.tolist() == [n + 1 for n in lens]
        for b, n in enumerate(lens):
            x = seen[i, "qkv"][1][b].view(8, 64)
            cos, sin = m.rope_cos[n], m.rope_sin[n]
            x1, x2 = x[:4].float().chunk(2, dim=-1)
            q = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1).to(x.dtype).double().view(2, 2, 64)
            t = torch.arange(n + 1, device="cuda")
            page = c.page_table[b, t // 16].long()
            k, v = c.k_pages[page, :, t % 16].double(), c.v_pages[page, :, t % 16].double()
            assert torch.equal(v[n], x[6:].double())
            p = (torch.einsum("hgd,thd->hgt", q, k) * 64 ** -0.5).softmax(-1)
            want = torch.einsum("hgt,thd->hgd", p, v).reshape(-1)
            size = torch.einsum("hgt,thd->hgd", p, v.abs()).reshape(-1)
            err = (seen[i, "o"][0][b].double() - want).abs()
            assert (err <= 2.0 ** -8 * (want.abs() + 2.0 ** -15 * size) + 2.0 ** -15 * size).all()
        h = h + seen[i, "o"][1]
        assert torch.equal(seen[i, "gate_up"][0], _rms_norm(h, layer.post_norm, m.cfg.rms_eps))
        gate, up = seen[i, "gate_up"][1].chunk(2, dim=-1)
        assert torch.equal(seen[i, "down"][0], F.silu(gate) * up)
        h = h + seen[i, "down"][1]
    assert torch.equal(logits, F.linear(_rms_norm(h, m.final_norm, m.cfg.rms_eps), m.lm_head).float())
