"""The paged decoder in 8 bits: int8 projections, norms of queries and keys, a cache
of 8 bits, pages that the sequences share.

Integer sums do not depend on the batch, so the first layer's keys and
values (which see the embeddings alone) are the same bits however a token came in.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

PROMPTS = [5, 33, 12, 1]
E4M3 = torch.float8_e4m3fn


def build(cache_dtype=torch.int8, qk_norm=True, pages=None, fmt="int8", max_len=80, **kw):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tensorshrink_b200.decoder import DecoderConfig
    from tensorshrink_b200.serving import PagedDecoder
    cfg = DecoderConfig(n_layers=2, hidden=512, n_heads=8, n_kv_heads=2, intermediate=1024, vocab=1000, seed=5)
    m = PagedDecoder(cfg, "cuda", format=fmt, max_batch=len(PROMPTS), max_len=max_len, page_size=16, cache_dtype=cache_dtype,
                     qk_norm=qk_norm, pages=pages, **kw)
    if qk_norm:
        g = torch.Generator(device="cuda").manual_seed(3)
        for layer in m.layers:
            for w in (layer.q_norm, layer.k_norm):
                w.data.copy_(1 + 0.2 * torch.randn(w.shape, generator=g, device="cuda"))
    return m


def prompts(extra=0, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n + extra,), generator=g) for n in PROMPTS]


def first_layer(m, b, n):
    """Keys, values and their scales of sequence b's first n tokens in the first layer."""
    import tensorshrink_b200 as ts
    c = m.caches[0]
    t = torch.arange(n, device="cuda")
    page, off = c.page_table[b, t // 16].long(), t % 16
    if isinstance(c, ts.PagedKVCache8):
        k, v = ts.paged_dequantize(c, torch.float32)
        return k[page, :, off], v[page, :, off], c.k_scales[page, :, off // 16], c.v_scales[page, :, off // 16]
    return c.k_pages[page, :, off].float(), c.v_pages[page, :, off].float()


@pytest.mark.parametrize("qk_norm", [True, False])
@pytest.mark.parametrize("pages", [None, 9, 40])
def test_shared_pages_hold_what_own_pages_do(qk_norm, pages):
    # bf16: page for page the same bits as the caches that deal their pages out up front
    a, b = build(torch.bfloat16, qk_norm, pages or 20), build(torch.bfloat16, qk_norm)
    assert a.packed and not b.packed
    full = prompts(extra=3)
    if pages == 9:
        with pytest.raises(ValueError):                           # 1 + 3 + 1 + 1 pages; 15 more tokens need 9, 30 do not fit
            a.prefill([torch.cat([p] * 4) for p in full])
    for m in (a, b):
        m.prefill([p[:-3] for p in full])
        for t in (3, 2, 1):
            m.decode_step(torch.stack([p[-t] for p in full]).cuda())
    assert a.caches[1].seq_lens.tolist() == [n + 3 for n in PROMPTS]
    for i, n in enumerate(PROMPTS):
        for x, y in zip(first_layer(a, i, n + 3), first_layer(b, i, n + 3)):
            assert torch.equal(x, y)
    used = sum(-(-(n + 3) // 16) for n in PROMPTS)
    assert int(a.pool.n_free) == (pages or 20) - used


@pytest.mark.parametrize("cache_dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("pages", [None, 12])
def test_the_cache_of_8_bits_holds_the_tokens(cache_dtype, pages):
    m, wide = build(cache_dtype, pages=pages), build(torch.bfloat16)
    full = prompts(extra=20)
    for x in (m, wide):
        x.prefill([p[:-20] for p in full])
        for t in range(20, 0, -1):
            x.decode_step(torch.stack([p[-t] for p in full]).cuda())
    for i, n in enumerate(PROMPTS):
        k8, v8, ks, vs = first_layer(m, i, n + 20)
        k, v = first_layer(wide, i, n + 20)
        for got, want, s in ((k8, k, ks), (v8, v, vs)):
            if cache_dtype == torch.int8:
                # half a step of rounding, and 2.5 of a scale that grew
                assert ((got - want).abs() <= 3.001 * s[..., None]).all()
            else:
                # half a step is 2^-4 of a value (or 2^-10 of a scale); after growth five of them at most
                assert ((got - want).abs() <= 5 * (2.0 ** -4 * want.abs() + 2.0 ** -10 * s[..., None])).all()


def test_a_step_retraced_with_the_operators():
    import tensorshrink_b200 as ts
    from tensorshrink_b200.serving import _rms_norm
    m, other = build(pages=20), build(pages=20)
    tok = m.prefill(prompts())
    assert torch.equal(other.prefill(prompts()), tok)
    for _ in range(3):
        logits = m.decode_step(tok, return_logits=True)
        c0, n_q, n_kv, D = other.caches[0], 8, 2, 64
        got = ts.paged_reserve(other.pool, c0, torch.ones(4, dtype=torch.int32, device="cuda"), 4)
        assert got.positions.tolist() == other.positions.tolist() and got.sequences.tolist() == [0, 1, 2, 3]
        h = other.embed[tok].float()
        for layer, cache in zip(other.layers, other.caches):
            qkv = ts.int8_linear(_rms_norm(h, layer.input_norm, other.cfg.rms_eps), layer.qkv.weight())
            qkv = ts.qk_norm_rope(qkv, n_q, n_kv, layer.q_norm, layer.k_norm, got.positions, other.rope_cos, other.rope_sin,
                                  other.cfg.rms_eps)
            q, k, v = qkv.view(4, -1, D).split([n_q, n_kv, n_kv], dim=1)
            ts.paged_append(k, v, cache, offsets=got.offsets)
            cache.seq_lens += 1
            a = ts.paged_attention(q.reshape(4, -1), cache)
            cache.seq_lens -= 1
            h = other._mlp(layer, h + layer.o(a))
        c0.advance(got.granted)
        other.positions += 1
        assert torch.equal(other._logits(h), logits)
        for x, y in zip(m.caches, other.caches):
            assert torch.equal(x.k_pages, y.k_pages) and torch.equal(x.v_scales, y.v_scales)
        tok = logits.argmax(-1)
    # one layer's attention against 64 bits over the values that its cache holds: the tokens' own weights
    cache = m.caches[1]
    n = int(cache.seq_lens[1])
    q = torch.randn(4, n_q * D, device="cuda").bfloat16()
    kk, vv = ts.paged_dequantize(cache, torch.float32)
    t = torch.arange(n, device="cuda")
    page, off = cache.page_table[1, t // 16].long(), t % 16
    k, v = (x[page, :, off].double().transpose(0, 1) for x in (kk, vv))
    w = torch.softmax(q[1].double().view(2, 4, D) @ k.transpose(1, 2) * D ** -0.5, -1)
    err = (ts.paged_attention(q, cache)[1].double().view(2, 4, D) - w @ v).abs()
    assert (err <= 2.0 ** -8 * (w @ v).abs() + 2.0 ** -10 * (w @ v.abs())).all()


@pytest.mark.parametrize("kw", [dict(), dict(pages=30), dict(cache_dtype=E4M3, pages=30, qk_norm=False),
                                dict(cache_dtype=torch.bfloat16, pages=30), dict(fmt="nvfp4", pages=30)])
def test_captured_step_equals_eager(kw):
    eager, graphed = build(**kw), build(**kw)
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
    for _ in range(20):
        want = eager.decode_step(want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, want)
    if eager.pages:
        assert torch.equal(eager.pool.n_free, graphed.pool.n_free)


def test_pages_run_out_and_come_back():
    m = build(pages=8)
    tok = m.prefill(prompts())                      # 1 + 3 + 1 + 1 pages; 11 more tokens: 1 + 3 + 2 + 1; 16: 2 + 4 + ..
    assert int(m.pool.n_free) == 2
    left = m.steps_left
    lens = list(PROMPTS)
    assert sum(-(-(n + left) // 16) for n in lens) <= 8 < sum(-(-(n + left + 1) // 16) for n in lens)
    for _ in range(left):
        tok = m.decode_step(tok)
    with pytest.raises(RuntimeError, match="pages"):
        m.decode_step(tok)
    m.drop(1)                                       # the longest goes, the others go on with its pages
    assert int(m.pool.n_free) >= 3 and m.caches[0].seq_lens[1] == -1 and m.steps_left > 0
    before = [int(x) for x in m.caches[0].seq_lens]
    for _ in range(m.steps_left):
        tok = m.decode_step(tok)
    after = m.caches[0].seq_lens.tolist()
    assert after[1] == -1 and all(b > a for i, (a, b) in enumerate(zip(before, after)) if i != 1)
    # uncounted replays past the pool: a sequence that gets no page keeps its cache
    for _ in range(40):
        m._tokens = [0] * 4                         # (as replays of a captured step go by)
        tok = m.decode_step(tok)
    used = sum(-(-max(0, n) // 16) for n in m.caches[0].seq_lens.tolist())
    assert used <= 8 and int(m.pool.n_free) >= 0
    m.prefill(prompts())
    assert int(m.pool.n_free) == 2 and m.caches[0].seq_lens.tolist() == PROMPTS


def test_norms_with_a_budget():
    m = build(torch.bfloat16, budget=24, recent=8, max_position=200)
    plain = build(torch.bfloat16)
    tok = m.prefill(prompts())
    plain.prefill(prompts())
    k, _ = first_layer(plain, 0, 5)
    assert torch.equal(first_layer(m, 0, 5)[0], k)
    for _ in range(30):
        tok = m.decode_step(tok)
    assert m.caches[1].seq_lens.tolist() == [min(n + 30, 24) for n in PROMPTS]


def test_calibration_and_sizes():
    m = build(fmt="nvfp4", pages=20)
    m.calibrate(prompts())
    assert all(float(p.input_scale) < 1 for layer in m.layers for p in layer.projections())
    build().calibrate(prompts())                    # nothing to set
    assert build().packed_nbytes() > m.packed_nbytes()


def test_refusals():
    with pytest.raises(ValueError):
        build(budget=24)
    with pytest.raises(ValueError):
        build(torch.bfloat16, pages=10, budget=24)
    with pytest.raises(NotImplementedError):
        build(torch.float16)
    with pytest.raises(ValueError):
        build(pages=3).prefill(prompts())


def test_all_dropped():
    m = build(pages=20)
    m.prefill(prompts())
    for i in range(4):
        m.drop(i)
    assert int(m.pool.n_free) == 20 and m.steps_left == m.longest_sequence
    with pytest.raises(RuntimeError, match="decode steps"):
        m.count_steps(10 ** 6)
    m.decode_step(torch.zeros(4, dtype=torch.long, device="cuda"))
    assert m.caches[0].seq_lens.tolist() == [-1] * 4 and int(m.pool.n_free) == 20


def test_threads_share_a_stream():
    """Host threads call all operators on one stream, with tensors of their own."""
    import threading
    import tensorshrink_b200 as ts
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")

    def round_of(i):
        g = torch.Generator(device="cuda").manual_seed(i)
        w = ts.int8_quantize(torch.randn(16 * 64, 300, generator=g, device="cuda"))
        cache, pool = ts.PagedKVCache8.allocate(3, 4, 64, 96, page_size=32, dtype=(torch.int8, E4M3)[i % 2]), ts.PagePool.allocate(9)
        cache.page_table.fill_(-1)
        qw = torch.rand(64, generator=g, device="cuda")
        x = torch.randn(3, 300, generator=g, device="cuda").bfloat16()
        one = torch.ones(3, dtype=torch.int32, device="cuda")
        outs = []
        for _ in range(40):
            got = ts.paged_reserve(pool, cache, one, 3)
            qkv = ts.qk_norm_rope(ts.int8_linear(x, w), 8, 4, qw, qw)
            outs.append(ts.paged_decode_attention(qkv, 8, cache))
            cache.advance(got.granted)
            x = torch.roll(x, 1, 1)
        ts.paged_release(pool, cache, torch.zeros_like(one))
        return torch.stack(outs), pool.free.clone(), cache.seq_lens.clone()

    want = [round_of(i) for i in range(4)]
    found = [None] * 4
    torch.cuda.synchronize()

    def work(i):
        found[i] = round_of(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(want, found):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_schemas_hold():
    """What the operators write is what their schemas say, and their shapes under tracing are the real ones."""
    import tensorshrink_b200 as ts
    from tensorshrink_b200 import _C
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    ops, utils = _C.serving_ops(), ("test_schema", "test_faketensor")

    def check(op, *args, **kw):
        torch.library.opcheck(op, args, kw, test_utils=utils)
    x = torch.randn(5, 200, device="cuda").bfloat16()
    w = ts.int8_quantize(torch.randn(64, 200, device="cuda"))
    check(ops.int8_quantize.default, x)
    check(ops.int8_dequantize.default, w.codes, w.scales, 200, torch.float16)
    check(ops.int8_matmul.default, w.codes, w.scales, w.codes, w.scales, 200, None, torch.float32)
    check(ops.int8_linear.default, x, w.codes, w.scales, 200, None)
    qkv = torch.randn(4, 8 * 64, device="cuda").bfloat16()
    qw = torch.rand(64, device="cuda")
    check(ops.qk_norm_rope.default, qkv, 4, 2, qw, qw, None, None, None, 1e-6)
    check(ops.qk_norm_rope.out, qkv, 4, 2, qw, qw, None, None, None, 1e-6, out=torch.empty_like(qkv))
    c16 = ts.PagedKVCache.allocate(4, 2, 64, 64, page_size=16)
    check(ops.qk_norm_rope_store.default, qkv, 4, 2, qw, qw, None, None, None, 1e-6, *c16._args(),
          torch.arange(4, device="cuda"))
    c = ts.PagedKVCache8.allocate(4, 2, 64, 64, page_size=16)
    c.seq_lens.fill_(3)
    kv = qkv.view(4, 1, 8, 64)
    check(ops.paged8_append.default, kv[:, :, 4:6], kv[:, :, 6:], *c._args(), None, None, None, None, None)
    check(ops.paged8_dequantize.default, *c._args(), torch.bfloat16)
    check(ops.paged8_attention.default, qkv[:, :256], *c._args(), None, None, None, None)
    check(ops.paged8_decode_attention.default, qkv, 4, *c._args(), None, None, None, None)
    pool, one = ts.PagePool.allocate(8), torch.ones(4, dtype=torch.int32, device="cuda")
    c.page_table[:, 1:] = -1
    check(ops.paged_reserve.default, pool.free, pool.n_free, c.page_table, c.seq_lens, 16, 16, one * 20, None, 80)
    check(ops.paged_release.default, pool.free, pool.n_free, c.page_table, c.seq_lens, 16, 16, one)
