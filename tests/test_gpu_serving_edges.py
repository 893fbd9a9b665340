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


def run_in_thread(f):
    import threading
    out = []
    t = threading.Thread(target=lambda: out.append(f()))
    t.start()
    t.join()
    return out[0]


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_small_batch_of_another_thread_leaves_room_for_a_large_one(ts, d):
    """The kernel's shared memory grows with the batch; how much it may have is
    one setting for all threads."""
    def attend(batch):
        c = filled_cache(ts, [30] * batch, d=d, track=False)
        qkv = torch.ones(batch, 8 * d, dtype=torch.bfloat16, device="cuda")
        return ts.paged_decode_attention(qkv, 4, c)
    want = attend(300)
    assert run_in_thread(lambda: attend(1).shape) == (1, 4 * d)
    assert torch.equal(attend(300), want)


def test_batches_at_the_kernels_limit(ts):
    """A block has 227 KB: 1 KB for the kernel's own variables, 98304 + 4352 bytes for
    stages and queries of 128 columns, 8 for a sequence and 4 more. That is room for
    16095 sequences; without the variables it would be 16223."""
    c = ts.PagedKVCache.allocate(16223, 1, 128, 1, 1)
    qkv = torch.randn(16223, 3 * 128, device="cuda").to(torch.bfloat16)
    with pytest.raises(NotImplementedError, match="batch too large"):
        ts.paged_decode_attention(qkv, 1, c)
    n = 16095
    fit = ts.PagedKVCache(c.k_pages, c.v_pages, c.page_table[:n], c.seq_lens[:n])
    assert torch.equal(ts.paged_decode_attention(qkv[:n], 1, fit), qkv[:n, 256:])
    assert torch.equal(c.v_pages[:n].view(n, 128), qkv[:n, 256:])
def in_threads(jobs, rounds):
    """Runs every job `rounds` times, each in a thread of its own, all on the
    default stream; returns the lists of their results."""
    import threading
    results, errors = [[] for _ in jobs], []
    start = threading.Barrier(len(jobs))

    def work(i):
        try:
            start.wait()
            for _ in range(rounds):
                results[i].append(jobs[i]())
        except Exception as e:                               # (an assertion here would be lost in the thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    return results


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_threads_on_one_stream_multiply_their_own_tokens(ts, fmt):
    """More tokens than the product quantises itself: quantiser and product are
    two launches with the tokens' codes between them."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = ts.fp4_quantize(torch.randn(640, 1024, generator=g, device="cuda"), fmt)
    xs = [torch.randn(40, 1024, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3)]
    want = [ts.fp4_linear(x, w) for x in xs]
    got = in_threads([lambda x=x: ts.fp4_linear(x, w) for x in xs], 300)
    for y, ys in zip(want, got):
        assert all(torch.equal(y, z) for z in ys)


def test_threads_on_one_stream_accumulate_their_own_weights(ts):
    """Attention leaves logits and sums for the kernel that adds up the weights."""
    pos = torch.tensor([300, 20], device="cuda")
    caches = [filled_cache(ts, [300, 20], seed=i) for i in range(3)]
    qkv = [torch.randn(2, 12 * 64, device="cuda").to(torch.bfloat16) for _ in range(3)]
    before = [c.scores.clone() for c in caches]

    def step(c, q):
        return ts.paged_decode_attention(q, 8, c, pos, accumulate=True), c.scores.clone()

    serial = [[step(c, q) for _ in range(200)] for c, q in zip(caches, qkv)]
    for c, s in zip(caches, before):
        c.scores.copy_(s)
    got = in_threads([lambda c=c, q=q: step(c, q) for c, q in zip(caches, qkv)], 200)
    for want, have in zip(serial, got):
        assert all(torch.equal(a, b) and torch.equal(s, t) for (a, s), (b, t) in zip(want, have))


def test_threads_on_one_stream_evict_from_their_own_caches(ts):
    """The selection leaves lists for the kernel that moves the slots."""
    def build(seed):
        return [filled_cache(ts, [600, 500], d=32, seed=seed * 100 + i) for i in range(40)]

    serial, threaded = [build(i) for i in range(3)], [build(i) for i in range(3)]
    for caches in serial:
        for c in caches:
            ts.paged_evict(c, 200, 10)
    todo = [list(caches) for caches in threaded]
    in_threads([lambda q=q: ts.paged_evict(q.pop(), 200, 10) for q in todo], 40)
    for a, b in zip(serial, threaded):
        for x, y in zip(a, b):
            for name in ("k_pages", "v_pages", "scores", "slot_pos", "seq_lens"):
                assert torch.equal(getattr(x, name), getattr(y, name)), name


def test_status_of_a_stalled_product_leaves_other_streams_alone(ts):
    """Attention on a side stream, joined through arrival counters, is on its way
    while a product that stalled is reported and cleared."""
    from tensorshrink_b200 import _C, kernels
    a = ts.fp4_quantize(torch.randn(1, 1024, device="cuda").to(torch.bfloat16))
    b = ts.fp4_quantize(torch.randn(9500, 1024, device="cuda"))
    c = filled_cache(ts, [9000, 40], n_kv=4, d=128, page=64, track=False)
    qkv = torch.randn(2, 24 * 128, device="cuda").to(torch.bfloat16)
    product, want = ts.fp4_matmul(a, b), ts.paged_decode_attention(qkv, 16, c)
    side = torch.cuda.Stream()
    kernels.device_status()
    for _ in range(3):
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            early = [ts.paged_decode_attention(qkv, 16, c) for _ in range(600)]
        assert _C.load().ts_test_inject_stall(1_000_000) == 0
        ts.fp4_matmul(a, b)
        with pytest.raises(RuntimeError, match="ts_fp4_status"):
            kernels.device_status()
        with torch.cuda.stream(side):
            late = [ts.paged_decode_attention(qkv, 16, c) for _ in range(50)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in early + late)
        kernels.device_status()
        assert torch.equal(ts.fp4_matmul(a, b), product)


def test_status_of_a_workspace_made_in_inference_mode(ts):
    from tensorshrink_b200 import _C, kernels
    side = torch.cuda.Stream()
    a, b = (ts.fp4_quantize(torch.randn(n, 1024, device="cuda")) for n in (1, 9500))
    want = ts.fp4_matmul(a, b)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.inference_mode():
            ts.fp4_matmul(a, b)
        assert _C.load().ts_test_inject_stall(1_000_000) == 0
        ts.fp4_matmul(a, b)
        with pytest.raises(RuntimeError, match="ts_fp4_status"):
            kernels.device_status()
        kernels.device_status()
        assert torch.equal(ts.fp4_matmul(a, b), want)


def test_operators_keep_their_schemas(ts):
    """What an operator writes and returns is what its schema says, and fake tensors get the same shapes."""
    from torch.library import opcheck
    ops = torch.ops.tensorshrink
    x, one = torch.randn(40, 200, device="cuda").to(torch.bfloat16), torch.full((1,), 0.01, device="cuda")
    c = filled_cache(ts, [30, 20], room=20)
    pos = c.seq_lens.long()
    kv, qkv = torch.randn(2, 3, 2, 64, device="cuda").to(torch.bfloat16), torch.randn(2, 8 * 64, device="cuda").to(torch.bfloat16)
    cache = (c.k_pages, c.v_pages, c.page_table, c.seq_lens, c.scores, c.slot_pos)
    tests = ("test_schema", "test_faketensor")
    for fmt in (0, 1):
        for g in ((None, one) if fmt == 0 else (None,)):
            codes, scales, found = ops.fp4_quantize(x, fmt, g)
            opcheck(ops.fp4_quantize.default, (x, fmt, g), test_utils=tests)
        g = found if g is None else g
        opcheck(ops.fp4_dequantize.default, (codes, scales, g, 40, 200, fmt, torch.float32), test_utils=tests)
        opcheck(ops.fp4_matmul.default, (codes, scales, g, 40, codes, scales, g, 40, 200, fmt, None, torch.float16), test_utils=tests)
        opcheck(ops.fp4_linear.default, (x, codes, scales, g, 40, 200, fmt, None, None, None), test_utils=tests)
    opcheck(ops.paged_append.default, (kv, kv, *cache, pos, None, None, None, None), test_utils=tests)
    attend = (qkv, 4, *cache, pos, None, None, None, True)
    opcheck(ops.paged_decode_attention.default, attend, test_utils=tests)
    opcheck(ops.paged_decode_attention.out, attend, dict(out=torch.empty(2, 256, device="cuda", dtype=torch.bfloat16)),
            test_utils=tests)
    opcheck(ops.paged_evict.default, (*cache, 16, 2), test_utils=tests)


def test_a_compiled_module_runs_the_operator(ts):
    w = ts.fp4_quantize(torch.randn(128, 256, device="cuda"))
    layer = ts.Fp4Linear(w, torch.randn(128, device="cuda"))
    f = torch.compile(lambda x: torch.nn.functional.silu(layer(x)), backend="aot_eager", fullgraph=True, dynamic=True)
    for m in (3, 40, 41):
        x = torch.randn(m, 256, device="cuda").to(torch.bfloat16)
        with torch.no_grad():
            assert torch.equal(f(x), torch.nn.functional.silu(layer(x)))


def test_gradients_are_refused_not_dropped(ts):
    x = torch.randn(4, 256, device="cuda", requires_grad=True)
    w = ts.fp4_quantize(torch.nn.Parameter(torch.randn(128, 256, device="cuda")))
    y = ts.fp4_linear(x, w)
    assert torch.equal(y.detach(), ts.fp4_linear(x.detach(), w))
    with pytest.raises(RuntimeError, match="derivative for tensorshrink::fp4_linear is not implemented"):
        y.sum().backward()
    assert not w.global_scale.requires_grad


def test_a_cast_module_multiplies_as_before(ts):
    layer = ts.Fp4Linear(ts.fp4_quantize(torch.randn(128, 256, device="cuda")))
    x = torch.randn(3, 256, device="cuda").to(torch.bfloat16)
    layer.calibrate(x)
    want = layer(x)
    for dtype in (torch.bfloat16, torch.float16, torch.float64):
        assert torch.equal(layer.to(dtype)(x), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,d", [([1500, 40], 64), ([700, 3], 128), ([300, 65], 256)])
def test_attention_weights_have_both_their_terms(ts, dtype, lens, d):
    """Against 64 bits with weights in two terms of the cache's type: the result's
    rounding, half a unit (2^-8 of it in bf16, with 8 bits, 2^-11 in fp16, with 11);
    2^-15 of sum p |v| for the weights' rounding (2^-16, 2^-22) and fp32 arithmetic on
    scores of this size (2^-16); where fp16 weights underflow, 2^-25 of max |v| a
    slot. One term alone would be off by up to 2^-8 (2^-11) of sum p |v|: 12 to 25%
    of the results outside the bound in bf16, up to 8% in fp16 (short sequences)."""
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    g = torch.Generator(device="cuda").manual_seed(d)
    c = ts.PagedKVCache.allocate(2, 2, d, max(lens) + 1, 16, dtype=dtype)
    for t in (c.k_pages, c.v_pages):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    qkv = torch.randn(2, 10 * d, generator=g, device="cuda").to(dtype)
    got = ts.paged_decode_attention(qkv, 6, c).double().view(2, 2, 3, d)
    for b, n in enumerate(lens):
        t = torch.arange(n + 1, device="cuda")
        page = c.page_table[b, t // 16].long()
        k, v = c.k_pages[page, :, t % 16].double(), c.v_pages[page, :, t % 16].double()
        q = qkv[b].double().view(10, d)[:6].view(2, 3, d)
        p = (torch.einsum("hgd,thd->hgt", q, k) * d ** -0.5).softmax(-1)
        want, size = torch.einsum("hgt,thd->hgd", p, v), torch.einsum("hgt,thd->hgd", p, v.abs())
        off = 2.0 ** -15 * size + (0 if dtype == torch.bfloat16 else (n + 1) * 2.0 ** -25 * v.abs().max())
        assert ((got[b] - want).abs() <= half * (want.abs() + off) + off + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d", [(0, 64), (1, 64), (40, 128), (900, 64), (300, 256)])
def test_infinite_values_come_out_as_the_formula_has_them(ts, dtype, n, d):
    """sum p v with an infinity in v is that infinity, with two of unlike sign or a
    NaN it is NaN, and the other columns are finite."""
    c = ts.PagedKVCache.allocate(1, 1, d, n + 1, 16, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(n)
    for t in (c.k_pages, c.v_pages):
        t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 0.2)
    c.seq_lens.fill_(n)
    qkv = (torch.randn(1, 6 * d, generator=g, device="cuda") * 0.2).to(dtype)
    clean = ts.paged_decode_attention(qkv, 4, c).view(4, d)
    inf, nan = float("inf"), float("nan")
    qkv[0, 5 * d] = inf                                      # the new token's v
    want = {0: inf}
    if n:
        v = c.v_pages.view(-1, d)
        for col, slots in ((1, {0: inf}), (2, {n - 1: -inf}), (3, {n // 2: nan}), (4, {0: inf, n - 1: inf}),
                           (d - 1, {n // 3: -inf})):
            for s, x in slots.items():
                v[s, col] = x
            want[col] = x
        if n > 1:
            v[0, 5], v[n - 1, 5] = inf, -inf
            want[5] = nan
    got = ts.paged_decode_attention(qkv, 4, c).view(4, d)
    for col in range(d):
        if col not in want:
            assert torch.equal(got[:, col], clean[:, col]), col
        else:
            assert torch.equal(got[:, col].nan_to_num(nan=7.0), torch.full_like(got[:, col], want[col]).nan_to_num(nan=7.0)), col


def test_nothing_to_do(ts):
    c = filled_cache(ts, [30, 20])
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.scores, c.slot_pos, c.seq_lens)]
    kv = torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    ts.paged_append(kv, kv, c, pos, scores=torch.zeros(2, 2, 0, device="cuda"))
    kv = torch.ones(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    ts.paged_append(kv[:, 3:], kv[:, 3:], c)
    ts.paged_append(kv, kv, c, n_new=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(before, (c.k_pages, c.v_pages, c.scores, c.slot_pos, c.seq_lens)))
    for none in (ts.PagedKVCache(c.k_pages, c.v_pages, c.page_table[:0], c.seq_lens[:0], c.scores, c.slot_pos),
                 ts.PagedKVCache.allocate(0, 2, 64, 32, 16, track=True)):
        qkv = torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device="cuda")
        out = ts.paged_decode_attention(qkv, 4, none, pos[:0], accumulate=True)
        assert out.shape == (0, 256) and out.dtype == torch.bfloat16
        ts.paged_append(kv[:0], kv[:0], none, pos[:0])
        ts.paged_evict(none, 4, 1)
    w = ts.fp4_quantize(torch.randn(8, 64, device="cuda"))
    empty = ts.fp4_quantize(torch.zeros(0, 64, device="cuda"))
    assert ts.fp4_matmul(empty, w).shape == (0, 8) and ts.fp4_matmul(w, empty).shape == (8, 0)
    assert ts.fp4_linear(torch.zeros(2, 0, 64, device="cuda"), w).shape == (2, 0, 8)
    assert ts.fp4_dequantize(empty).shape == (0, 64)


def test_rotary_tables_without_rows_are_refused(ts):
    """They used to count as no tables: keys were stored without their rotation."""
    c = filled_cache(ts, [30, 20])
    before = c.k_pages.clone()
    none, pos = torch.zeros(0, 32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    qkv = torch.ones(2, 8 * 64, dtype=torch.bfloat16, device="cuda")
    kv = torch.ones(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="rotary tables are empty"):
        ts.paged_decode_attention(qkv, 4, c, pos, none, none)
    with pytest.raises(ValueError, match="rotary tables are empty"):
        ts.paged_append(kv, kv, c, pos, none, none)
    assert torch.equal(before, c.k_pages)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_compiled_step_over_the_cache_is_the_step(ts, backend):
    """Append, attention and eviction traced as one graph: what they write is written."""
    a, b = (filled_cache(ts, [20, 9], room=40) for _ in range(2))
    pos = a.seq_lens.long()

    def step(cache, qkv, kv, pos):
        ts.paged_append(kv, kv, cache, pos)
        cache.advance(5)
        y = ts.paged_decode_attention(qkv, 4, cache, pos + 5, accumulate=True)
        cache.advance()
        ts.paged_evict(cache, 12, 2)
        return y * 2
    compiled = torch.compile(step, backend=backend, fullgraph=True)
    for _ in range(3):
        qkv, kv = torch.randn(2, 8 * 64, device="cuda").to(torch.bfloat16), torch.randn(2, 5, 2, 64, device="cuda").to(torch.bfloat16)
        with torch.no_grad():
            assert torch.equal(step(a, qkv, kv, pos), compiled(b, qkv, kv, pos))
        for name in ("k_pages", "v_pages", "scores", "slot_pos", "seq_lens"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
