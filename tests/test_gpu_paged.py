"""The paged key-value cache on the GPU: appending, attention of one new token
and eviction, against plain 64-bit (attention) or exact (the rest)
restatements.

Tolerance of an attention output in type T with unit roundoff e (2^-9 for
bf16, 2^-12 for fp16): the weights are rounded to T for their product with v (e
per term, plus T's smallest spacing where it underflows), the result once more;
fp32 arithmetic on scores of this size adds 2^-16: |err| <= 2 e |o| + (2 e + 2^-15)
sum p |v| + n 2^-24 max|v|. Accumulated weights stay in fp32: 2^-15 of the weight
and 2^-23 of the score.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


def tables(n, d):
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
    ang = torch.outer(torch.arange(n, device="cuda", dtype=torch.float32), inv)
    return ang.cos().contiguous(), ang.sin().contiguous()


def rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


def make(ts, lens, n_kv, d, page, dtype, seed, room=1, layout="heads", track=True, spare=2):
    """A cache of random content whose sequences have room for `room` more tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-(max(n, 0) + room) // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (total, n_kv, page, d) if layout == "heads" else (total, page, n_kv, d)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    if layout != "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    scores = torch.rand(total, n_kv, page, generator=g, device="cuda") if track else None
    pos = torch.randint(0, 1000, (total, n_kv, page), generator=g, device="cuda", dtype=torch.int32) if track else None
    return ts.PagedKVCache(k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scores, pos)


def clone(ts, c):
    def cp(t):
        return None if t is None else t.clone()
    return ts.PagedKVCache(cp(c.k_pages), cp(c.v_pages), c.page_table.clone(), c.seq_lens.clone(), cp(c.scores),
                           cp(c.slot_pos))


def reference(c, qkv, nq, positions, cos, sin, scale, accumulate):
    """Attention in 64 bits over the cache as the call finds it; the new token
    is put into `c` (a copy). Returns (out, tolerance, score additions)."""
    h, d, page = c.n_kv, c.head_dim, c.k_pages.shape[2]
    B = c.batch
    out = torch.zeros(B, nq, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    e = E[qkv.dtype]
    add = torch.zeros_like(c.scores, dtype=torch.float64) if c.scores is not None else None
    table = c.page_table.cpu().numpy()
    total = c.k_pages.shape[0]
    for b in range(B):
        n = int(c.seq_lens[b])
        if n < 0 or n >= table.shape[1] * page:
            continue
        p_new = table[b, n // page]
        if not 0 <= p_new < total:
            continue
        x = qkv[b].view(nq + 2 * h, d)
        q, k, v = x[:nq], x[nq:nq + h], x[nq + h:]
        if cos is not None:
            pos = int(positions[b])
            if not 0 <= pos < cos.shape[0]:
                continue
            q, k = rotate(q, cos[pos], sin[pos]), rotate(k, cos[pos], sin[pos])
        c.k_pages[p_new, :, n % page] = k
        c.v_pages[p_new, :, n % page] = v
        if c.scores is not None:
            c.scores[p_new, :, n % page] = 0
        if c.slot_pos is not None:
            c.slot_pos[p_new, :, n % page] = int(positions[b])
        slots = np.arange(n + 1)
        pg = table[b, slots // page]
        live = (pg >= 0) & (pg < total)
        pg, off = pg[live], (slots % page)[live]
        pt, ot = torch.from_numpy(pg).long().cuda(), torch.from_numpy(off).cuda()
        for j in range(h):
            kk, vv = c.k_pages[pt, j, ot].double(), c.v_pages[pt, j, ot].double()
            qs = q[j * (nq // h):(j + 1) * (nq // h)].double()
            p = torch.softmax(qs @ kk.t() * scale, -1)
            sl = slice(j * (nq // h), (j + 1) * (nq // h))
            out[b, sl] = p @ vv
            tol[b, sl] = 2 * e * out[b, sl].abs() + (2 * e + 2.0 ** -15) * (p @ vv.abs()) + len(pg) * 2.0 ** -24 * vv.abs().max()
            if accumulate:
                add[pt, j, ot] += p.sum(0)
    return out.reshape(B, -1), tol.reshape(B, -1), add


def check_attention(ts, c, nq, dtype, seed, rope=True, accumulate=False, scale=None, positions=None):
    g = torch.Generator(device="cuda").manual_seed(seed + 77)
    h, d = c.n_kv, c.head_dim
    wide = torch.randn(c.batch, (nq + 2 * h) * d + 8, generator=g, device="cuda").to(dtype)
    qkv = wide[:, :(nq + 2 * h) * d]                     # rows with a stride of their own
    if positions is None:
        positions = c.seq_lens.long().clamp(min=0) + 3
    cos, sin = tables(int(positions.max()) + 2, d) if rope else (None, None)
    ref = clone(ts, c)
    want, tol, add = reference(ref, qkv, nq, positions, cos, sin, d ** -0.5 if scale is None else scale, accumulate)
    got = ts.paged_decode_attention(qkv, nq, c, positions, cos, sin, scale=scale, accumulate=accumulate)
    assert got.dtype == dtype
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol.clamp(min=1e-30)).max().item():.3g} tolerances"
    assert torch.equal(c.k_pages, ref.k_pages) and torch.equal(c.v_pages, ref.v_pages)
    assert torch.equal(c.seq_lens, ref.seq_lens)
    if c.scores is not None:
        total = ref.scores.double() + (add if add is not None else 0)
        err = (c.scores.double() - total).abs()
        bound = 2.0 ** -15 * (add if add is not None else 0) + 2.0 ** -22 * total
        assert (err <= bound).all()
        assert torch.equal(c.slot_pos, ref.slot_pos)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("d,page", [(16, 16), (64, 1), (80, 7), (96, 64), (128, 16), (128, 100), (192, 32), (256, 64)])
def test_attention_shapes(ts, dtype, layout, d, page):
    c = make(ts, [0, 1, 15, 16, 63, 64, 65, 130, 400], 2, d, page, dtype, d + page, layout=layout)
    check_attention(ts, c, 8, dtype, 1, accumulate=True)


@pytest.mark.parametrize("nq,h", [(1, 1), (2, 2), (7, 1), (12, 4), (16, 1), (17, 1), (40, 2), (71, 1)])
def test_attention_head_groups(ts, nq, h):
    c = make(ts, [5, 200, 33], h, 128, 16, torch.bfloat16, nq)
    check_attention(ts, c, nq, torch.bfloat16, 2, accumulate=True)


@pytest.mark.parametrize("lens", [[0], [1], [5000], [9000, 3], [700] * 40, [0] * 300, [1, 2, 3] * 100, [-1, 50, -1], [-1]])
def test_attention_lengths(ts, lens):
    c = make(ts, lens, 4, 64, 32, torch.bfloat16, len(lens), track=len(lens) < 10)
    check_attention(ts, c, 8, torch.bfloat16, 3, accumulate=len(lens) < 10)


def test_attention_without_rotation_and_with_a_scale(ts):
    c = make(ts, [40, 300], 2, 128, 16, torch.bfloat16, 8, track=False)
    check_attention(ts, c, 8, torch.bfloat16, 4, rope=False, scale=0.3)


def test_sequences_that_cannot_take_the_token(ts):
    c = make(ts, [10, 64, 20, 30, 128], 2, 64, 64, torch.bfloat16, 9, track=True)
    c.page_table[1, 1] = -1                     # no page for slot 64
    c.page_table[4, 2:] = 10 ** 6               # a page outside the pool
    pos = torch.tensor([10, 64, 10 ** 6, -1, 5], device="cuda")    # two positions without a rotary row
    cos, sin = tables(100, 64)
    before = clone(ts, c)
    qkv = torch.randn(5, 8 * 64, device="cuda").to(torch.bfloat16)
    ref = clone(ts, c)
    want, tol, add = reference(ref, qkv, 4, pos, cos, sin, 0.125, True)
    got = ts.paged_decode_attention(qkv, 4, c, pos, cos, sin, accumulate=True)
    assert ((got.double() - want).abs() <= tol).all()
    assert (got[1:] == 0).all() and (got[0] != 0).any()
    assert torch.equal(c.k_pages, ref.k_pages)
    assert ((c.scores != before.scores).sum((0, 2)) <= 11).all()
    # a full table
    full = make(ts, [63], 1, 64, 64, torch.bfloat16, 3, room=1)
    full.page_table = full.page_table[:, :1].contiguous()
    full = ts.PagedKVCache(full.k_pages, full.v_pages, full.page_table, full.seq_lens + 1, full.scores, full.slot_pos)
    out = ts.paged_decode_attention(qkv[:1, :6 * 64], 4, full, pos[:1], cos, sin)
    assert (out == 0).all()


def test_holes_in_the_table_carry_no_weight(ts):
    c = make(ts, [200, 200], 2, 64, 16, torch.bfloat16, 10)
    c.page_table[0, 3] = -1
    c.page_table[0, 0] = 10 ** 6
    c.page_table[1, :12] = -1                   # only the new token's page is left
    check_attention(ts, c, 4, torch.bfloat16, 5, accumulate=True)


def test_nothing_behind_the_length_is_read(ts):
    """NaN in unused slots and pages, and in the new token's slot before it is written."""
    c = make(ts, [0, 17, 100, 63], 2, 128, 16, torch.bfloat16, 11)
    used = torch.zeros(c.k_pages.shape[0], 16, dtype=torch.bool, device="cuda")
    for b, n in enumerate([0, 17, 100, 63]):
        for s in range(n):
            used[int(c.page_table[b, s // 16]), s % 16] = True
    dead = ~used[:, None, :, None].expand_as(c.k_pages)
    c.k_pages[dead] = float("nan")
    c.v_pages[dead] = float("inf")
    c.scores[~used[:, None, :].expand_as(c.scores)] = float("nan")
    g = torch.Generator(device="cuda").manual_seed(5)
    qkv = torch.randn(4, 12 * 128, generator=g, device="cuda").to(torch.bfloat16)
    cos, sin = tables(200, 128)
    ref = clone(ts, c)
    want, tol, _ = reference(ref, qkv, 8, c.seq_lens.long(), cos, sin, 128 ** -0.5, True)
    got = ts.paged_decode_attention(qkv, 8, c, c.seq_lens.long(), cos, sin, accumulate=True)
    assert ((got.double() - want).abs() <= tol).all()
    for b, n in enumerate([0, 17, 100, 63]):
        assert c.scores[int(c.page_table[b, n // 16]), :, n % 16].isfinite().all()


def test_peaked_and_infinite_scores(ts):
    """One key far above the rest; keys that drive scores to -inf leave the others' weights alone."""
    c = make(ts, [150], 1, 64, 16, torch.bfloat16, 12, track=False)
    qkv = torch.randn(1, 4 * 64, device="cuda").to(torch.bfloat16)
    c.k_pages[int(c.page_table[0, 2]), 0, 5] = 40 * qkv[0, :64]
    check = clone(ts, c)
    want, tol, _ = reference(check, qkv, 2, None, None, None, 1.0, False)
    got = ts.paged_decode_attention(qkv, 2, c, scale=1.0)
    assert ((got.double() - want).abs() <= tol).all()
    c.k_pages[int(c.page_table[0, 1]), 0, 3] = -float("inf")
    q = torch.ones(1, 4 * 64, device="cuda", dtype=torch.bfloat16)
    check = clone(ts, c)
    want, tol, _ = reference(check, q, 2, None, None, None, 0.1, False)
    got = ts.paged_decode_attention(q, 2, c, scale=0.1)
    live = (want.isfinite()).all()
    assert not live or ((got.double() - want).abs() <= tol.nan_to_num(1.0, 1.0, 1.0) + 2.0 ** -8).all()


def test_attention_repeats_and_leaves_the_workspace(ts):
    runs = []
    for lens, h, d, nq in [([3000, 5], 2, 128, 8), ([17] * 60, 8, 64, 8), ([4000], 1, 256, 5)]:
        c = make(ts, lens, h, d, 32, torch.bfloat16, d, track=False)
        qkv = torch.randn(len(lens), (nq + 2 * h) * d, device="cuda").to(torch.bfloat16)
        runs.append((qkv, nq, c, ts.paged_decode_attention(qkv, nq, c)))
    for _ in range(3):
        for qkv, nq, c, want in runs:
            assert torch.equal(ts.paged_decode_attention(qkv, nq, c), want)


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("d,page", [(16, 5), (64, 16), (128, 64), (256, 8)])
def test_append(ts, layout, d, page):
    lens, T, h = [0, 7, 130, -1], 37, 3
    c = make(ts, lens, h, d, page, torch.bfloat16, d, room=T, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(d)
    kv = torch.randn(4, T, 2 * h, d, generator=g, device="cuda").to(torch.bfloat16)
    k, v = kv[:, :, :h], kv[:, :, h:]                    # strided rows of a fused projection
    first = torch.tensor([0, 9, 2, 4], device="cuda")
    n_new = torch.tensor([T, 5, 0, 3], dtype=torch.int32, device="cuda")
    init = torch.rand(4, h, T, generator=g, device="cuda")
    cos, sin = tables(60, d)
    ref = clone(ts, c)
    for b, n in enumerate(lens):
        for t in range(int(n_new[b]) if n >= 0 else 0):
            p, o = int(ref.page_table[b, (n + t) // page]), (n + t) % page
            ref.k_pages[p, :, o] = rotate(k[b, t], cos[first[b] + t], sin[first[b] + t])
            ref.v_pages[p, :, o] = v[b, t]
            ref.scores[p, :, o] = init[b, :, t]
            ref.slot_pos[p, :, o] = int(first[b]) + t
    ts.paged_append(k, v, c, first, cos, sin, n_new=n_new, scores=init)
    for name in ("k_pages", "v_pages", "scores", "slot_pos", "seq_lens"):
        assert torch.equal(getattr(c, name), getattr(ref, name)), name


def test_append_drops_what_has_no_slot(ts):
    c = make(ts, [10], 1, 64, 8, torch.float16, 1, room=6)      # two pages, and a -1 behind them
    kv = torch.randn(1, 40, 1, 64, device="cuda").half()
    before = clone(ts, c)
    ts.paged_append(kv, kv, c)
    for s in range(10):
        p = int(c.page_table[0, s // 8])
        assert torch.equal(c.k_pages[p, 0, s % 8], before.k_pages[p, 0, s % 8])
    for s in range(10, 16):
        p = int(c.page_table[0, s // 8])
        assert torch.equal(c.k_pages[p, 0, s % 8], kv[0, s - 10, 0])
        assert c.scores[p, 0, s % 8] == 0 and c.slot_pos[p, 0, s % 8] == s
    rest = [i for i in range(c.k_pages.shape[0]) if i not in c.page_table[0, :2].tolist()]
    assert torch.equal(c.k_pages[rest], before.k_pages[rest])


def evict_reference(c, budget, recent):
    table, page, h = c.page_table.cpu().numpy(), c.k_pages.shape[2], c.n_kv
    total = c.k_pages.shape[0]
    for b in range(c.batch):
        n = min(int(c.seq_lens[b]), table.shape[1] * page)
        if n <= budget:
            continue
        pg, off = table[b, np.arange(n) // page], np.arange(n) % page
        live = (pg >= 0) & (pg < total)
        for j in range(h):
            w = np.full(n, np.nan)
            pos = np.full(n, -1, np.int64)
            w[live] = c.scores[torch.from_numpy(pg[live]).long().cuda(), j, torch.from_numpy(off[live]).cuda()].cpu().numpy()
            pos[live] = c.slot_pos[torch.from_numpy(pg[live]).long().cuda(), j, torch.from_numpy(off[live]).cuda()].cpu().numpy()
            w[np.isnan(w)] = -np.inf
            w[live & (pos > pos[live].max(initial=-2 ** 31) - recent)] = np.inf
            order = sorted(range(n), key=lambda i: (not live[i], -w[i], i))
            stay = set(order[:budget])
            fr = [i for i in range(budget, n) if i in stay]
            to = [i for i in range(budget) if i not in stay]
            assert len(fr) == len(to)
            for a, z in zip(fr, to):
                if not (live[a] and live[z]):
                    continue
                for t in (c.k_pages, c.v_pages, c.scores, c.slot_pos):
                    t[int(pg[z]), j, int(off[z])] = t[int(pg[a]), j, int(off[a])]
        c.seq_lens[b] = budget


def check_evict(ts, c, budget, recent):
    ref = clone(ts, c)
    evict_reference(ref, budget, recent)
    ts.paged_evict(c, budget, recent)
    for name in ("k_pages", "v_pages", "scores", "slot_pos", "seq_lens"):
        assert torch.equal(getattr(c, name).nan_to_num(), getattr(ref, name).nan_to_num()), name


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("d,page", [(16, 1), (64, 16), (128, 24), (256, 64)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (40, 0), (64, 10), (100, 100), (129, 3)])
def test_evict(ts, layout, d, page, budget, recent):
    c = make(ts, [0, 1, 40, 65, 130, 131, 300, -1], 2, d, page, torch.bfloat16, budget + d, layout=layout)
    check_evict(ts, c, budget, recent)


def test_evict_ties_nan_and_signs(ts):
    c = make(ts, [90, 90, 90, 90], 1, 64, 16, torch.float16, 4)
    t = c.page_table.long()
    c.scores[t[0, :6]] = 0.5                                     # all equal: the lowest slots stay
    c.scores[t[1, :3]] = float("nan")
    c.scores[t[2, :6]] = torch.randn_like(c.scores[t[2, :6]])
    c.scores[t[2, 1]] = -0.0
    c.scores[t[2, 3]] = 0.0
    c.scores[t[3, 2]] = float("inf")
    c.scores[t[3, 4]] = -float("inf")
    check_evict(ts, c, 33, 4)


def test_evict_with_holes_in_the_table(ts):
    c = make(ts, [200, 64], 2, 64, 16, torch.bfloat16, 6)
    c.page_table[0, 2] = -1
    c.page_table[0, 9] = 10 ** 6
    check_evict(ts, c, 100, 20)


def test_evict_of_a_long_sequence(ts):
    """More slots than fit the selection's shared memory."""
    c = make(ts, [60000, 3000], 1, 16, 64, torch.bfloat16, 7)
    check_evict(ts, c, 2048, 100)


def test_decode_and_evict_over_steps(ts):
    """A cache held at its budget over decode steps, against the reference step by step."""
    c = make(ts, [60, 20], 2, 64, 16, torch.bfloat16, 13, room=40)
    for b in range(2):                                           # positions of the cached tokens: their slots
        for s in range(int(c.seq_lens[b])):
            c.slot_pos[int(c.page_table[b, s // 16]), :, s % 16] = s
    pos = c.seq_lens.long().clone()
    for step in range(6):
        check_attention(ts, c, 8, torch.bfloat16, step, accumulate=True, positions=pos.clone())
        c.advance()
        pos += 1
        check_evict(ts, c, 48, 8)
    assert c.seq_lens.tolist() == [48, 26]


def test_captured_in_a_graph(ts):
    c = make(ts, [100, 30], 2, 64, 16, torch.bfloat16, 14, room=8)
    eager = clone(ts, c)
    qkv = torch.randn(2, 12 * 64, device="cuda").to(torch.bfloat16)
    cos, sin = tables(300, 64)

    def step(cache, pos):
        out = ts.paged_decode_attention(qkv, 8, cache, pos, cos, sin, accumulate=True)
        cache.advance()
        ts.paged_evict(cache, 101, 8)
        pos.add_(1)
        return out

    p0, p1 = (torch.tensor([200, 30], device="cuda") for _ in range(2))
    saved = clone(ts, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(c, p1)
    torch.cuda.synchronize()
    for name in ("k_pages", "v_pages", "scores", "slot_pos", "seq_lens"):
        getattr(c, name).copy_(getattr(saved, name))
    p1.copy_(p0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step(c, p1)
    for _ in range(4):
        want = step(eager, p0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    for name in ("k_pages", "scores", "slot_pos", "seq_lens"):
        assert torch.equal(getattr(c, name), getattr(eager, name)), name


def test_captured_without_a_warm_up(ts):
    """Graphs of one stream do not depend on calls outside of them, nor on one another's order."""
    c = make(ts, [300, 30], 2, 64, 16, torch.bfloat16, 15, room=8)
    qkv = [torch.randn(2, 12 * 64, device="cuda").to(torch.bfloat16) for _ in range(2)]
    want = [ts.paged_decode_attention(q, 8, clone(ts, c), c.seq_lens.long()) for q in qkv]
    pos = c.seq_lens.long()
    s = torch.cuda.Stream()
    graphs, got = [], []
    for q in qkv:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            got.append(ts.paged_decode_attention(q, 8, c, pos))
    with torch.cuda.stream(s):
        outside = ts.paged_decode_attention(qkv[0], 8, c, pos)
    torch.cuda.synchronize()
    assert torch.equal(outside, want[0])
    for i in (1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(got[i], want[i]), i


def test_evict_keeps_recent_slots_beside_infinite_scores(ts):
    c = make(ts, [90], 1, 64, 16, torch.bfloat16, 16)
    t = c.page_table.long()[0]
    c.scores[t[:5]] = float("inf")                               # 80 slots, more than the budget
    for i in range(90):
        c.slot_pos[t[i // 16], 0, i % 16] = i
    newest = set(range(86, 90))
    ts.paged_evict(c, 33, 4)
    pos = [int(c.slot_pos[t[i // 16], 0, i % 16]) for i in range(33)]
    assert newest <= set(pos) and len(set(pos)) == 33


def test_refusals(ts):
    c = make(ts, [5, 9], 2, 64, 16, torch.bfloat16, 1)
    plain = make(ts, [5, 9], 2, 64, 16, torch.bfloat16, 1, track=False)
    qkv = torch.randn(2, 8 * 64, device="cuda").to(torch.bfloat16)
    pos = torch.zeros(2, dtype=torch.int64, device="cuda")
    cos, sin = tables(20, 64)
    kv = torch.randn(2, 3, 2, 64, device="cuda").to(torch.bfloat16)
    for bad, err in [(lambda: ts.paged_decode_attention(qkv, 3, c, pos), ValueError),
                     (lambda: ts.paged_decode_attention(qkv, 4, c), ValueError),
                     (lambda: ts.paged_decode_attention(qkv.half(), 4, c, pos), ValueError),
                     (lambda: ts.paged_decode_attention(qkv[:1], 4, c, pos), ValueError),
                     (lambda: ts.paged_decode_attention(qkv, 4, c, pos.int()), ValueError),
                     (lambda: ts.paged_decode_attention(qkv, 4, c, pos, cos), ValueError),
                     (lambda: ts.paged_decode_attention(qkv, 4, c, pos, cos[:, :8], sin[:, :8]), ValueError),
                     (lambda: ts.paged_decode_attention(qkv, 4, plain, pos, accumulate=True), ValueError),
                     (lambda: ts.paged_decode_attention(qkv.cpu(), 4, c, pos), RuntimeError),
                     (lambda: ts.paged_append(kv[:1], kv[:1], c), ValueError),
                     (lambda: ts.paged_append(kv.half(), kv.half(), c), ValueError),
                     (lambda: ts.paged_append(kv, kv, plain, scores=torch.zeros(2, 2, 3, device="cuda")), ValueError),
                     (lambda: ts.paged_evict(plain, 4), ValueError),
                     (lambda: ts.paged_evict(c, 0), ValueError),
                     (lambda: ts.paged_evict(c, 4, 5), ValueError),
                     (lambda: ts.PagedKVCache(c.k_pages, c.v_pages[:, :1], c.page_table, c.seq_lens), ValueError),
                     (lambda: ts.PagedKVCache(c.k_pages, c.v_pages, c.page_table.long(), c.seq_lens), ValueError),
                     (lambda: ts.PagedKVCache(c.k_pages.float(), c.v_pages.float(), c.page_table, c.seq_lens), NotImplementedError),
                     (lambda: ts.paged_decode_attention(torch.zeros(2, 8 * 40, device="cuda").to(torch.bfloat16), 4,
                                                        ts.PagedKVCache.allocate(2, 2, 40, 32)), NotImplementedError)]:
        with pytest.raises(err):
            bad()
