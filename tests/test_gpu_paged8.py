"""The paged cache of 8 bits on the GPU.

Appending is exact: codes and scales follow from fp32 operations that torch
rounds the same way. Attention is compared with 64 bits over the values that the
cache holds. Tolerance of an output o of type T: the result is rounded by half a step
(eps / 2 of T); weights enter their product in fp16, one term of 2^-11 for bf16
results, two (2^-22) for fp16; scores of this size, their exponentials and the sums over the
slots are fp32, 2^-14 of the weight together; weights under fp16's range (2^-35 of
the largest) are lost: |err| <= eps / 2 |o| + (u + 2^-14) sum p |v| + n 2^-35
max|v|, u = 2^-11 or 2^-22.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
TOP = {INT8: 127.0, E4M3: 448.0}


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


def encode(y, held):
    if held == INT8:
        return torch.round(y).clamp(-127, 127).to(INT8)
    return y.clamp(-448, 448).to(E4M3)


def make(ts, lens, n_kv, d, page, block, held, seed, room=1, layout="heads", spare=2):
    """A cache of random codes and scales whose sequences have pages for `room` more tokens."""
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
    k, v = (encode(torch.randn(shape, generator=g, device="cuda") * TOP[held] / 4, held) for _ in range(2))
    if layout != "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    ks, vs = (torch.exp(0.5 * torch.randn(total, n_kv, page // block, generator=g, device="cuda")) * 4 / TOP[held] for _ in range(2))
    return ts.PagedKVCache8(k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))


def raw(x):
    return x.view(torch.uint8) if x.is_contiguous() else x.transpose(1, 2).view(torch.uint8).transpose(1, 2)


def clone(ts, c):
    k, v = (t.clone() for t in (c.k_pages, c.v_pages))          # (strides are kept)
    return ts.PagedKVCache8(k, v, c.k_scales.clone(), c.v_scales.clone(), c.page_table.clone(), c.seq_lens.clone())


def same(a, b):
    assert torch.equal(raw(a.k_pages), raw(b.k_pages)) and torch.equal(raw(a.v_pages), raw(b.v_pages))
    for x, y in ((a.k_scales, b.k_scales), (a.v_scales, b.v_scales)):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(nan=3.0), y.nan_to_num(nan=3.0))
    assert torch.equal(a.page_table, b.page_table) and torch.equal(a.seq_lens, b.seq_lens)


def append(c, rows, which):
    """Stores rows[b]: a list of (slot, [n_kv, d]) of sequence b's tokens, by the formulas."""
    held, page, bs = c.k_pages.dtype, c.page_size, c.block
    codes, scales = (c.k_pages, c.k_scales) if which == "k" else (c.v_pages, c.v_scales)
    bits = raw(codes)
    for b, toks in enumerate(rows):
        blocks = {}
        for slot, x in toks:
            blocks.setdefault(slot // bs, []).append((slot, x))
        n = int(c.seq_lens[b])
        for blk, items in sorted(blocks.items()):
            p, o = int(c.page_table[b, blk * bs // page]), blk * bs % page
            x = torch.stack([i[1] for i in items], 1).float()                                # [n_kv, tokens, d]
            need = (x.abs().amax(dim=(1, 2)) * (1.0 / TOP[held])).clamp(min=2.0 ** -100)
            earlier = max(0, n - blk * bs)
            old = scales[p, :, o // bs].clone()
            s = need
            if earlier:
                s = torch.where(need > old, torch.maximum(need, 1.25 * old), old)
                grown = (need > old) & x.isfinite().all(dim=2).all(dim=1)                    # (else the codes are left alone)
                was = codes[p, :, o:o + earlier].float()
                again = encode(was * (old / s)[:, None, None], held)
                keep = torch.where(grown[:, None, None], again.view(torch.uint8), bits[p, :, o:o + earlier])
                bits[p, :, o:o + earlier] = keep
            bad = ~x.isfinite().all(dim=2).all(dim=1) | s.isnan()
            s = torch.where(bad, torch.full_like(s, math.nan), s)
            y = encode(torch.nan_to_num(x, 0, 0, 0) * (1.0 / s)[:, None, None].nan_to_num(0), held)
            y = torch.where(bad[:, None, None], torch.zeros_like(y.view(torch.uint8)), y.view(torch.uint8))
            for i, (slot, _) in enumerate(items):
                bits[p, :, o + slot - blk * bs] = y[:, i]
            scales[p, :, o // bs] = s


def places(c, b, count, positions=None, rope_rows=None):
    """Slots that `count` new tokens of sequence b go to (None: dropped)."""
    n = int(c.seq_lens[b])
    out = []
    for t in range(count):
        slot = n + t
        ok = 0 <= n and slot < c.capacity
        if ok:
            ok = 0 <= int(c.page_table[b, slot // c.page_size]) < c.k_pages.shape[0]
        pos = (int(positions[b]) if positions is not None else n) + t
        if rope_rows is not None:
            ok = ok and 0 <= pos < rope_rows
        out.append((slot if ok else None, pos))
    return out


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n_kv,d,page,block,layout", [(8, 128, 64, 16, "heads"), (2, 64, 16, 16, "tokens"), (1, 96, 64, 64, "tokens"),
                                                      (3, 16, 32, 32, "heads"), (2, 80, 48, 16, "heads"), (1, 256, 128, 128, "heads")])
def test_append(ts, n_kv, d, page, block, layout, dtype, held):
    lens = [0, 5, 16, 70, -1, 33]
    c = make(ts, lens, n_kv, d, page, block, held, 1, room=100, layout=layout)
    c.page_table[3, 96 // page] = -1                              # a page that is missing
    g = torch.Generator(device="cuda").manual_seed(2)
    for step, tokens in enumerate((1, 1, 37, 16)):
        loud = 2.0 ** (step - 1)                                  # scales have to grow
        k, v = (torch.randn(2, len(lens), tokens, n_kv, d, generator=g, device="cuda") * loud).to(dtype).unbind(0)
        want = clone(ts, c)
        rows = {w: [[(s, x[b, t]) for t, (s, _) in enumerate(places(c, b, tokens)) if s is not None] for b in range(len(lens))]
                for w, x in (("k", k), ("v", v))}
        append(want, rows["k"], "k")
        append(want, rows["v"], "v")
        ts.paged_append(k, v, c)
        same(c, want)
        c.advance(torch.where(c.seq_lens >= 0, tokens, 0).int())


@pytest.mark.parametrize("held", [INT8, E4M3])
def test_append_packed_counted_and_rotated(ts, held):
    n_kv, d = 2, 64
    lens = [3, 0, 20, 7, -1, 100]
    c = make(ts, lens, n_kv, d, 32, 16, held, 3, room=60)
    counts = [40, 1, 0, 17, 4, 30]
    off = [0]
    for n in counts:
        off.append(off[-1] + n)
    offsets = torch.tensor(off, dtype=torch.int32, device="cuda")
    wide = torch.randn(off[-1], 2 + 2 * n_kv, d, device="cuda").half()      # (strided rows: part of a projection's output)
    k, v = wide[:, 2:2 + n_kv], wide[:, 2 + n_kv:]
    cos, sin = tables(60, d)
    positions = torch.tensor([2, 9, 0, 50, 0, -4], device="cuda")            # some fall off either end of the tables
    n_new = torch.tensor([40, 5, 1, 15, 4, 0], dtype=torch.int32, device="cuda")
    want = clone(ts, c)
    rk, rv = [], []
    for b, n in enumerate(counts):
        pl = places(c, b, min(n, int(n_new[b])), positions, 60)
        rk.append([(s, rotate(k[off[b] + t], cos[p], sin[p])) for t, (s, p) in enumerate(pl) if s is not None])
        rv.append([(s, v[off[b] + t]) for t, (s, p) in enumerate(pl) if s is not None])
    append(want, rk, "k")
    append(want, rv, "v")
    ts.paged_append(k, v, c, positions, cos, sin, n_new, offsets=offsets)
    same(c, want)


@pytest.mark.parametrize("held", [INT8, E4M3])
def test_append_of_infinities_and_at_the_end_of_the_table(ts, held):
    n_kv, d = 2, 32
    c = make(ts, [4, 0, 30], n_kv, d, 16, 16, held, 5, room=8)
    k, v = torch.randn(2, 3, 20, n_kv, d, device="cuda").bfloat16().unbind(0)
    k[0, 3, 1, 5] = float("inf")
    v[1, 0, 0, 0] = float("nan")
    want = clone(ts, c)
    for which, x in (("k", k), ("v", v)):
        append(want, [[(s, x[b, t]) for t, (s, _) in enumerate(places(c, b, 20)) if s is not None] for b in range(3)], which)
    ts.paged_append(k, v, c)
    same(c, want)
    kk, vv = ts.paged_dequantize(c, torch.float32)
    p = int(c.page_table[0, 0])
    assert kk[p, 1].isnan().all() and kk[p, 0].isfinite().all() and vv[int(c.page_table[1, 0]), 0].isnan().all()
    # the NaN stays while the block is filled, and ends when it begins anew
    c.seq_lens.copy_(torch.tensor([10, 0, 0], dtype=torch.int32))
    ts.paged_append(k[:, :1].nan_to_num(0, 0, 0), v[:, :1].nan_to_num(0, 0, 0), c)
    assert c.k_scales[p, 1, 0].isnan() and c.v_scales[int(c.page_table[1, 0]), 0, 0].isfinite()


def test_growth_is_bounded(ts):
    # sixteen tokens, each 1% louder than the one before: the scale grows a few times only, and the first
    # token's codes are off by less than 2.5 steps and the last rounding
    c = ts.PagedKVCache8.allocate(1, 1, 64, 16, page_size=16)
    x = torch.randn(64, device="cuda").bfloat16().float()
    x = x / x.abs().max()
    seen = set()
    for t in range(16):
        row = (x * 1.01 ** t).bfloat16().view(1, 1, 1, 64)
        ts.paged_append(row, row, c)
        c.advance()
        seen.add(float(c.k_scales[0, 0, 0]))
    k, _ = ts.paged_dequantize(c, torch.float32)
    s = float(c.k_scales[0, 0, 0])
    assert len(seen) <= 2 and (k[0, 0, 0] - x.bfloat16().float()).abs().max() <= 3 * s


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_dequantize(ts, held, layout):
    c = make(ts, [40, 3], 3, 48, 32, 16, held, 8, layout=layout)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for got, codes, scales in zip(ts.paged_dequantize(c, dtype), (c.k_pages, c.v_pages), (c.k_scales, c.v_scales)):
            want = codes.float().reshape(codes.shape[0], 3, 2, 16, 48) * scales[..., None, None]
            assert torch.equal(got, want.view(codes.shape).to(dtype))


def reference(c, q, lens, scale=None):
    """Attention in 64 bits over slots [0, lens[b]): (out, tolerance)."""
    h, d, page, bs = c.n_kv, c.head_dim, c.page_size, c.block
    B = c.batch
    g = q.shape[1] // (h * d)
    x = q.double().view(B, h, g, d)
    out, tol = torch.zeros_like(x), torch.zeros_like(x)
    u = 2.0 ** -11 if q.dtype == torch.bfloat16 else 2.0 ** -22
    half = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        slot = torch.arange(max(0, lens[b]), device="cuda")
        p = c.page_table[b].long()[slot // page]
        ok = (p >= 0) & (p < c.k_pages.shape[0])
        slot, p = slot[ok], p[ok]
        if not len(slot):
            continue
        o = slot % page
        for j in range(h):
            k = c.k_pages[p, j, o].double() * c.k_scales[p, j, o // bs].double()[:, None]
            v = c.v_pages[p, j, o].double() * c.v_scales[p, j, o // bs].double()[:, None]
            w = torch.softmax(x[b, j] @ k.t() * (scale or d ** -0.5), -1)
            out[b, j] = w @ v
            tol[b, j] = half * out[b, j].abs() + (u + 2.0 ** -14) * (w @ v.abs()) + len(slot) * 2.0 ** -35 * v.abs().max() \
                + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    return out.view(B, -1), tol.view(B, -1)


def close(got, want, tol):
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), int((err > tol).sum()))


CASES = [  # n_q, n_kv, d, page, block, layout, lens
    (32, 8, 128, 64, 16, "heads", [512]),
    (32, 8, 128, 64, 64, "tokens", [0, 1, 15, 16, 17, 63, 64, 65, 1000, 4097]),
    (8, 8, 64, 16, 16, "heads", [300, 7]),
    (7, 1, 96, 32, 32, "tokens", [129, 2000, 31]),
    (16, 1, 128, 64, 16, "heads", [1, 700, 64, 3000]),
    (18, 2, 64, 128, 32, "heads", [513, 0, 90]),
    (33, 1, 80, 48, 48, "heads", [200, 95]),
    (4, 2, 16, 16, 16, "heads", [40, 333]),
    (6, 2, 160, 64, 16, "tokens", [100, 2500]),
    (32, 2, 256, 64, 64, "heads", [65, 900]),
    (8, 2, 128, 64, 16, "heads", [20000]),
    (4, 1, 128, 16, 16, "heads", [33] * 200),
]


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(ts, case, dtype, held):
    n_q, n_kv, d, page, block, layout, lens = CASES[case]
    c = make(ts, lens, n_kv, d, page, block, held, case, layout=layout)
    q = torch.randn(len(lens), n_q * d, device="cuda").to(dtype)
    # what lies behind the last token may be anything: bytes that are no number, scales that are none
    bits = (raw(c.k_pages), raw(c.v_pages))
    for b, n in enumerate(lens):
        p, o = int(c.page_table[b, n // page]), n % page
        for x in bits:
            x[p, :, o:] = 0x7F if held == E4M3 else 0x80
        for s in (c.k_scales, c.v_scales):
            s[p, :, -(-o // block):] = math.nan
    out = ts.paged_attention(q, c)
    close(out, *reference(c, q, lens))
    assert torch.equal(ts.paged_attention(q, c), out)
    buf = torch.full((len(lens), n_q * d + 6), 3.0, dtype=dtype, device="cuda")
    ts.paged_attention(q, c, scale=0.05, out=buf[:, 2:2 + n_q * d])
    close(buf[:, 2:2 + n_q * d], *reference(c, q, lens, 0.05))
    assert (buf[:, :2] == 3).all() and (buf[:, 2 + n_q * d:] == 3).all()


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("n_q,n_kv,d,page,lens", [
    (6, 3, 128, 64, [1, 900, 0, 129, 6000]), (12, 6, 64, 16, [700, 33]), (5, 5, 128, 64, [2000, 128]), (40, 2, 128, 64, [300, 5000, 0]),
    (34, 2, 80, 32, [1500]), (14, 7, 96, 64, [40] * 90), (24, 3, 256, 64, [70, 3000, 1]), (12, 12, 128, 64, [5000, 1, 700] * 6)])
def test_heads_taken_side_by_side(ts, n_q, n_kv, d, page, lens, held):
    # token-major pages, numbers of heads that two, three, four or no CTAs share
    c = make(ts, lens, n_kv, d, page, 16, held, 3, layout="tokens")
    q = torch.randn(len(lens), n_q * d, device="cuda").to(torch.bfloat16)
    out = ts.paged_attention(q, c)
    close(out, *reference(c, q, lens))
    assert torch.equal(ts.paged_attention(q, c), out)


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,layout", [(128, "heads"), (112, "tokens"), (96, "heads"), (64, "tokens"), (48, "heads")])
def test_many_rows(ts, d, layout, dtype, held):
    lens = [1, 900, 64, 0, 2500] * 16
    c = make(ts, lens, 4, d, 64, 32, held, 4, layout=layout)
    q = torch.randn(len(lens), 12 * d, device="cuda").to(dtype)
    out = ts.paged_attention(q, c)
    close(out, *reference(c, q, lens))
    assert torch.equal(ts.paged_attention(q, c), out)


@pytest.mark.parametrize("held", [INT8, E4M3])
def test_attention_without_pages_lengths_and_rows(ts, held):
    c = make(ts, [200, 64, 40, 100, 10], 2, 64, 16, 16, held, 4, room=1)
    c.page_table[0, 3] = -1                                       # holes
    c.page_table[0, 7] = c.k_pages.shape[0]
    c.page_table[1, :] = -1                                       # no page at all
    c.seq_lens[2] = -3
    c.seq_lens[3] = 10 ** 6                                       # longer than the table
    q = torch.randn(5, 8 * 64, device="cuda").bfloat16()
    out = ts.paged_attention(q, c)
    want, tol = reference(c, q, [200, 64, 0, 0, 10])
    close(out, want, tol)
    assert (out[1:4] == 0).all()
    cos, sin = tables(50, 64)
    pos = torch.tensor([0, 1, 2, 3, 50], device="cuda")
    out = ts.paged_attention(q, c, pos, cos, sin)
    rq = rotate(q.view(5, 8, 64), cos[pos.clamp(max=49)][:, None], sin[pos.clamp(max=49)][:, None]).view(5, -1)
    close(out[:4], *(x[:4] for x in reference(c, rq, [200, 64, 0, 0, 10])))
    assert (out[4] == 0).all()                                    # no rotary row


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_with_scales_far_apart(ts, held, dtype):
    c = make(ts, [400, 90], 2, 64, 32, 16, held, 6)
    g = torch.Generator(device="cuda").manual_seed(1)
    # values: every block another power of two, from 2^-12 to 2^8; keys quiet enough for the softmax to see all of them
    e = torch.randint(-12, 9, c.v_scales.shape, generator=g, device="cuda")
    c.v_scales.copy_(torch.exp2(e.float()) * 1.3 / TOP[held])
    c.k_scales.mul_(0.3)
    q = torch.randn(2, 4 * 64, device="cuda").to(dtype)
    close(ts.paged_attention(q, c), *reference(c, q, [400, 90]))
    # queries of any size: the scores are the same where the keys are as much smaller
    if dtype == torch.bfloat16:
        big = (q.float() * 2.0 ** 90).to(dtype)
        c2 = clone(ts, c)
        c2.k_scales.mul_(2.0 ** -90)
        assert torch.equal(ts.paged_attention(big, c2), ts.paged_attention(q, c))


def test_numbers_that_are_none_come_through(ts):
    c = make(ts, [100, 100, 100], 1, 64, 32, 16, INT8, 7)
    q = torch.randn(3, 2 * 64, device="cuda").bfloat16()
    q[0, 5] = math.nan                                            # one head of a sequence
    c.v_scales[int(c.page_table[1, 1]), 0, 0] = math.nan
    out = ts.paged_attention(q, c).view(3, 2, 64)
    assert out[0, 0].isnan().all() and out[0, 1].isfinite().all() and out[1].isnan().all() and out[2].isfinite().all()


@pytest.mark.parametrize("held", [INT8, E4M3])
@pytest.mark.parametrize("rope", [False, True])
def test_decode_is_append_then_attention(ts, held, rope):
    n_q, n_kv, d = 8, 2, 128
    lens = [0, 1, 31, 32, 500, -1, 95, 64]
    c = make(ts, lens, n_kv, d, 32, 16, held, 9)
    c.page_table[6, 2] = -1                                       # no page for slot 95
    cos, sin = tables(600, d)
    pos = torch.tensor([0, 9, 31, 600, 500, 3, 95, 64], device="cuda")       # sequence 3: no rotary row
    args = (pos, cos, sin) if rope else (None, None, None)
    for _ in range(3):
        qkv = torch.randn(len(lens), (n_q + 2 * n_kv) * d, device="cuda").bfloat16()
        want = clone(ts, c)
        k, v = qkv.view(len(lens), 1, -1, d)[:, :, n_q:].split(n_kv, dim=2)
        ts.paged_append(k, v, want, *args)
        out = ts.paged_decode_attention(qkv, n_q, c, *args)
        same(c, want)
        taken = torch.tensor([places(want, b, 1, pos if rope else None, 600 if rope else None)[0][0] is not None
                              for b in range(len(lens))], device="cuda").int()
        c.advance(taken)
        want.advance(taken)
        att = ts.paged_attention(qkv[:, :n_q * d], want, *args)
        t = taken.bool()
        assert torch.equal(out[t], att[t]) and (out[~t] == 0).all()
        q = qkv[:, :n_q * d]
        if rope:
            p = pos.clamp(max=599)
            q = rotate(q.reshape(len(lens), n_q, d), cos[p][:, None], sin[p][:, None]).view(len(lens), -1)
        ref, tol = reference(c, q, c.seq_lens.tolist())
        close(out[t], ref[t], tol[t])


def test_a_pool_past_32_bits(ts):
    # pages whose bytes lie beyond 2^32: 5 GB of keys and of values
    n_kv, d, page = 8, 128, 128
    pages = 5 * (1 << 30) // (n_kv * page * d)
    k = torch.zeros(pages, n_kv, page, d, dtype=INT8, device="cuda")
    v = torch.zeros_like(k)
    ks = torch.ones(pages, n_kv, page // 16, device="cuda")
    i = {"dtype": torch.int32, "device": "cuda"}
    c = ts.PagedKVCache8(k, v, ks, ks.clone(), torch.tensor([[pages - 1, pages - 3], [pages - 2, 5]], **i),
                         torch.tensor([0, 0], **i))
    x = torch.randn(2, 2, 200, n_kv, d, device="cuda").bfloat16()
    ts.paged_append(x[0], x[1], c)
    c.advance(200)
    q = torch.randn(2, 4 * n_kv * d, device="cuda").bfloat16()
    close(ts.paged_attention(q, c), *reference(c, q, [200, 200]))
    assert int(k[5].abs().sum()) > 0 and not k[6].any() and not k[pages - 4].any()


def test_captured_on_a_side_stream_and_next_to_others(ts):
    lens = [100, 700, 3]
    c = make(ts, lens, 2, 128, 64, 16, INT8, 11, room=8)
    start = clone(ts, c)
    qkvs = torch.randn(4, 3, 12 * 128, device="cuda").bfloat16()
    want = []
    for x in qkvs:
        want.append(ts.paged_decode_attention(x, 8, c))
        c.advance()
    final = clone(ts, c)
    for dst, src in zip(c._args(), start._args()):
        dst.copy_(src)
    buf = qkvs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ts.paged_decode_attention(buf, 8, c)
        c.advance()
    side = torch.cuda.Stream()
    other = make(ts, [5000], 8, 128, 64, 16, E4M3, 12)
    oq = torch.randn(1, 32 * 128, device="cuda").bfloat16()
    ow = ts.paged_attention(oq, other)
    torch.cuda.synchronize()
    for x, w in zip(qkvs, want):
        buf.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        outs = [ts.paged_attention(oq, other) for _ in range(5)]  # while the replay runs
        torch.cuda.synchronize()
        assert torch.equal(y, w) and all(torch.equal(o, ow) for o in outs)
    same(c, final)


def test_a_wait_that_runs_out_is_reported(ts):
    from tensorshrink_b200 import _C
    c = make(ts, [300, 20], 2, 64, 16, 16, INT8, 3)
    q = torch.randn(2, 4 * 64, device="cuda").bfloat16()
    want = ts.paged_attention(q, c)
    torch.cuda.synchronize()
    _C.load().ts_test_inject_stall(20_000_000)
    ts.paged_attention(q, c)
    with pytest.raises(RuntimeError, match="ts_paged8_status"):
        _C.serving_ops().serving_status(0)
    _C.serving_ops().serving_status(0)
    assert torch.equal(ts.paged_attention(q, c), want)


def test_refusals(ts):
    c = make(ts, [20, 3], 2, 64, 32, 16, INT8, 1)
    i = c.page_table
    new = lambda **kw: ts.PagedKVCache8(**{n: kw.get(n, getattr(c, n)) for n in c.__slots__})  # noqa: E731
    with pytest.raises(NotImplementedError):
        new(k_pages=c.k_pages.half(), v_pages=c.v_pages.half())
    with pytest.raises(ValueError):
        new(v_pages=c.v_pages.view(E4M3))
    with pytest.raises(ValueError):
        new(k_scales=c.k_scales[:, :1])
    with pytest.raises(ValueError):
        new(k_scales=c.k_scales.double())
    with pytest.raises(NotImplementedError):
        new(k_scales=c.k_scales.repeat(1, 1, 2), v_scales=c.v_scales.repeat(1, 1, 2))     # blocks of 8
    with pytest.raises(ValueError):
        new(page_table=i.long())
    with pytest.raises(RuntimeError):
        new(seq_lens=c.seq_lens.cpu())
    with pytest.raises(ValueError):
        ts.PagedKVCache8.allocate(1, 1, 64, 64, page_size=64, block=48)
    with pytest.raises(NotImplementedError):
        ts.PagedKVCache8.allocate(1, 1, 40, 64)
    q = torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ts.paged_attention(q[:1], c)
    with pytest.raises(ValueError):
        ts.paged_attention(q[:, :192], c)                        # three query heads over two
    with pytest.raises(NotImplementedError):
        ts.paged_attention(q.float(), c)
    with pytest.raises(ValueError):
        ts.paged_attention(q, c, scale=0.0)
    with pytest.raises(ValueError):
        ts.paged_attention(q, c, None, *tables(9, 64))
    with pytest.raises(ValueError):
        ts.paged_attention(q, c, out=q.half())
    with pytest.raises(NotImplementedError):
        ts.paged_attention(q, ts.PagedKVCache.allocate(2, 2, 64, 64))
    with pytest.raises(NotImplementedError):
        ts.paged_evict(c, 4)
    with pytest.raises(ValueError):
        ts.paged_decode_attention(torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device="cuda"), 4, c, accumulate=True)
    k = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ts.paged_append(k, k, c, scores=torch.zeros(2, 2, 3, device="cuda"))
    with pytest.raises(ValueError):
        ts.paged_append(k, k, c, offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ts.paged_append(k[0], k[0], c, offsets=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(NotImplementedError):
        ts.paged_append(k.float(), k.float(), c)
    with pytest.raises(NotImplementedError):
        ts.paged_append(k, k, ts.PagedKVCache.allocate(2, 2, 64, 64), offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(NotImplementedError):
        ts.paged_dequantize(ts.PagedKVCache.allocate(2, 2, 64, 64))
    y = ts.paged_attention(q.clone().requires_grad_(), c)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()
    none = ts.PagedKVCache8(c.k_pages, c.v_pages, c.k_scales, c.v_scales, i[:0], c.seq_lens[:0])
    assert ts.paged_attention(q[:0], none).shape == (0, 256)
    ts.paged_append(k[:0], k[:0], none)
    ts.paged_append(k[:, :0], k[:, :0], c)
