"""Workloads of a decoder served in 8 bits: the 8-bit integer product with a
scale for each token and channel, norms of queries and keys with their
rotation, a paged key-value cache held in 8 bits (append and attention of one
token), and the page tables and slot maps of a batch of requests.

Each case is one call, or one round of calls, as a serving program makes it.
`run` computes it from elementary torch operations, or, with `own` set,
through the public entry points of tensorshrink_b200 on the same inputs. Shapes
are those of the decoder configurations of tensorshrink_b200.decoder (hidden
4096 and 8192, intermediate 14336 and 28672, 32 or 64 query heads over 8
key-value heads of 128).

8-bit integers of a matrix: row r of x has the scale s = max(max|x_r| / 127,
2^-100) and the codes rint(x / s). 8 bits in the cache: a block of tokens of one
kv head has a scale s = max(max|x| / q, 2^-100), q = 127 (int8) or 448 (e4m3
floating point), and the codes of x / s. Tokens that come into a block that
holds earlier ones keep its scale where it is large enough; where it is not, the
new scale is a quarter more than the old one at least, and the earlier
tokens' codes are rounded anew to it.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
HELD = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
LEAST = 2.0 ** -100                            # of a scale
GROWTH = 1.25                                  # of a scale that has to grow
EPS = 1e-6
ROPE_THETA = 500000.0
LARGEST_LINEAR = 2 * 8191 * 28672 * 8192       # flops of the largest listed product
LARGEST_CACHE = 1 << 29                        # bytes of codes of the largest listed cache
LARGEST_QKV = 8191 * 80 * 128                  # elements of the largest listed projection output
LARGEST_NEW = 2 * 16 * 4096 * 8 * 128          # elements of k and v of the largest listed append


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _linear(name, m, n, k, dtype, bias=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _norm(name, tokens, n_q, n_kv, dim, dtype, norm, rope, store):
    return {"name": name, "op": "norm", "tokens": tokens, "n_q": n_q, "n_kv": n_kv, "dim": dim, "dtype": dtype,
            "norm": norm, "rope": rope, "store": store}


def _append(name, batch, n_kv, dim, page, block, held, cached, new, packed, dtype):
    return {"name": name, "op": "append", "batch": batch, "n_kv": n_kv, "dim": dim, "page": page, "block": block,
            "held": held, "cached": cached, "new": new, "packed": packed, "dtype": dtype}


def _attend(name, batch, n_q, n_kv, dim, page, block, held, longest, ragged, dtype, layout="heads"):
    return {"name": name, "op": "attend", "batch": batch, "n_q": n_q, "n_kv": n_kv, "dim": dim, "page": page,
            "block": block, "held": held, "longest": longest, "ragged": ragged, "dtype": dtype, "layout": layout}


def _tables(name, batch, page, longest, prompt, prompts):
    return {"name": name, "op": "tables", "batch": batch, "page": page, "longest": longest, "prompt": prompt,
            "prompts": prompts}


def listed():
    return [
        # decode, one sequence: a gate projection
        _linear("linear 1x14336x4096", 1, 14336, 4096, "bf16"),
        # decode of a batch of 33 sequences: a down projection, with bias
        _linear("linear 33x4096x14336 bias", 33, 4096, 14336, "fp16", True),
        # 8191 tokens of prompts through the largest projection of the configurations
        _linear("linear 8191x28672x8192", 8191, 28672, 8192, "bf16"),
        # one token's queries and keys on their way to the attention
        _norm("norm 1x48 heads", 1, 32, 8, 128, "bf16", True, True, False),
        # 8191 tokens of ragged prompts, keys and values put into their pages in the same pass
        _norm("norm 8191x80 heads stored", 8191, 64, 8, 128, "bf16", True, True, True),
        # one new token of each of 64 sequences into blocks that hold earlier ones
        _append("append 64x1 int8", 64, 8, 128, 16, 16, "int8", 9, 1, False, "bf16"),
        # the prompts of sixteen sequences, packed
        _append("append 16x4096 e4m3", 16, 8, 128, 64, 16, "e4m3", 0, 4096, True, "bf16"),
        # one sequence, early in its answer: latency counts
        _attend("attend 1x512 int8", 1, 32, 8, 128, 16, 16, "int8", 512, False, "bf16"),
        # a served batch of 64 sequences of all lengths up to 8191 cached tokens, 8 query heads to a key-value head
        _attend("attend 64x8191 int8 ragged", 64, 64, 8, 128, 64, 16, "int8", 8191, True, "bf16", "tokens"),
        # four long contexts
        _attend("attend 4x32768 e4m3", 4, 32, 8, 128, 64, 64, "e4m3", 32768, False, "fp16"),
        # a small batch takes one token each
        _tables("tables 8 decode", 8, 16, 700, 1, 0),
        # a large one, eight of whose sequences are prompts that come in
        _tables("tables 256 with prompts", 256, 64, 16384, 8000, 8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("linear", "norm", "append", "attend", "tables"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    held = rng.choice(("int8", "e4m3"))
    n_kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 96, 128))
    page = rng.choice((16, 32, 64, 128))
    block = rng.choice([b for b in (16, 32, 64) if b <= page])
    batch = _log_int(rng, 1, 64)
    if op == "linear":
        n, k = _log_int(rng, 256, 28672), _log_int(rng, 256, 28672)
        if rng.random() < 0.5:
            n, k = n // 64 * 64, k // 64 * 64
        m = _log_int(rng, 1, 8191)
        while 2 * m * n * k > LARGEST_LINEAR:
            m = max(1, m // 2)
        c = _linear("", m, n, k, rng.choice((dtype, dtype, "fp32")), rng.random() < 0.5)
    elif op == "norm":
        n_q = n_kv * rng.choice((1, 2, 4, 7, 8))
        tokens = _log_int(rng, 1, min(16384, LARGEST_QKV // ((n_q + 2 * n_kv) * dim)))
        c = _norm("", tokens, n_q, n_kv, dim, dtype, rng.random() < 0.8, rng.random() < 0.8, rng.random() < 0.5)
    elif op == "append":
        new = _log_int(rng, 1, 4096)
        while 2 * batch * n_kv * dim * new > LARGEST_NEW:
            new = max(1, new // 2)
        c = _append("", batch, n_kv, dim, page, block, held, rng.choice((0, rng.randint(1, 40))), new,
                    rng.random() < 0.5, dtype)
    elif op == "attend":
        longest = _log_int(rng, 1, 32768)
        while 2 * batch * n_kv * dim * longest > LARGEST_CACHE // 2:
            longest = max(1, longest // 2)
        c = _attend("", batch, n_kv * rng.choice((1, 2, 4, 7, 8, 16)), n_kv, dim, page, block, held, longest,
                    rng.random() < 0.7, dtype, rng.choice(("heads", "tokens")))
    else:
        batch = _log_int(rng, 1, 256)
        longest = _log_int(rng, 1, 16384)
        prompts = rng.randint(0, min(8, batch))
        c = _tables("", batch, page, longest, _log_int(rng, 1, 8000) if prompts else 1, prompts)
    del c["name"]
    return c


def _lengths(case, longest=None):
    """Cached tokens of each sequence, a function of the case alone: spread
    over [0, longest] by the golden ratio, the first at `longest`, and an
    empty one among six or more."""
    n, b = case["longest"] if longest is None else longest, case["batch"]
    if not case.get("ragged", True):
        return [n] * b
    out = [n] + [int(n * math.fmod(0.6180339887498949 * i, 1.0)) for i in range(1, b)]
    if b >= 6:
        out[b // 2] = 0
    return out


def _new_counts(case):
    """New tokens of each sequence: all alike, or, packed, of unlike counts."""
    return _lengths(case, case["new"]) if case["packed"] else [case["new"]] * case["batch"]


def _requests(case):
    """(cached, new) tokens of each sequence: prompts that come in hold
    nothing yet, the others take one token."""
    lens = _lengths(case)
    new = [1] * case["batch"]
    for i in range(case["prompts"]):
        lens[i], new[i] = 0, max(1, case["prompt"] * (i + 1) // case["prompts"])
    return lens, new


def work(case):
    op = case["op"]
    e = BYTES.get(case.get("dtype"), 0)
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * e + n * k + 4 * n + m * n * e + case["bias"] * n * e, "flops": 2 * m * n * k}
    if op == "norm":
        heads = case["n_q"] + 2 * case["n_kv"]
        n = case["tokens"] * heads * case["dim"]
        store = 2 * case["tokens"] * case["n_kv"] * case["dim"] * e + 8 * case["tokens"] if case["store"] else 0
        return {"bytes": 2 * n * e + store + case["rope"] * case["tokens"] * (case["dim"] * 4 + 8), "flops": 8 * n}
    if op == "append":
        row = case["n_kv"] * case["dim"]
        n = 2 * sum(_new_counts(case)) * row
        pool = 2 * _pool_pages(case) * case["page"] * row
        scales = 4 * pool // (case["dim"] * case["block"])
        # the tokens read, their codes written; then the pool's codes and scales read and their values written
        return {"bytes": n * (e + 1) + pool * (1 + e) + 2 * scales, "flops": 4 * n + pool}
    if op == "attend":
        tokens, d = sum(_lengths(case)), case["dim"]
        kv = 2 * tokens * case["n_kv"] * d
        return {"bytes": kv + 4 * kv // (d * case["block"]) + 2 * case["batch"] * case["n_q"] * d * e
                + 4 * sum(-(-t // case["page"]) for t in _lengths(case)), "flops": 4 * tokens * case["n_q"] * d}
    lens, new = _requests(case)
    pages = sum(-(-(a + b) // case["page"]) - a // case["page"] for a, b in zip(lens, new))
    # a slot, a position and a sequence for each token; the pages from the pool to the table and back
    return {"bytes": 20 * sum(new) + 16 * pages + 32 * case["batch"], "flops": 8 * sum(new)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 11)


def _rope_tables(length, dim):
    inv = 1.0 / (ROPE_THETA ** (torch.arange(0, dim, 2, device=DEV, dtype=torch.float32) / dim))
    ang = torch.outer(torch.arange(length, device=DEV, dtype=torch.float32), inv)
    return ang.cos(), ang.sin()


def _capacity(case):
    """Slots that each sequence of an append or attend case has pages for."""
    if case["op"] == "append":
        return [case["cached"] + n for n in _new_counts(case)]
    return [n + 1 for n in _lengths(case)]


def _pool_pages(case):
    return sum(-(-c // case["page"]) for c in _capacity(case)) + 3


def _page_table(case, g):
    """Each sequence's pages, in random order of the pool, ended by -1."""
    need = [-(-c // case["page"]) for c in _capacity(case)]
    order = torch.randperm(sum(need) + 3, generator=g, device=DEV).to(torch.int32)
    table = torch.full((case["batch"], max(1, max(need))), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def _held_pages(case, g):
    """Pages of random keys and values as codes with their scales."""
    h, d, ps, bs = case["n_kv"], case["dim"], case["page"], case["block"]
    pages = _pool_pages(case)
    out = []
    for _ in range(2):
        codes = torch.empty(pages, h, ps, d, dtype=HELD[case["held"]], device=DEV)
        scales = torch.empty(pages, h, ps // bs, device=DEV)
        loud = torch.exp(0.5 * torch.randn(h, 1, d, generator=g, device=DEV))      # channels of unlike size
        step = max(1, (1 << 26) // (h * ps * d))
        for i in range(0, pages, step):
            x = torch.randn(min(step, pages - i), h, ps, d, generator=g, device=DEV) * loud
            x = x.view(-1, h, ps // bs, bs, d)
            s = (x.abs().amax(dim=(3, 4)) * (1.0 / TOP[case["held"]])).clamp(min=LEAST)
            codes[i:i + step] = _codes(x * (1.0 / s)[..., None, None], case["held"]).reshape(-1, h, ps, d)
            scales[i:i + step] = s
        if case.get("layout") == "tokens":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)      # [pages, heads, slots, dim] over token-major memory
        out += [codes, scales]
    return out


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    dt = DTYPES.get(case.get("dtype"))
    if op == "linear":
        w = torch.randn(case["n"], case["k"], generator=g, device=DEV) * 0.02
        codes, scales = _plain_rows(w)
        del w
        stored = torch.zeros(case["n"], -(-case["k"] // 16) * 16, dtype=torch.int8, device=DEV)
        stored[:, :case["k"]] = codes
        del codes
        x = torch.randn(case["m"], case["k"], generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn(1, case["k"], generator=g, device=DEV))      # channels of unlike size
        bias = torch.randn(case["n"], generator=g, device=DEV).to(dt) if case["bias"] else None
        return {"case": case, "x": x.to(dt), "codes": stored, "scales": scales, "bias": bias}
    if op == "tables":
        lens, new = _requests(case)
        ps = case["page"]
        need = [-(-n // ps) for n in lens]
        want = [-(-(a + b) // ps) for a, b in zip(lens, new)]
        total = sum(want) + 5
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((case["batch"], max(want)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        free = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        free[:total - at] = order[at:]
        i32 = {"dtype": torch.int32, "device": DEV}
        h, d = 1, 16                                       # the tables do not look at the pages' content
        pages = torch.zeros(total, h, ps, d, dtype=torch.bfloat16, device=DEV)
        return {"case": case, "table": table, "lens": torch.tensor(lens, **i32), "keep": torch.tensor(lens, **i32),
                "n_new": torch.tensor(new, **i32), "free": free, "n_free": torch.tensor([total - at], **i32),
                "tokens": -(-sum(new) // 64) * 64, "k": pages, "v": pages.clone()}
    h, d = case["n_kv"], case["dim"]
    if op == "norm":
        t, n_q = case["tokens"], case["n_q"]
        x = torch.randn(t, n_q + 2 * h, d, generator=g, device=DEV)
        x *= torch.exp(torch.randn(1, n_q + 2 * h, 1, generator=g, device=DEV))       # heads of unlike size
        s = {"case": case, "qkv": x.to(dt).reshape(t, -1), "qw": None, "kw": None, "positions": None, "cos": None,
             "sin": None, "k": None, "v": None, "slots": None, "table": None, "lens": None}
        if case["norm"]:
            s["qw"], s["kw"] = (1 + 0.2 * torch.randn(2, d, generator=g, device=DEV)).unbind(0)
        if case["rope"]:
            s["positions"] = torch.randint(0, 32768, (t,), generator=g, device=DEV)
            s["cos"], s["sin"] = _rope_tables(32768, d)
        if case["store"]:
            pages = -(-t // 64) + 2
            s["k"], s["v"] = torch.randn(2, pages, h, 64, d, generator=g, device=DEV).to(dt).unbind(0)
            s["slots"] = torch.randperm(pages * 64, generator=g, device=DEV)[:t]
            s["slots"][t // 2] = -1                                                    # a token that found no page
            s["table"] = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
            s["lens"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        return s
    if op == "append":
        new = _new_counts(case)
        kc, ks, vc, vs = _held_pages(case, g)
        shape = (sum(new), h, d) if case["packed"] else (case["batch"], case["new"], h, d)
        k, v = (torch.randn(2, *shape, generator=g, device=DEV) * 1.2).to(dt).unbind(0)
        offsets = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)
        lens = torch.full((case["batch"],), case["cached"], dtype=torch.int32, device=DEV)
        return {"case": case, "k_new": k, "v_new": v, "offsets": offsets if case["packed"] else None, "k": kc, "ks": ks,
                "v": vc, "vs": vs, "table": _page_table(case, g), "lens": lens}
    kc, ks, vc, vs = _held_pages(case, g)
    q = torch.randn(case["batch"], case["n_q"] * d, generator=g, device=DEV).to(dt)
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    return {"case": case, "q": q, "k": kc, "ks": ks, "v": vc, "vs": vs, "table": _page_table(case, g), "lens": lens,
            "longest": max(_lengths(case))}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _codes(y, held):
    """Codes of values that were divided by their scale."""
    if held == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_rows(x):
    """8-bit integers of x's rows, and the rows' scales."""
    x = x.float()
    s = (x.abs().amax(dim=1) * (1.0 / 127.0)).clamp(min=LEAST)
    return _codes(x * (1.0 / s)[:, None], "int8"), s


def _plain_linear(s):
    k = s["case"]["k"]
    codes, xs = _plain_rows(s["x"])
    y = codes.float() @ s["codes"][:, :k].float().t()
    ws = s["scales"][None, :]
    y = (y * torch.minimum(xs[:, None], ws)) * torch.maximum(xs[:, None], ws)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_norm(s):
    c = s["case"]
    t, n_q, h, d = c["tokens"], c["n_q"], c["n_kv"], c["dim"]
    x = s["qkv"].float().view(t, n_q + 2 * h, d)
    qk, v = x[:, :n_q + h], x[:, n_q + h:]
    if c["norm"]:
        w = torch.cat([s["qw"].expand(n_q, d), s["kw"].expand(h, d)])
        qk = qk * torch.rsqrt((qk * qk).mean(dim=-1, keepdim=True) + EPS) * w
    if c["rope"]:
        cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
        a, b = qk.chunk(2, dim=-1)
        qk = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    y = torch.cat([qk, v], dim=1).to(s["qkv"].dtype)
    res = {"out": y.view(t, -1)}
    if c["store"]:
        at = s["slots"]
        kept = at >= 0
        page, off = at[kept] // 64, at[kept] % 64
        s["k"][page, :, off] = y[kept, n_q:n_q + h]
        s["v"][page, :, off] = y[kept, n_q + h:]
        res |= {"k": s["k"], "v": s["v"]}
    return res


def _plain_store(codes, scales, new, s):
    """Puts new[b, i] (fp32, NaN where slot i of the touched blocks gets no
    token) into the cache."""
    c = s["case"]
    bs, ps, held, h = c["block"], c["page"], c["held"], c["n_kv"]
    b, n = new.shape[:2]
    first = s["lens"].long() // bs                                              # the first block that is touched
    slot = (first * bs)[:, None] + torch.arange(n, device=DEV)
    page = s["table"].long().gather(1, (slot // ps).clamp(max=s["table"].shape[1] - 1))
    hi = torch.arange(h, device=DEV)
    x = new.view(b, n // bs, bs, h, -1)
    comes = ~x[:, :, :, 0, 0].isnan()                                          # [b, blocks, block]
    touched = comes.any(dim=2)
    x = torch.where(x.isnan(), torch.zeros_like(x), x)
    need = (x.abs().amax(dim=(2, 4)) * (1.0 / TOP[held])).clamp(min=LEAST)      # [b, blocks, heads]
    bp, bo = page[:, ::bs].clamp(min=0), (slot[:, ::bs] % ps) // bs             # page and block in it
    old = scales[bp[..., None], hi, bo[..., None]]
    earlier = (slot[:, ::bs] < s["lens"][:, None])[..., None]
    grown = torch.where(need > old, torch.maximum(need, GROWTH * old), old)
    scale = torch.where(earlier, grown, need)
    was = codes[page.clamp(min=0)[..., None], hi, (slot % ps)[..., None]].view(b, n // bs, bs, h, -1)
    ratio = torch.where(earlier, old / scale, torch.ones_like(scale))
    moved = _codes(was.float() * ratio[:, :, None, :, None], held)
    fresh = _codes(x * (1.0 / scale)[:, :, None, :, None], held)
    res = torch.where(comes[..., None, None], fresh.float(), moved.float()).to(codes.dtype)
    live = (touched[:, :, None] & (comes | (slot < s["lens"][:, None]).view(b, n // bs, bs))).nonzero(as_tuple=True)
    p, o = page.view(b, -1, bs)[live], (slot % ps).view(b, -1, bs)[live]
    codes[p[:, None], hi, o[:, None]] = res[live]
    bi = touched.nonzero(as_tuple=True)
    scales[bp[bi][:, None], hi, bo[bi][:, None]] = scale[bi]


def _plain_append(s):
    c = s["case"]
    b, bs, h, d = c["batch"], c["block"], c["n_kv"], c["dim"]
    counts = _new_counts(c)
    lead = s["lens"].long() % bs
    n = -(-(c["cached"] % bs + max(counts)) // bs) * bs
    for codes, scales, src in ((s["k"], s["ks"], s["k_new"]), (s["v"], s["vs"], s["v_new"])):
        new = torch.full((b, n, h, d), math.nan, device=DEV)
        if c["packed"]:
            at = torch.arange(sum(counts), device=DEV)
            i = torch.searchsorted(s["offsets"][1:].long(), at, right=True)
            new[i, lead[i] + at - s["offsets"].long()[i]] = src.float()
        else:
            new[:, c["cached"] % bs:c["cached"] % bs + c["new"]] = src.float()
        _plain_store(codes, scales, new, s)
    return {"k": _plain_values(s["k"], s["ks"], c), "v": _plain_values(s["v"], s["vs"], c), "k_scales": s["ks"],
            "v_scales": s["vs"]}


def _plain_values(codes, scales, c):
    x = codes.float().reshape(codes.shape[0], c["n_kv"], -1, c["block"], c["dim"])
    return (x * scales[..., None, None]).view(codes.shape).to(DTYPES[c["dtype"]])


def _plain_attend(s):
    c = s["case"]
    b, h, d, ps, nq, bs = c["batch"], c["n_kv"], c["dim"], c["page"], c["n_q"], c["block"]
    n = max(1, s["longest"])
    slot = torch.arange(n, device=DEV)
    live = slot[None, :] < s["lens"][:, None]
    page = s["table"][:, slot // ps].long().clamp(min=0)[:, None, :]
    hi, off = torch.arange(h, device=DEV)[None, :, None], (slot % ps)[None, None, :]
    kk = s["k"][page, hi, off].float() * s["ks"][page, hi, off // bs][..., None]        # [b, h, n, d]
    vv = s["v"][page, hi, off].float() * s["vs"][page, hi, off // bs][..., None]
    sc = (s["q"].float().view(b, h, nq // h, d) @ kk.transpose(2, 3)) * (d ** -0.5)
    sc = sc.masked_fill(~live[:, None, None, :], -math.inf)
    top = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))                        # (an empty sequence: zeros)
    return (p @ (vv * live[:, None, :, None])).reshape(b, nq * d).to(s["q"].dtype)


def _plain_tables(s):
    c = s["case"]
    ps, table, lens, new = c["page"], s["table"], s["lens"].long(), s["n_new"].long()
    # pages for the new tokens
    p = torch.arange(table.shape[1], device=DEV)
    empty = (p >= (lens // ps)[:, None]) & (p < (-(-(lens + new) // ps))[:, None]) & (table < 0)
    need = empty.sum(dim=1)
    upto = need.cumsum(0)
    served = (need == 0) | (upto <= s["n_free"])
    rank = (upto - need)[:, None] + empty.cumsum(1) - 1
    popped = s["free"][(s["n_free"] - 1 - rank).clamp(min=0)]
    table.copy_(torch.where(empty & served[:, None], popped, table))
    s["n_free"].sub_((need * served).sum().to(torch.int32))
    granted = torch.where(served, new, torch.zeros_like(new))
    # the slots of the packed tokens
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), new.cumsum(0)])
    t = torch.arange(s["tokens"], device=DEV)
    within = t < offsets[-1]
    i = torch.searchsorted(offsets[1:], t, right=True).clamp(max=c["batch"] - 1)
    slot = lens[i] + t - offsets[i]
    has = within & served[i]
    page = table[i, (slot // ps).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(has, page * ps + slot % ps, torch.full_like(t, -1))
    positions = torch.where(has, slot, torch.zeros_like(t))
    sequences = torch.where(within, i, torch.full_like(t, -1)).to(torch.int32)
    res = {"granted": granted.to(torch.int32), "offsets": offsets.to(torch.int32), "slots": slots, "positions": positions,
           "sequences": sequences, "table": table.clone()}
    # the tokens are in; then the sequences are cut back, and their pages return
    s["lens"].add_(granted.to(torch.int32))
    s["lens"].copy_(torch.minimum(s["lens"], s["keep"]))
    back = (p >= (-(-s["lens"].long() // ps))[:, None]) & (table >= 0)
    n = back.sum()
    at = s["n_free"].long() + back.flatten().cumsum(0).view(back.shape) - 1
    s["free"][at[back]] = table[back]
    table.masked_fill_(back, -1)
    s["n_free"].add_(n.to(torch.int32))
    return res | {"lens": s["lens"], "free": s["free"], "n_free": s["n_free"], "table after": table}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    c, s = state["case"], state
    op = c["op"]
    if not own:
        return {"linear": _plain_linear, "norm": _plain_norm, "append": _plain_append, "attend": _plain_attend,
                "tables": _plain_tables}[op](s)
    import tensorshrink_b200 as ts
    if op == "linear":
        return ts.int8_linear(s["x"], ts.Int8Tensor(s["codes"], s["scales"], c["k"]), bias=s["bias"])
    if op == "norm":
        cache = ts.PagedKVCache(s["k"], s["v"], s["table"], s["lens"]) if c["store"] else None
        out = ts.qk_norm_rope(s["qkv"], c["n_q"], c["n_kv"], s["qw"], s["kw"], s["positions"], s["cos"], s["sin"],
                              eps=EPS, cache=cache, slots=s["slots"])
        return {"out": out, "k": s["k"], "v": s["v"]} if c["store"] else {"out": out}
    if op == "append":
        cache = ts.PagedKVCache8(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"])
        ts.paged_append(s["k_new"], s["v_new"], cache, offsets=s["offsets"])
        k, v = ts.paged_dequantize(cache, DTYPES[c["dtype"]])
        return {"k": k, "v": v, "k_scales": s["ks"], "v_scales": s["vs"]}
    if op == "attend":
        cache = ts.PagedKVCache8(s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"])
        return ts.paged_attention(s["q"], cache)
    pool, cache = ts.PagePool(s["free"], s["n_free"]), ts.PagedKVCache(s["k"], s["v"], s["table"], s["lens"])
    got = ts.paged_reserve(pool, cache, s["n_new"], s["tokens"])
    res = got._asdict() | {"table": s["table"].clone()}
    cache.advance(got.granted)
    ts.paged_release(pool, cache, s["keep"])
    return res | {"lens": s["lens"], "free": s["free"], "n_free": s["n_free"], "table after": s["table"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _grid(y, held):
    """y (64 bits) as the nearest value that 8 bits hold, ties to even."""
    if held == "int8":
        return torch.round(y).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -1000))).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _exact_linear(s):
    k = s["case"]["k"]
    x = s["x"].double()
    xs = (x.abs().amax(dim=1, keepdim=True) / 127).clamp(min=LEAST)
    y = _grid(x / xs, "int8") @ s["codes"][:, :k].double().t()
    y = y * xs * s["scales"].double()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_norm(s):
    c = s["case"]
    n_q, h, d = c["n_q"], c["n_kv"], c["dim"]
    y = s["qkv"].double().view(c["tokens"], n_q + 2 * h, d)
    heads = list(range(n_q + h))
    if c["norm"]:
        root = torch.sqrt(y[:, heads].square().sum(-1, keepdim=True) / d + EPS)
        y[:, :n_q] = y[:, :n_q] / root[:, :n_q] * s["qw"].double()
        y[:, n_q:n_q + h] = y[:, n_q:n_q + h] / root[:, n_q:] * s["kw"].double()
    if c["rope"]:
        z = torch.complex(y[:, :n_q + h, :d // 2].contiguous(), y[:, :n_q + h, d // 2:].contiguous())
        turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]]
        z = z * turn[:, None]
        y[:, :n_q + h] = torch.cat([z.real, z.imag], -1)
    res = {"out": y.view(c["tokens"], -1)}
    if c["store"]:
        k, v = s["k"].double(), s["v"].double()
        for first, pages in ((n_q, k), (n_q + h, v)):
            flat = pages.permute(0, 2, 1, 3).contiguous().clone().view(-1, h, d)
            ok = s["slots"] >= 0
            flat[s["slots"][ok]] = y[ok, first:first + h]
            pages.copy_(flat.view(pages.shape[0], -1, h, d).permute(0, 2, 1, 3))
        res |= {"k": k, "v": v}
    return res


def _exact_append(s):
    c = s["case"]
    bs, ps, held, cached = c["block"], c["page"], c["held"], c["cached"]
    counts = _new_counts(c)
    if sum(-(-n // bs) + 1 for n in counts) > 8192:
        return None
    table = s["table"].cpu()
    start = np.concatenate([[0], np.cumsum(counts)])
    res = {}
    for name, codes, scales, src in (("k", s["k"], s["ks"], s["k_new"]), ("v", s["v"], s["vs"], s["v_new"])):
        val = codes.double().reshape(codes.shape[0], c["n_kv"], -1, bs, c["dim"])
        sc = scales.double()
        val = val * sc[..., None, None]
        for i, n in enumerate(counts):
            x = (src[start[i]:start[i + 1]] if c["packed"] else src[i]).double()
            at = 0
            while at < n:
                slot = cached + at
                page, blk, o = int(table[i, slot // ps]), slot % ps // bs, slot % bs
                m = min(n - at, bs - o)
                y = x[at:at + m].transpose(0, 1)                                   # [heads, tokens, dim]
                scale = (y.abs().amax(dim=(1, 2)) / TOP[held]).clamp(min=LEAST)
                if o:
                    old = sc[page, :, blk]
                    scale = torch.where(scale > old, torch.maximum(scale, GROWTH * old), old)
                    val[page, :, blk, :o] = _grid(val[page, :, blk, :o] / scale[:, None, None], held) * scale[:, None, None]
                sc[page, :, blk] = scale
                # (what lies behind the tokens counts in the new scale)
                rest = codes.view(val.shape)[page, :, blk, o + m:].double()
                val[page, :, blk, o + m:] = rest * scale[:, None, None]
                val[page, :, blk, o:o + m] = _grid(y / scale[:, None, None], held) * scale[:, None, None]
                at += m
        res[name] = val.reshape(codes.shape)
        res[name + "_scales"] = sc
    return {n: res[n] for n in ("k", "v", "k_scales", "v_scales")}


def _exact_attend(s):
    c = s["case"]
    b, h, d, ps, g = c["batch"], c["n_kv"], c["dim"], c["page"], c["n_q"] // c["n_kv"]
    out = torch.zeros(b, h, g, d, dtype=torch.float64, device=DEV)
    q = s["q"].view(b, h, g, d).double()
    for i, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        slot = torch.arange(n, device=DEV)
        page, off = s["table"][i, slot // ps].long(), slot % ps
        for j in range(h):
            kk = s["k"][page, j, off].double() * s["ks"][page, j, off // c["block"]].double()[:, None]
            vv = s["v"][page, j, off].double() * s["vs"][page, j, off // c["block"]].double()[:, None]
            out[i, j] = torch.softmax(q[i, j] @ kk.t() / math.sqrt(d), dim=-1) @ vv
    return out.reshape(b, -1)


def exact(case, seed):
    if case["op"] == "tables":
        return None                                        # whole numbers
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "append": _exact_append, "attend": _exact_attend}[case["op"]](s)
