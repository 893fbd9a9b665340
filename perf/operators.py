"""The serving operators' workloads: microscaled 4-bit quantisation and
product, attention of one new token over a paged key-value cache, and
eviction from that cache by accumulated attention weight.

Each case is one call as a serving program makes it. `run` computes it from
elementary torch operations in 32 bits, or, with `own` set, through the
public entry points of tensorshrink_b200 on the same inputs. Weight shapes are those of the
decoder configurations of tensorshrink_b200.decoder (hidden 4096 and 8192,
intermediate 14336 and 28672, 32 or 64 query heads over 8 key-value heads of
128).

Formats (both hold E2M1 elements, two to a byte, the even column in the low
nibble; columns padded with zeros to a multiple of 64):
  nvfp4  blocks of 16 columns with an E4M3 scale, and one fp32 scale g of
         the whole tensor; value = e2m1 * (scale * g)
  mxfp4  blocks of 32 columns with a power of two (E8M0) as scale
Scales lie in tiles of 128 rows x 4 blocks, 512 bytes each, tile by tile
along a row of tiles: the byte of (row r, block j) within its tile is
(r % 32) * 16 + (r % 128) // 32 * 4 + j % 4.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = {"nvfp4": 16, "mxfp4": 32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
ROPE_THETA = 500000.0
LARGEST_LINEAR = 2 * 8192 * 28672 * 8192      # flops of the largest listed product
LARGEST_CACHE = 1 << 30                       # bytes of keys and values of the largest listed cache
LARGEST_ROWS = 14336 * 4096                   # elements of the largest listed quantisation


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _quant(name, rows, cols, fmt, dtype, given):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "format": fmt, "dtype": dtype, "given": given}


def _linear(name, m, n, k, fmt, dtype, bias=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "format": fmt, "dtype": dtype, "bias": bias}


def _attend(name, batch, n_q, n_kv, dim, page, longest, ragged, dtype, weights, layout="heads"):
    return {"name": name, "op": "attend", "batch": batch, "n_q": n_q, "n_kv": n_kv, "dim": dim, "page": page,
            "longest": longest, "ragged": ragged, "dtype": dtype, "weights": weights, "layout": layout}


def _evict(name, batch, n_kv, dim, page, budget, chunk, recent, dtype):
    return {"name": name, "op": "evict", "batch": batch, "n_kv": n_kv, "dim": dim, "page": page, "budget": budget,
            "chunk": chunk, "recent": recent, "dtype": dtype}


def listed():
    return [
        # one token's activations in front of a 4-bit projection, with the scale a calibration gave
        _quant("quantize 1x4096 nvfp4", 1, 4096, "nvfp4", "bf16", True),
        # a gate projection's weights as they are shrunk at load time: the tensor's scale is found too
        _quant("quantize 14336x4096 nvfp4", 14336, 4096, "nvfp4", "fp16", False),
        # activations of a ragged prompt, with columns that fill neither a block nor a 16-byte load
        _quant("quantize 2047x14330 mxfp4", 2047, 14330, "mxfp4", "bf16", False),
        # decode, one sequence: a gate projection
        _linear("linear 1x14336x4096 nvfp4", 1, 14336, 4096, "nvfp4", "bf16"),
        # decode of a batch of 33 sequences: a down projection, with bias
        _linear("linear 33x4096x14336 mxfp4", 33, 4096, 14336, "mxfp4", "fp16", True),
        # a prompt of 2047 tokens through a gate projection
        _linear("linear 2047x14336x4096 nvfp4", 2047, 14336, 4096, "nvfp4", "bf16"),
        # 8192 tokens of prompts through the largest projection of the configurations
        _linear("linear 8192x28672x8192 nvfp4", 8192, 28672, 8192, "nvfp4", "bf16"),
        # one sequence, early in its answer: latency counts
        _attend("attend 1x512", 1, 32, 8, 128, 16, 512, False, "bf16", False),
        # a served batch of 64 sequences of all lengths up to 8191 cached tokens, 8 query heads to a key-value head
        _attend("attend 64x8191 ragged", 64, 64, 8, 128, 64, 8191, True, "bf16", False, "tokens"),
        # four long contexts, with the attention weights kept for the eviction
        _attend("attend 4x32768 weights", 4, 32, 8, 128, 64, 32768, False, "bf16", True),
        # one sequence held at 1024 tokens: one new token in, one out
        _evict("evict 1x1024+1", 1, 8, 128, 16, 1024, 1, 128, "bf16"),
        # sixteen sequences take a prompt chunk of 4096 tokens and are cut back to 4096
        _evict("evict 16x4096+4096", 16, 8, 128, 64, 4096, 4096, 256, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "attend", "evict"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    fmt = rng.choice(("nvfp4", "mxfp4"))
    if op == "quantize":
        cols = _log_int(rng, 32, 16384)
        rows = _log_int(rng, 1, max(1, min(16384, LARGEST_ROWS // cols)))
        c = _quant("", rows, cols, fmt, rng.choice(("bf16", "fp16", "fp32")), rng.random() < 0.5)
    elif op == "linear":
        n, k = _log_int(rng, 256, 28672), _log_int(rng, 256, 28672)
        if rng.random() < 0.5:
            n, k = n // 64 * 64, k // 64 * 64
        m = _log_int(rng, 1, 8192)
        while 2 * m * n * k > LARGEST_LINEAR:
            m = max(1, m // 2)
        c = _linear("", m, n, k, fmt, dtype, rng.random() < 0.5)
    else:
        n_kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 96, 128))
        page = rng.choice((8, 16, 32, 64, 128))
        batch = _log_int(rng, 1, 64)
        if op == "attend":
            longest = _log_int(rng, 1, 32768)
            while 4 * batch * n_kv * dim * longest > LARGEST_CACHE // 2:
                longest = max(1, longest // 2)
            c = _attend("", batch, n_kv * rng.choice((1, 2, 4, 7, 8, 16)), n_kv, dim, page, longest, rng.random() < 0.7,
                        dtype, rng.random() < 0.4, rng.choice(("heads", "tokens")))
        else:
            budget, chunk = _log_int(rng, 64, 8192), _log_int(rng, 1, 8192)
            while 4 * batch * n_kv * dim * (budget + chunk) > LARGEST_CACHE // 2:
                budget, chunk = max(32, budget // 2), max(1, chunk // 2)
                batch = max(1, batch // 2)
            c = _evict("", batch, n_kv, dim, page, budget, chunk, rng.randint(0, budget), dtype)
    del c["name"]
    return c


def _lengths(case):
    """Cached tokens of each sequence, a function of the case alone: spread
    over [0, longest] by the golden ratio, the first at `longest`, and an
    empty one among six or more."""
    n, b = case["longest"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    out = [n] + [int(n * math.fmod(0.6180339887498949 * i, 1.0)) for i in range(1, b)]
    if b >= 6:
        out[b // 2] = 0
    return out


def _pad64(k):
    return -(-k // 64) * 64


def work(case):
    op = case["op"]
    if op == "quantize":
        n, kp = case["rows"] * case["cols"], case["rows"] * _pad64(case["cols"])
        e = BYTES[case["dtype"]]
        # the elements read once, codes and scales written and read by the caller, the values written
        return {"bytes": n * e + kp / 2 + kp / BLOCK[case["format"]] + n * e, "flops": 4 * n}
    if op == "linear":
        m, n, kp = case["m"], case["n"], _pad64(case["k"])
        e = BYTES[case["dtype"]]
        return {"bytes": m * case["k"] * e + n * kp / 2 + n * kp / BLOCK[case["format"]] + m * n * e + case["bias"] * n * e,
                "flops": 2 * m * n * case["k"]}
    e, d = BYTES[case["dtype"]], case["dim"]
    if op == "attend":
        tokens = sum(_lengths(case))
        b, g = case["batch"], case["n_q"]
        kv = 2 * tokens * case["n_kv"] * d * e
        new = b * (g + 2 * case["n_kv"]) * d * e + 2 * b * case["n_kv"] * d * e + b * g * d * e
        acc = 8 * tokens * case["n_kv"] if case["weights"] else 0
        return {"bytes": kv + new + acc + 4 * sum(-(-(t + 1) // case["page"]) for t in _lengths(case)),
                "flops": 4 * (tokens + b) * g * d}
    rows = case["batch"] * case["n_kv"]
    n = case["budget"] + case["chunk"]
    moved = min(case["budget"], case["chunk"], max(1, case["recent"]))   # the protected ones among the new at least
    append = rows * case["chunk"] * (4 * d * e + 12)
    return {"bytes": append + rows * n * 8 + rows * moved * (4 * d * e + 16), "flops": rows * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 11)


def _rope_tables(length, dim):
    inv = 1.0 / (ROPE_THETA ** (torch.arange(0, dim, 2, device=DEV, dtype=torch.float32) / dim))
    ang = torch.outer(torch.arange(length, device=DEV, dtype=torch.float32), inv)
    return ang.cos(), ang.sin()


def _pool(case, lengths, capacity, g):
    """Pages of keys and values in random order; each sequence's table lists
    its pages and ends with -1."""
    b, h, d, ps = case["batch"], case["n_kv"], case["dim"], case["page"]
    dt = DTYPES[case["dtype"]]
    need = [-(-c // ps) for c in capacity]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (total, ps, h, d) if case.get("layout") == "tokens" else (total, h, ps, d)
    k = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)
    v = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dt)
    if case.get("layout") == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)      # [pages, heads, slots, dim] over token-major memory
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    return k, v, table, lens


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "quantize":
        dt = DTYPES[case["dtype"]]
        x = torch.randn(case["rows"], case["cols"], generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn(1, case["cols"], generator=g, device=DEV))     # channels of unlike size
        x = (x * (1.0 if case["given"] else 0.02)).to(dt)
        scale = torch.full((1,), 0.01 + 0.001 * (seed % 7), device=DEV) if case["given"] and case["format"] == "nvfp4" else None
        return {"case": case, "x": x, "g": scale}
    if op == "linear":
        dt, fmt = DTYPES[case["dtype"]], case["format"]
        w = torch.randn(case["n"], case["k"], generator=g, device=DEV) * 0.02
        codes, scales, wg = _plain_quantize(w, fmt, None)
        del w
        x = torch.randn(case["m"], case["k"], generator=g, device=DEV).to(dt)
        bias = torch.randn(case["n"], generator=g, device=DEV).to(dt) if case["bias"] else None
        xg = torch.full((1,), 0.004, device=DEV) if fmt == "nvfp4" else None     # as a calibration gives it
        return {"case": case, "x": x, "xg": xg, "codes": _pack(codes), "scales": _tile_scales(scales), "wg": wg, "bias": bias}
    h, d = case["n_kv"], case["dim"]
    dt = DTYPES[case["dtype"]]
    if op == "attend":
        lens = _lengths(case)
        k, v, table, seq_lens = _pool(case, lens, [n + 1 for n in lens], g)
        qkv = torch.randn(case["batch"], (case["n_q"] + 2 * h) * d, generator=g, device=DEV).to(dt)
        positions = seq_lens.to(torch.int64) + 5          # the cache may have lost tokens before
        cos, sin = _rope_tables(case["longest"] + 8, d)
        s = {"case": case, "qkv": qkv, "k": k, "v": v, "table": table, "lens": seq_lens, "positions": positions,
             "cos": cos, "sin": sin, "longest": max(lens), "scores": None, "slot_pos": None}
        if case["weights"]:
            shape = (k.shape[0], h, case["page"])
            s["scores"] = torch.rand(shape, generator=g, device=DEV)
            s["slot_pos"] = torch.randint(0, case["longest"] + 1, shape, generator=g, device=DEV, dtype=torch.int32)
        return s
    b, budget, chunk = case["batch"], case["budget"], case["chunk"]
    n = budget + chunk
    k, v, table, seq_lens = _pool(case, [budget] * b, [n] * b, g)
    shape = (k.shape[0], h, case["page"])
    scores = torch.rand(shape, generator=g, device=DEV).square()      # few heavy tokens, many light ones
    slot_pos = torch.zeros(shape, dtype=torch.int32, device=DEV)
    # the cached tokens' positions: the first `budget`, in an order that earlier evictions left
    where = torch.arange(budget, device=DEV)
    pages, offs = table[:, where // case["page"]].long(), where % case["page"]
    perm = torch.rand(b, h, budget, generator=g, device=DEV).argsort(dim=-1).to(torch.int32)
    slot_pos[pages[:, None, :], torch.arange(h, device=DEV)[None, :, None], offs[None, None, :]] = perm
    new = torch.randn(2, b, chunk, h, d, generator=g, device=DEV).to(dt)
    new_scores = torch.rand(b, h, chunk, generator=g, device=DEV).square()
    first = torch.full((b,), budget, dtype=torch.int64, device=DEV)
    # the chunk's keys come rotated out of its own attention
    return {"case": case, "k_new": new[0], "v_new": new[1], "new_scores": new_scores, "first": first, "k": k, "v": v,
            "table": table, "lens": seq_lens, "scores": scores, "slot_pos": slot_pos}


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _to_e2m1(y):
    """Codes of the nearest E2M1 values, ties to the even code, saturating."""
    a = y.abs()
    c = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8)
         + (a >= 1.75).to(torch.uint8) + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8)
         + (a > 5.0).to(torch.uint8))
    return c | (torch.signbit(y).to(torch.uint8) << 3)


def _tensor_scale(x):
    """nvfp4: the fp32 scale of a tensor, its largest magnitude over 448 * 6."""
    return (x.float().abs().amax() / 2688.0).clamp(min=2.0 ** -100).reshape(1)


def _plain_quantize(x, fmt, g):
    """(codes [rows, padded columns], scales as bytes [rows, blocks], g)."""
    n, k = x.shape
    blk = BLOCK[fmt]
    xp = torch.nn.functional.pad(x.float(), (0, _pad64(k) - k)).reshape(n, -1, blk)
    amax = xp.abs().amax(dim=-1)
    if fmt == "nvfp4":
        g = _tensor_scale(x) if g is None else g
        sc = (amax * (1.0 / (6.0 * g))).clamp(max=448.0).to(torch.float8_e4m3fn)
        sf = sc.float()
        r = torch.where(sf > 0, 1.0 / (sf * g), torch.zeros_like(sf))
        raw = sc.view(torch.uint8)
    else:
        g = None
        raw = ((amax.view(torch.int32) >> 23) - 2).clamp(min=0)
        r = ((254 - raw) << 23).view(torch.float32)
        raw = raw.to(torch.uint8)
    return _to_e2m1(xp * r[..., None]).reshape(n, -1), raw, g


def _pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def _tile_scales(raw):
    n, nb = raw.shape
    p = torch.nn.functional.pad(raw, (0, -nb % 4, 0, -n % 128))
    t = p.reshape(p.shape[0] // 128, 4, 32, p.shape[1] // 4, 4)      # (row tile, row // 32, row % 32, block tile, block % 4)
    return t.permute(0, 3, 2, 1, 4).contiguous().reshape(-1)


def _untile_scales(flat, n, nb):
    nt, kt = -(-n // 128), -(-nb // 4)
    t = flat.reshape(nt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return t.reshape(nt * 128, kt * 4)[:n, :nb]


def _plain_values(codes, raw, fmt, g):
    """The values that codes [rows, padded columns] stand for, in fp32."""
    table = torch.tensor(E2M1, device=codes.device)
    v = table[codes.to(torch.int32)].reshape(codes.shape[0], -1, BLOCK[fmt])
    if fmt == "nvfp4":
        s = raw.contiguous().view(torch.float8_e4m3fn).float() * g
    else:
        s = torch.ldexp(torch.ones((), device=raw.device), raw.to(torch.int32) - 127)
    return (v * s[..., None]).reshape(codes.shape[0], -1)


def _plain_quantize_run(s):
    c, x = s["case"], s["x"]
    codes, raw, g = _plain_quantize(x, c["format"], s["g"])
    return _plain_values(codes, raw, c["format"], g)[:, :c["cols"]].to(x.dtype)


def _plain_linear(s):
    c, x, fmt = s["case"], s["x"], s["case"]["format"]
    codes, raw, g = _plain_quantize(x, fmt, s["xg"])
    a = _plain_values(codes, raw, fmt, g)
    wc = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=-1).reshape(c["n"], -1)
    w = _plain_values(wc, _untile_scales(s["scales"], c["n"], wc.shape[1] // BLOCK[fmt]), fmt, s["wg"])
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def _rotate(x, cos, sin):
    """Rotary embedding of x [..., d], halves paired, in fp32, kept in x's type."""
    x1, x2 = x.float().chunk(2, dim=-1)
    return torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1).to(x.dtype)


def _plain_attend(s):
    c = s["case"]
    b, h, d, ps, nq = c["batch"], c["n_kv"], c["dim"], c["page"], c["n_q"]
    lens, dev = s["lens"].long(), s["qkv"].device
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    q, k, v = s["qkv"].view(b, nq + 2 * h, d).split([nq, h, h], dim=1)
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    bi, hi = torch.arange(b, device=dev)[:, None], torch.arange(h, device=dev)[None, :]
    page, off = s["table"][bi[:, 0], lens // ps].long()[:, None], (lens % ps)[:, None]
    s["k"][page, hi, off] = k
    s["v"][page, hi, off] = v
    n = s["longest"] + 1
    slot = torch.arange(n, device=dev)
    live = slot[None, :] <= lens[:, None]
    pages = s["table"][:, slot // ps].long().clamp(min=0)
    at = (pages[:, None, :], torch.arange(h, device=dev)[None, :, None], (slot % ps)[None, None, :])
    kk, vv = s["k"][at].float(), s["v"][at].float()                      # [b, h, n, d]
    sc = (q.float().reshape(b, h, nq // h, d) @ kk.transpose(2, 3)) * (d ** -0.5)
    sc = sc.masked_fill(~live[:, None, None, :], -math.inf)
    p = torch.exp(sc - sc.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    vv = vv * live[:, None, :, None]
    out = (p @ vv).reshape(b, nq * d).to(s["qkv"].dtype)
    res = {"out": out, "k": s["k"], "v": s["v"]}
    if s["scores"] is not None:
        add = p.sum(dim=2)                                               # [b, h, n]
        old = torch.where(slot[None, None, :] < lens[:, None, None], s["scores"][at], torch.zeros_like(add))
        idx = live[:, None, :].expand(b, h, n).nonzero(as_tuple=True)
        full = tuple(t.expand(b, h, n)[idx] for t in at)
        s["scores"][full] = (old + add)[idx]
        s["slot_pos"][page, hi, off] = s["positions"].to(torch.int32)[:, None].expand(b, h)
        res |= {"scores": s["scores"], "slot_pos": s["slot_pos"]}
    return res


def _plain_evict(s):
    c = s["case"]
    b, h, ps, m, budget = c["batch"], c["n_kv"], c["page"], c["chunk"], c["budget"]
    lens, dev = s["lens"].long(), s["k"].device
    # the chunk goes behind the cached tokens
    t = torch.arange(m, device=dev)
    pos = s["first"][:, None] + t[None, :]
    slot = lens[:, None] + t[None, :]
    page, off = s["table"].long().gather(1, slot // ps)[:, :, None], (slot % ps)[:, :, None]
    hi = torch.arange(h, device=dev)[None, None, :]
    s["k"][page, hi, off] = s["k_new"]
    s["v"][page, hi, off] = s["v_new"]
    s["scores"][page, hi, off] = s["new_scores"].transpose(1, 2)
    s["slot_pos"][page, hi, off] = pos.to(torch.int32)[:, :, None].expand(b, m, h)
    # the budget's worth of tokens that stay: the recent ones, then the heaviest
    n = budget + m
    slots = torch.arange(n, device=dev)
    at = (s["table"][:, slots // ps].long()[:, None, :], torch.arange(h, device=dev)[None, :, None],
          (slots % ps)[None, None, :])
    key, p = s["scores"][at], s["slot_pos"][at]
    key = torch.where(key.isnan(), torch.full_like(key, -math.inf), key)
    newest = p.amax(dim=-1, keepdim=True)
    key = torch.where(p > newest - c["recent"], torch.full_like(key, math.inf), key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(b, h, n, dtype=torch.bool, device=dev).scatter_(2, order[..., :budget], True)
    # the kept tokens behind the budget fill the holes before it, both in ascending order
    src = kept[..., budget:].nonzero(as_tuple=True)
    dst = (~kept[..., :budget]).nonzero(as_tuple=True)
    at = [x.expand(b, h, n) for x in at]
    fr = tuple(x[src[0], src[1], src[2] + budget] for x in at)
    to = tuple(x[dst] for x in at)
    for name in ("k", "v", "scores", "slot_pos"):
        s[name][to] = s[name][fr]
    s["lens"].fill_(budget)
    s["first"].add_(m)                                                    # where the next chunk's positions begin
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "slot_pos": s["slot_pos"], "lens": s["lens"]}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _cache(ts, s):
    return ts.PagedKVCache(s["k"], s["v"], s["table"], s["lens"], scores=s["scores"], slot_pos=s["slot_pos"])


def run(state):
    c = state["case"]
    op = c["op"]
    if not own:
        return {"quantize": _plain_quantize_run, "linear": _plain_linear, "attend": _plain_attend,
                "evict": _plain_evict}[op](state)
    import tensorshrink_b200 as ts
    s = state
    if op == "quantize":
        return ts.fp4_dequantize(ts.fp4_quantize(s["x"], c["format"], global_scale=s["g"]), s["x"].dtype)
    if op == "linear":
        w = ts.Fp4Tensor(s["codes"], s["scales"], s["wg"], c["n"], c["k"], c["format"])
        return ts.fp4_linear(s["x"], w, bias=s["bias"], input_scale=s["xg"])
    cache = _cache(ts, s)
    if op == "attend":
        out = ts.paged_decode_attention(s["qkv"], c["n_q"], cache, s["positions"], s["cos"], s["sin"],
                                        accumulate=c["weights"])
        res = {"out": out, "k": s["k"], "v": s["v"]}
        if c["weights"]:
            res |= {"scores": s["scores"], "slot_pos": s["slot_pos"]}
        return res
    ts.paged_append(s["k_new"], s["v_new"], cache, s["first"], scores=s["new_scores"])
    cache.advance(c["chunk"])
    ts.paged_evict(cache, c["budget"], recent=c["recent"])
    s["first"].add_(c["chunk"])
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "slot_pos": s["slot_pos"], "lens": s["lens"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _grid(y, bits, least, most):
    """y (64 bits) rounded to a binary grid of `bits` fraction bits whose
    smallest exponent is `least`, ties to even, saturating at `most`."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -1000))).clamp(min=least)
    step = torch.exp2(e - bits)
    return (torch.round(y / step) * step).clamp(-most, most)


def _exact_scales(x, fmt, g):
    n, k = x.shape
    blk = BLOCK[fmt]
    xp = torch.zeros(n, -(-k // blk) * blk, dtype=torch.float64, device=x.device)
    xp[:, :k] = x
    xp = xp.view(n, -1, blk)
    top = xp.abs().amax(-1)
    if fmt == "nvfp4":
        g = float(g) if g is not None else float(x.double().abs().max()) / 2688
        return xp, _grid(top / (6 * g), 3, -6, 448.0) * g
    return xp, torch.exp2((torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2).clamp(min=-127))


def _exact_values(x, fmt, g):
    xp, s = _exact_scales(x, fmt, g)
    q = _grid(xp / s.clamp(min=2.0 ** -300)[..., None], 1, 0, 6.0)
    return (q * s[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _exact_weight(s):
    """The weight's values from its bytes, in 64 bits."""
    c = s["case"]
    n, k, blk = c["n"], c["k"], BLOCK[c["format"]]
    cols = torch.arange(k, device=DEV)
    byte = s["codes"][:, cols // 2].to(torch.int64)
    code = torch.where(cols % 2 == 0, byte & 15, byte >> 4)
    e, man = (code >> 1) & 3, code & 1
    mag = torch.where(e == 0, man * 0.5, (1 + man * 0.5) * torch.exp2(e.double() - 1))
    mag = torch.where(code >= 8, -mag, mag)
    nbt = -(-(_pad64(k) // blk) // 4)
    r, j = torch.arange(n, device=DEV)[:, None], torch.arange(-(-k // blk), device=DEV)[None, :]
    raw = s["scales"][((r // 128) * nbt + j // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4].to(torch.int64)
    if c["format"] == "nvfp4":
        e, man = raw >> 3, raw & 7
        sc = torch.where(e == 0, man * 2.0 ** -9, (8 + man) * torch.exp2(e.double() - 10)) * float(s["wg"])
    else:
        sc = torch.exp2(raw.double() - 127)
    return mag * sc[:, cols // blk]


def _rotate64(x, cos, sin):
    d = x.shape[-1] // 2
    a, b = x[..., :d].double(), x[..., d:].double()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _exact_attend(s):
    c = s["case"]
    b, h, d, ps, nq = c["batch"], c["n_kv"], c["dim"], c["page"], c["n_q"]
    dt = s["qkv"].dtype
    x = s["qkv"].view(b, nq + 2 * h, d)
    out = torch.empty(b, nq, d, dtype=torch.float64, device=DEV)
    ko = s["k"].clone()
    vo = s["v"].clone()
    so = None if s["scores"] is None else s["scores"].double()
    for i in range(b):
        n = int(s["lens"][i])
        cos, sin = s["cos"][s["positions"][i]].double(), s["sin"][s["positions"][i]].double()
        q = _rotate64(x[i, :nq], cos, sin).to(dt).double()           # held in the cache's type
        k = _rotate64(x[i, nq:nq + h], cos, sin).to(dt)
        slot = torch.arange(n + 1, device=DEV)
        page, off = s["table"][i, slot // ps].long(), slot % ps
        ko[page[n], :, off[n]] = k
        vo[page[n], :, off[n]] = x[i, nq + h:]
        for j in range(h):
            kk, vv = ko[page, j, off].double(), vo[page, j, off].double()
            qs = q[j * (nq // h):(j + 1) * (nq // h)]
            p = torch.softmax(qs @ kk.t() / math.sqrt(d), dim=-1)
            out[i, j * (nq // h):(j + 1) * (nq // h)] = p @ vv
            if so is not None:
                so[page[n], j, off[n]] = 0.0
                so[page, j, off] += p.sum(0)
    res = {"out": out.reshape(b, -1), "k": ko, "v": vo}
    if so is not None:
        res |= {"scores": so, "slot_pos": None}
    return res


def _exact_evict(s):
    c = s["case"]
    b, h, ps, m, budget = c["batch"], c["n_kv"], c["page"], c["chunk"], c["budget"]
    if b * h * (budget + m) > 6_000_000:
        return None
    k, v = s["k"].clone(), s["v"].clone()
    score, where = s["scores"].cpu().numpy().copy(), s["slot_pos"].cpu().numpy().copy()
    table, lens, first = s["table"].cpu().numpy(), s["lens"].tolist(), s["first"].tolist()
    given = s["new_scores"].cpu().numpy()
    for i in range(b):
        slot = lens[i] + np.arange(m)
        page, off = table[i, slot // ps], slot % ps
        pos = first[i] + np.arange(m)
        pt, ot = torch.from_numpy(page).long().to(DEV), torch.from_numpy(off).to(DEV)
        k[pt, :, ot] = s["k_new"][i]
        v[pt, :, ot] = s["v_new"][i]
        n = lens[i] + m
        allp, allo = table[i, np.arange(n) // ps], np.arange(n) % ps
        for j in range(h):
            score[page, j, off] = given[i, j]
            where[page, j, off] = pos
            w, p = score[allp, j, allo].astype(np.float64), where[allp, j, allo]
            w[np.isnan(w)] = -np.inf
            w[p > p.max() - c["recent"]] = np.inf
            stay = np.zeros(n, bool)
            stay[np.lexsort((np.arange(n), -w))[:budget]] = True
            fr = np.nonzero(stay[budget:])[0] + budget
            to = np.nonzero(~stay[:budget])[0]
            a, ao, z, zo = allp[fr], allo[fr], allp[to], allo[to]
            score[z, j, zo], where[z, j, zo] = score[a, j, ao], where[a, j, ao]
            a, ao, z, zo = (torch.from_numpy(np.asarray(y, dtype=np.int64)).to(DEV) for y in (a, ao, z, zo))
            k[z, j, zo], v[z, j, zo] = k[a, j, ao], v[a, j, ao]
    return {"k": k, "v": v, "scores": torch.from_numpy(score).double(), "slot_pos": None, "lens": None}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_values(s["x"], case["format"], s["g"])
    if op == "linear":
        y = _exact_values(s["x"], case["format"], s["xg"]) @ _exact_weight(s).t()
        return y if s["bias"] is None else y + s["bias"].double()
    return _exact_attend(s) if op == "attend" else _exact_evict(s)
