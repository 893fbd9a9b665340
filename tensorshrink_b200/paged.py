"""A paged key-value cache: sequences of unequal length in pages of a common
pool, in 16 or 8 bits, attention of one new token over it, eviction by
accumulated attention weight, and the page tables of a batch of requests; and what
comes in front of the cache, norms and rotation of queries and keys.

`decode_attention` of `kernels` serves sequences that all stand at one
position of a dense cache; here every sequence has its own length, position
and list of pages. The reference keeps no cache of its own (its models
bring theirs). The functions are thin layers over
`torch.ops.tensorshrink.paged_*`, `paged8_*` and `qk_norm_rope*`, which check their arguments and launch on the
current stream of the cache's device; nothing synchronises, so calls can be
captured in a graph.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from .fp4 import _op


class _Paged:
    """What caches of both widths tell of their pages."""

    __slots__ = ()

    @property
    def batch(self) -> int:
        return self.page_table.shape[0]

    @property
    def n_kv(self) -> int:
        return self.k_pages.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_pages.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k_pages.shape[3]

    @property
    def capacity(self) -> int:
        """Slots that a sequence's row of the page table can name."""
        return self.page_table.shape[1] * self.page_size

    def advance(self, n: Union[int, torch.Tensor] = 1) -> None:
        """Count `n` appended tokens as cached, or n[b] of sequence b (int32
        [batch]). (A negative count, of a sequence that takes no part, has to
        be put back by the caller, and a token that found no slot is not to be
        counted.)"""
        self.seq_lens.add_(n)


class PagedKVCache(_Paged):
    """Keys and values of a batch of sequences in pages.

    k_pages, v_pages: fp16 or bf16 [num_pages, n_kv, page_size, head_dim],
    any strides with contiguous rows (a token-major pool is a transposed
    view), the same for both. page_table: int32 [batch, max_pages]; slot s of
    sequence b is row s % page_size of page page_table[b, s // page_size]; an
    entry outside the pool (e.g. -1) has no memory. seq_lens: int32 [batch],
    the cached tokens of each sequence (negative: the sequence takes no part).
    scores (fp32) and slot_pos (int32), both [num_pages, n_kv, page_size]:
    each slot's accumulated attention weight and its token's position, needed
    by eviction."""

    __slots__ = ("k_pages", "v_pages", "page_table", "seq_lens", "scores", "slot_pos")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, scores: Optional[torch.Tensor] = None,
                 slot_pos: Optional[torch.Tensor] = None):
        _op("paged_check")(k_pages, v_pages, page_table, seq_lens, scores, slot_pos)
        self.k_pages, self.v_pages = k_pages, v_pages
        self.page_table, self.seq_lens = page_table, seq_lens
        self.scores, self.slot_pos = scores, slot_pos

    @classmethod
    def allocate(cls, batch: int, n_kv: int, head_dim: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", track: bool = False) -> "PagedKVCache":
        """A pool with room for `max_len` tokens of every sequence, its pages
        dealt out in order. `track`: keep scores and positions."""
        per = -(-max_len // page_size)
        shape = (batch * per, n_kv, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        lens = torch.zeros(batch, dtype=torch.int32, device=device)
        scores = torch.zeros(shape[:3], dtype=torch.float32, device=device) if track else None
        slot_pos = torch.zeros(shape[:3], dtype=torch.int32, device=device) if track else None
        return cls(k, v, table, lens, scores, slot_pos)

    def _args(self):
        return self.k_pages, self.v_pages, self.page_table, self.seq_lens, self.scores, self.slot_pos


class PagedKVCache8(_Paged):
    """Keys and values of a batch of sequences in pages of 8 bits.

    k_pages, v_pages: int8 or float8_e4m3fn [num_pages, n_kv, page_size,
    head_dim], any strides with contiguous rows, the same for both. k_scales,
    v_scales: fp32, contiguous [num_pages, n_kv, page_size / block]: `block`
    neighbouring slots (a multiple of 16) of a kv head share a scale, and a
    code stands for code * scale. page_table and seq_lens as in
    `PagedKVCache`. int8 codes are -127 to 127. There is no eviction from such a
    cache: slots that move to another block would be rounded anew."""

    __slots__ = ("k_pages", "v_pages", "k_scales", "v_scales", "page_table", "seq_lens")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                 page_table: torch.Tensor, seq_lens: torch.Tensor):
        _op("paged8_check")(k_pages, v_pages, k_scales, v_scales, page_table, seq_lens)
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self.page_table, self.seq_lens = page_table, seq_lens

    @classmethod
    def allocate(cls, batch: int, n_kv: int, head_dim: int, max_len: int, page_size: int = 64, block: int = 16,
                 dtype: torch.dtype = torch.int8, device="cuda") -> "PagedKVCache8":
        """A pool with room for `max_len` tokens of every sequence, its pages
        dealt out in order."""
        per = -(-max_len // page_size)
        if block <= 0 or page_size % block:
            raise ValueError(f"pages of {page_size} tokens do not hold whole blocks of {block}")
        shape = (batch * per, n_kv, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.ones(*shape[:2], page_size // block, dtype=torch.float32, device=device) for _ in range(2))
        table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        return cls(k, v, ks, vs, table, torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def block(self) -> int:
        """Tokens of a kv head that share a scale."""
        return self.page_size // self.k_scales.shape[2]

    def _args(self):
        return self.k_pages, self.v_pages, self.k_scales, self.v_scales, self.page_table, self.seq_lens


AnyCache = Union[PagedKVCache, PagedKVCache8]


def paged_append(k: torch.Tensor, v: torch.Tensor, cache: AnyCache, positions: Optional[torch.Tensor] = None,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                 n_new: Optional[torch.Tensor] = None, scores: Optional[torch.Tensor] = None,
                 offsets: Optional[torch.Tensor] = None) -> None:
    """Store new tokens (a prompt, or a chunk of one) behind the cached ones:
    k, v [batch, tokens, n_kv, head_dim] go to slots seq_lens[b] + t, k rotated to
    position positions[b] + t (int64 [batch]; None: the slot's number) when
    rotary tables (fp32 [positions, head_dim / 2]) are given. n_new (int32
    [batch]): how many of a sequence's tokens count. scores (fp32 [batch,
    n_kv, tokens]): the slots' initial scores (default 0). Tokens without a
    slot, a page or a rotary row are dropped. seq_lens is not changed (see
    `PagedKVCache.advance`).

    A cache of 8 bits keeps no scores, and takes packed tokens too: with offsets
    (int32 [batch + 1], as `paged_reserve` gives them) k and v are [tokens, n_kv,
    head_dim], sequence b's from offsets[b] to offsets[b + 1]. k and v (fp16
    or bf16; k after its rotation) are quantised block by block. A block
    that holds earlier tokens keeps its scale if that is large enough;
    otherwise the scale grows, by a quarter at least, and the earlier tokens' codes
    are rounded anew: int8 codes are off by 2.5 steps at most then, e4m3 values by
    (1 + 2^-4)^(growths + 1) - 1 of themselves, 15% of the block's largest. An infinity or a NaN makes its block's scale NaN, which
    stays until a token comes to the block's first slot again. Sequences must
    not share a page that gets tokens."""
    if isinstance(cache, PagedKVCache8):
        if scores is not None:
            raise ValueError("scores were given for a cache that keeps none")
        _op("paged8_append")(k, v, *cache._args(), positions, rope_cos, rope_sin, n_new, offsets)
        return
    if offsets is not None:
        raise NotImplementedError("packed tokens go to a cache of 16 bits through qk_norm_rope (cache=, slots=)")
    _op("paged_append")(k, v, *cache._args(), positions, rope_cos, rope_sin, n_new, scores)


def paged_decode_attention(qkv: torch.Tensor, n_q: int, cache: AnyCache, positions: Optional[torch.Tensor] = None,
                           rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None, accumulate: bool = False,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One decode step of grouped-query attention over the cache.

    qkv [batch, (n_q + 2 n_kv) head_dim] holds each sequence's new token; q
    and k are rotated to positions[b] (int64 [batch]) when rotary tables are
    given; k and v are stored in slot seq_lens[b]; every query head attends over
    slots [0, seq_lens[b]] with scores scale * q.k (default head_dim ** -0.5).
    `accumulate`: add to each slot's score the weights that its kv head's
    query heads gave it; sequences must not share pages then (each adds to its own
    slots' scores, and one of two additions to the same would be lost). A sequence that has no slot for the token (negative
    seq_lens, no page left, a position without a rotary row) answers with
    zeros and stores nothing. Returns [batch, n_q head_dim] in qkv's type, or
    `out`, which may be qkv's own query columns and shares no other memory with it.
    seq_lens is not changed (see `PagedKVCache.advance`).

    Over a cache of 8 bits (which accumulates nothing) the token is stored as
    `paged_append` stores it, and attended to as it is stored."""
    if isinstance(cache, PagedKVCache8):
        if accumulate:
            raise ValueError("the cache has no scores to accumulate into")
        args = (qkv, n_q, *cache._args(), positions, rope_cos, rope_sin, scale)
        name = "paged8_decode_attention"
    else:
        args = (qkv, n_q, *cache._args(), positions, rope_cos, rope_sin, scale, accumulate)
        name = "paged_decode_attention"
    if out is not None:
        return _op(name, "out")(*args, out=out)
    return _op(name)(*args)


def paged_attention(q: torch.Tensor, cache: PagedKVCache8, positions: Optional[torch.Tensor] = None,
                    rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per sequence over what a cache of 8 bits
    holds, slots [0, seq_lens[b]); nothing is stored. q [batch, n_q head_dim]
    (fp16 or bf16) is rotated to positions[b] when rotary tables are given;
    scores are scale * q.k (default head_dim ** -0.5). Slots without a page do
    not count; a sequence without tokens, or with a position that has no
    rotary row, answers with zeros. Returns [batch, n_q head_dim] in q's type, or
    `out`, which may be q itself and overlaps it in no other way."""
    if not isinstance(cache, PagedKVCache8):
        raise NotImplementedError("paged_attention reads a cache of 8 bits (paged_decode_attention reads both)")
    args = (q, *cache._args(), positions, rope_cos, rope_sin, scale)
    if out is not None:
        return _op("paged8_attention", "out")(*args, out=out)
    return _op("paged8_attention")(*args)


def paged_dequantize(cache: PagedKVCache8, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of all pages of a cache of 8 bits: keys and values, contiguous
    [num_pages, n_kv, page_size, head_dim] of `dtype`."""
    if not isinstance(cache, PagedKVCache8):
        raise NotImplementedError("a cache of 16 bits holds its values as they are")
    return _op("paged8_dequantize")(*cache._args(), dtype)


def paged_evict(cache: PagedKVCache, budget: int, recent: int = 0) -> None:
    """Cut every sequence longer than `budget` back to `budget` tokens per kv
    head: the `recent` newest positions stay, then the slots of the largest
    scores (equal ones: the lowest slot; NaN counts as -inf). Kept slots at or
    behind `budget` move into the holes before it, both in ascending order,
    and seq_lens becomes `budget`; pages behind it are free. The pages of a
    sequence must not be shared with another one."""
    if isinstance(cache, PagedKVCache8):
        raise NotImplementedError("there is no eviction from a cache of 8 bits")
    _op("paged_evict")(*cache._args(), budget, recent)


class PagePool:
    """The pages that no sequence holds, as a stack: free (int32 [pages]), of
    which the first n_free (int32, one value) are free and the last of those is
    taken first."""

    __slots__ = ("free", "n_free")

    def __init__(self, free: torch.Tensor, n_free: torch.Tensor):
        _op("pool_check")(free, n_free)
        self.free, self.n_free = free, n_free

    @classmethod
    def allocate(cls, num_pages: int, device="cuda") -> "PagePool":
        """All of `num_pages` pages free, page 0 taken first."""
        free = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(free, torch.full((1,), num_pages, dtype=torch.int32, device=device))


class PagedSlots(NamedTuple):
    """What `paged_reserve` found. granted (int32 [batch]): how many of its new
    tokens each sequence has room for, all or 0. offsets (int32 [batch + 1]):
    where each sequence's tokens begin in a packed batch. Of each packed token: its
    slot in the pages (int64, page * page_size + offset; -1: none), its position
    (int64; 0 without a slot) and its sequence (int32; -1 behind the last
    token)."""
    granted: torch.Tensor
    offsets: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    sequences: torch.Tensor


def paged_reserve(pool: PagePool, cache: AnyCache, n_new: torch.Tensor, tokens: int,
                  positions: Optional[torch.Tensor] = None) -> PagedSlots:
    """Pages for n_new[b] (int32 [batch]) tokens behind each sequence's cached
    ones, and the slots of all new tokens packed one sequence after the other into
    `tokens` places (at least their sum).

    Entries of the page table that the tokens need and that name no page get
    one from the pool; an entry that names one keeps it. Sequences are served in
    order, each for all of its tokens or for none; the first that needs more
    pages than are left, and those behind it that need any, get nothing, nor does
    a sequence out of use (negative seq_lens) or one that would pass the
    table's end. positions (int64 [batch]): the position of each sequence's first new
    token (None: its slot's number). seq_lens is not changed: `cache.advance(granted)`
    once the tokens are stored. Caches of several layers can share one page
    table and seq_lens."""
    return PagedSlots(*_op("paged_reserve")(pool.free, pool.n_free, cache.page_table, cache.seq_lens, cache.page_size,
                                            cache.k_pages.shape[0], n_new, positions, tokens))


def paged_release(pool: PagePool, cache: AnyCache, keep: torch.Tensor) -> None:
    """Cut sequences back to keep[b] tokens (int32 [batch]; 0: the request is
    over; negative: left alone) and return the pages that they no longer need, in order of
    the sequences and of their pages: seq_lens[b] becomes min(seq_lens[b], keep[b]), the
    pages' entries -1. Sequences must not share such pages."""
    _op("paged_release")(pool.free, pool.n_free, cache.page_table, cache.seq_lens, cache.page_size, cache.k_pages.shape[0],
                         keep)


def qk_norm_rope(qkv: torch.Tensor, n_q: int, n_kv: int, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 out: Optional[torch.Tensor] = None, cache: Optional[PagedKVCache] = None,
                 slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Norms of each query and key head, and their rotation, in one pass.

    qkv [tokens, (n_q + 2 n_kv) head_dim] (fp16 or bf16): query, key and value
    heads. A query (key) head becomes x * rsqrt(mean(x^2) + eps) * q_weight
    (k_weight; [head_dim], fp32 or qkv's type; None: no norm) and is then
    rotated to positions[t] (int64 [tokens]) when rotary tables are given, all in
    fp32 and rounded once; values are copied. A token whose position has no
    rotary row comes out as zeros. Returns a tensor like qkv, or `out`, which
    may be qkv itself and overlaps it in no other way.

    With a cache of 16 bits and slots (int64 [tokens], as `paged_reserve` gives
    them) key and value heads also go to their slots in the pages, whose scores
    become 0 and positions the tokens', if the cache keeps them. A slot outside the pool
    is not written; no slot may be given twice. (For a cache of 8 bits, whose tokens share scales:
    `paged_append`.)"""
    args = (qkv, n_q, n_kv, q_weight, k_weight, positions, rope_cos, rope_sin, eps)
    name = "qk_norm_rope"
    if cache is not None or slots is not None:
        if isinstance(cache, PagedKVCache8):
            raise NotImplementedError("tokens go to a cache of 8 bits through paged_append")
        if cache is None or slots is None:
            raise ValueError("a cache and slots come both or neither")
        args += (*cache._args(), slots)
        name = "qk_norm_rope_store"
    if out is not None:
        return _op(name, "out")(*args, out=out)
    return _op(name)(*args)
