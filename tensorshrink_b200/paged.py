"""A paged key-value cache: sequences of unequal length in pages of a common
pool, attention of one new token over it, and eviction by accumulated
attention weight.

`decode_attention` of `kernels` serves sequences that all stand at one
position of a dense cache; here every sequence has its own length, position
and list of pages. The reference keeps no cache of its own (its models
bring theirs). The functions are thin layers over
`torch.ops.tensorshrink.paged_*`, which check their arguments and launch on the
current stream of the cache's device; nothing synchronises, so calls can be
captured in a graph.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .fp4 import _op


class PagedKVCache:
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

    def _args(self):
        return self.k_pages, self.v_pages, self.page_table, self.seq_lens, self.scores, self.slot_pos


def paged_append(k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, positions: Optional[torch.Tensor] = None,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                 n_new: Optional[torch.Tensor] = None, scores: Optional[torch.Tensor] = None) -> None:
    """Store new tokens (a prompt, or a chunk of one) behind the cached ones:
    k, v [batch, tokens, n_kv, head_dim] go to slots seq_lens[b] + t, k rotated to
    position positions[b] + t (int64 [batch]; None: the slot's number) when
    rotary tables (fp32 [positions, head_dim / 2]) are given. n_new (int32
    [batch]): how many of a sequence's tokens count. scores (fp32 [batch,
    n_kv, tokens]): the slots' initial scores (default 0). Tokens without a
    slot, a page or a rotary row are dropped. seq_lens is not changed (see
    `PagedKVCache.advance`)."""
    _op("paged_append")(k, v, *cache._args(), positions, rope_cos, rope_sin, n_new, scores)


def paged_decode_attention(qkv: torch.Tensor, n_q: int, cache: PagedKVCache, positions: Optional[torch.Tensor] = None,
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
    zeros and stores nothing. Returns [batch, n_q head_dim] in qkv's type.
    seq_lens is not changed (see `PagedKVCache.advance`)."""
    args = (qkv, n_q, *cache._args(), positions, rope_cos, rope_sin, scale, accumulate)
    if out is not None:
        return _op("paged_decode_attention", "out")(*args, out=out)
    return _op("paged_decode_attention")(*args)


def paged_evict(cache: PagedKVCache, budget: int, recent: int = 0) -> None:
    """Cut every sequence longer than `budget` back to `budget` tokens per kv
    head: the `recent` newest positions stay, then the slots of the largest
    scores (equal ones: the lowest slot; NaN counts as -inf). Kept slots at or
    behind `budget` move into the holes before it, both in ascending order,
    and seq_lens becomes `budget`; pages behind it are free. The pages of a
    sequence must not be shared with another one."""
    _op("paged_evict")(*cache._args(), budget, recent)
