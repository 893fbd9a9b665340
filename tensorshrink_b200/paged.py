"""A paged key-value cache: sequences of unequal length in pages of a common
pool, attention of one new token over it, and eviction by accumulated
attention weight.

`decode_attention` of `kernels` serves sequences that all stand at one
position of a dense cache; here every sequence has its own length, position
and list of pages. The reference keeps no cache of its own (its models
bring theirs). Every launch goes to `torch.cuda.current_stream()` of the
cache's device; nothing synchronises, so calls can be captured in a graph.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _C
from .fp4 import _on
from .kernels import _ptr, _require_cuda, _serving_workspace, _stream_handle, dtype_code

_I64x3 = C.c_int64 * 3


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

    __slots__ = ("k_pages", "v_pages", "page_table", "seq_lens", "scores", "slot_pos", "_c")

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, scores: Optional[torch.Tensor] = None,
                 slot_pos: Optional[torch.Tensor] = None):
        _require_cuda(k_pages, v_pages, page_table, seq_lens, scores, slot_pos, what="PagedKVCache")
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
            raise ValueError("k_pages and v_pages must both be [num_pages, n_kv, page_size, head_dim]")
        if k_pages.dtype not in (torch.float16, torch.bfloat16) or v_pages.dtype != k_pages.dtype:
            raise NotImplementedError("the cache holds fp16 or bf16")
        if k_pages.stride() != v_pages.stride() or k_pages.stride(-1) != 1:
            raise ValueError("k_pages and v_pages must share their strides and have contiguous rows")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
            raise ValueError("page_table must be int32 [batch, max_pages] with contiguous rows")
        if seq_lens.dtype != torch.int32 or seq_lens.shape != page_table.shape[:1] or not seq_lens.is_contiguous():
            raise ValueError("seq_lens must be contiguous int32 [batch]")
        num_pages, n_kv, page_size, dim = k_pages.shape
        for t, dt, name in ((scores, torch.float32, "scores"), (slot_pos, torch.int32, "slot_pos")):
            if t is not None and (t.dtype != dt or t.shape != k_pages.shape[:3] or not t.is_contiguous()):
                raise ValueError(f"{name} must be contiguous {dt} [num_pages, n_kv, page_size]")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.page_table, self.seq_lens = page_table, seq_lens
        self.scores, self.slot_pos = scores, slot_pos
        sp, sh, st, _ = k_pages.stride()
        self._c = _C.TsPagedCache(
            k_pages.data_ptr(), v_pages.data_ptr(), sp, sh, st, page_table.data_ptr(), page_table.stride(0),
            seq_lens.data_ptr(), _ptr(scores), _ptr(slot_pos), dtype_code(k_pages.dtype), page_table.shape[0], n_kv,
            dim, page_size, num_pages, page_table.shape[1], 0)

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
        stats = [torch.zeros(shape[:3], dtype=dt, device=device) for dt in (torch.float32, torch.int32)] if track else [None] * 2
        return cls(k, v, table, lens, *stats)

    @property
    def batch(self) -> int:
        return self._c.batch

    @property
    def n_kv(self) -> int:
        return self._c.n_kv

    @property
    def head_dim(self) -> int:
        return self._c.head_dim

    @property
    def capacity(self) -> int:
        """Slots that a sequence's row of the page table can name."""
        return self._c.max_pages * self._c.page_size

    def advance(self, n: int = 1) -> None:
        """Count `n` appended tokens as cached. (A negative count, of a
        sequence that takes no part, has to be put back by the caller.)"""
        self.seq_lens.add_(n)


def _rope(cache: PagedKVCache, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], what: str) -> int:
    if cos is None and sin is None:
        return 0
    if cos is None or sin is None:
        raise ValueError(f"{what}: rope_cos and rope_sin come both or neither")
    for t in (cos, sin):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != cache.head_dim // 2 or not t.is_contiguous():
            raise ValueError(f"{what}: the rotary tables must be contiguous fp32 [positions, head_dim / 2]")
    if cos.shape != sin.shape:
        raise ValueError(f"{what}: the rotary tables differ in shape")
    return cos.shape[0]


def _per_sequence(t: Optional[torch.Tensor], cache: PagedKVCache, dtype: torch.dtype, what: str) -> None:
    if t is not None and (t.dtype != dtype or tuple(t.shape) != (cache.batch,) or not t.is_contiguous()):
        raise ValueError(f"{what} must be contiguous {dtype} [batch]")


def paged_append(k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, positions: Optional[torch.Tensor] = None,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None,
                 n_new: Optional[torch.Tensor] = None, scores: Optional[torch.Tensor] = None) -> None:
    """Store new tokens (a prompt, or a chunk of one) behind the cached ones:
    k, v [batch, tokens, n_kv, head_dim] go to slots seq_lens[b] + t, k rotated to
    position positions[b] + t (int64 [batch]; None: the slot's number) when
    rotary tables are given. n_new (int32 [batch]): how many of a sequence's
    tokens count. scores (fp32 [batch, n_kv, tokens]): the slots' initial
    scores (default 0). seq_lens is not changed (see `PagedKVCache.advance`)."""
    dev = _require_cuda(cache.k_pages, k, v, positions, rope_cos, rope_sin, n_new, scores, what="paged_append")
    rows = _rope(cache, rope_cos, rope_sin, "paged_append")
    c = cache._c
    if k.dim() != 4 or k.shape != v.shape or k.shape[0] != c.batch or tuple(k.shape[2:]) != (c.n_kv, c.head_dim):
        raise ValueError(f"k and v must be [batch, tokens, n_kv, head_dim], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != cache.k_pages.dtype or v.dtype != k.dtype:
        raise ValueError("k and v must have the cache's type")
    k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (k, v))
    _per_sequence(positions, cache, torch.int64, "positions")
    _per_sequence(n_new, cache, torch.int32, "n_new")
    if scores is not None:
        if cache.scores is None:
            raise ValueError("scores were given for a cache that keeps none")
        if scores.dtype != torch.float32 or tuple(scores.shape) != (c.batch, c.n_kv, k.shape[1]):
            raise ValueError("scores must be fp32 [batch, n_kv, tokens]")
    with _on(dev):
        rc = _C.load().ts_paged_append(
            k.data_ptr(), _I64x3(*k.stride()[:3]), v.data_ptr(), _I64x3(*v.stride()[:3]), k.shape[1], _ptr(n_new), c,
            _ptr(positions), _ptr(rope_cos), _ptr(rope_sin), rows, _ptr(scores),
            _I64x3(*scores.stride()) if scores is not None else None, _stream_handle(dev))
    _C.check(rc, "ts_paged_append")


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
    query heads gave it. A sequence that has no slot for the token (negative
    seq_lens, no page left, a position without a rotary row) answers with
    zeros. Returns [batch, n_q head_dim] in qkv's type. seq_lens is not
    changed (see `PagedKVCache.advance`)."""
    dev = _require_cuda(cache.k_pages, qkv, positions, rope_cos, rope_sin, out, what="paged_decode_attention")
    rows = _rope(cache, rope_cos, rope_sin, "paged_decode_attention")
    c = cache._c
    n_q = int(n_q)
    if n_q <= 0 or n_q % c.n_kv:
        raise ValueError(f"{n_q} query heads over {c.n_kv} kv heads")
    if qkv.dim() != 2 or tuple(qkv.shape) != (c.batch, (n_q + 2 * c.n_kv) * c.head_dim) or qkv.stride(1) != 1:
        raise ValueError(f"qkv must be [batch, (n_q + 2 n_kv) head_dim] with contiguous rows, got {tuple(qkv.shape)}")
    if qkv.dtype != cache.k_pages.dtype:
        raise ValueError("qkv must have the cache's type")
    _per_sequence(positions, cache, torch.int64, "positions")
    if positions is None and (rows or cache.slot_pos is not None):
        raise ValueError("positions are needed for the rotation and for slot_pos")
    if accumulate and cache.scores is None:
        raise ValueError("the cache has no scores to accumulate into")
    if out is None:
        out = torch.empty(c.batch, n_q * c.head_dim, dtype=qkv.dtype, device=dev)
    elif tuple(out.shape) != (c.batch, n_q * c.head_dim) or out.dtype != qkv.dtype or out.stride(1) != 1:
        raise ValueError("out must be [batch, n_q head_dim] of qkv's type with contiguous rows")
    lib = _C.load()
    acc = 1 if accumulate else 0
    with _on(dev):
        ws = _serving_workspace(dev, lib.ts_paged_attention_workspace_size(c, n_q, acc))
        rc = lib.ts_paged_decode_attention(
            qkv.data_ptr(), qkv.stride(0), n_q, c, _ptr(positions), _ptr(rope_cos), _ptr(rope_sin), rows,
            c.head_dim ** -0.5 if scale is None else scale, acc, out.data_ptr(), out.stride(0), ws.data_ptr(),
            ws.numel(), _stream_handle(dev))
    _C.check(rc, "ts_paged_decode_attention")
    return out


def paged_evict(cache: PagedKVCache, budget: int, recent: int = 0) -> None:
    """Cut every sequence longer than `budget` back to `budget` tokens per kv
    head: the `recent` newest positions stay, then the slots of the largest
    scores (equal ones: the lowest slot; NaN counts as -inf). Kept slots at or
    behind `budget` move into the holes before it, both in ascending order,
    and seq_lens becomes `budget`; pages behind it are free. The pages of a
    sequence must not be shared with another one."""
    if cache.scores is None or cache.slot_pos is None:
        raise ValueError("eviction needs the cache's scores and slot_pos")
    budget, recent = int(budget), int(recent)
    if budget <= 0 or not 0 <= recent <= budget:
        raise ValueError(f"budget must be positive and recent in [0, budget], got {budget} and {recent}")
    dev = cache.k_pages.device
    lib = _C.load()
    with _on(dev):
        ws = _serving_workspace(dev, lib.ts_paged_evict_workspace_size(cache._c, budget))
        rc = lib.ts_paged_evict(cache._c, budget, recent, ws.data_ptr(), ws.numel(), _stream_handle(dev))
    _C.check(rc, "ts_paged_evict")
