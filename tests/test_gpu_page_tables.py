"""Page tables and slot maps on the GPU, against a walk through the requests."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ts():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    import tensorshrink_b200 as m
    return m


class Walk:
    """Pool, table and lengths as lists."""

    def __init__(self, free, n_free, table, lens, page, num_pages):
        self.free, self.n, self.table, self.lens = list(free), n_free, [list(r) for r in table], list(lens)
        self.page, self.num = page, num_pages

    def is_page(self, p):
        return 0 <= p < self.num

    def reserve(self, new, tokens, first=None):
        cap = len(self.table[0]) * self.page
        granted, offsets, slots, pos, seqs = [], [0], [-1] * tokens, [0] * tokens, [-1] * tokens
        wanted = 0
        n_free = self.n
        for b, (n, row) in enumerate(zip(new, self.table)):
            n = max(0, n)
            length, t0 = self.lens[b], offsets[-1]
            offsets.append(t0 + n)
            holes = []
            ok = n > 0 and length >= 0 and length + n <= cap
            if ok:
                holes = [p for p in range(length // self.page, -(-(length + n) // self.page)) if not self.is_page(row[p])]
            wanted += len(holes)
            ok = ok and (not holes or wanted <= n_free)
            if ok:
                for p in holes:
                    self.n -= 1
                    row[p] = self.free[self.n]
            granted.append(n if ok else 0)
            for i in range(n):
                if t0 + i < tokens:
                    seqs[t0 + i] = b
                    if ok:
                        s = length + i
                        slots[t0 + i] = row[s // self.page] * self.page + s % self.page
                        pos[t0 + i] = (first[b] if first is not None else length) + i
        return granted, offsets, slots, pos, seqs

    def release(self, keep):
        for b, (k, row) in enumerate(zip(keep, self.table)):
            if k < 0:
                continue
            for p in range(-(-max(0, min(self.lens[b], k)) // self.page), len(row)):
                if self.is_page(row[p]):
                    self.free[self.n] = row[p]
                    self.n += 1
                    row[p] = -1
            self.lens[b] = min(self.lens[b], k)


def build(ts, lens, page, max_pages, spare, seed):
    """A table in which every sequence has the pages of its tokens, and the walk beside it."""
    rng = random.Random(seed)
    need = [-(-max(0, n) // page) for n in lens]
    total = sum(need) + spare
    order = list(range(total))
    rng.shuffle(order)
    table = [[-1] * max_pages for _ in lens]
    at = 0
    for b, n in enumerate(need):
        table[b][:n] = order[at:at + n]
        at += n
    free = order[at:] + [-7] * at
    i32 = {"dtype": torch.int32, "device": "cuda"}
    pages = torch.zeros(total, 1, page, 16, dtype=torch.bfloat16, device="cuda")
    cache = ts.PagedKVCache(pages, pages.clone(), torch.tensor(table, **i32), torch.tensor(lens, **i32))
    pool = ts.PagePool(torch.tensor(free, **i32), torch.tensor([total - at], **i32))
    return cache, pool, Walk(free, total - at, table, lens, page, total)


def check(got, want, cache, pool, walk):
    if got is not None:
        for g, w, name in zip(got, want, got._fields):
            assert g.tolist() == w, name
    assert cache.page_table.tolist() == walk.table
    assert cache.seq_lens.tolist() == walk.lens
    assert int(pool.n_free) == walk.n and pool.free.tolist()[:walk.n] == walk.free[:walk.n]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("batch,page,longest", [(1, 16, 0), (1, 64, 100), (7, 16, 300), (32, 24, 500), (33, 16, 200), (100, 64, 3000),
                                                (256, 16, 700), (1000, 128, 1000), (5000, 16, 40)])
def test_rounds_of_requests(ts, batch, page, longest):
    rng = random.Random(batch)
    lens = [rng.randint(0, longest) if rng.random() < 0.9 else -1 for _ in range(batch)]
    max_pages = -(-(longest + 400) // page)
    cache, pool, walk = build(ts, lens, page, max_pages, batch * 2 + 40, batch)
    for step in range(3):
        new = [rng.choice((0, 1, 1, 1, rng.randint(1, 2 * page), -3)) for _ in range(batch)]
        first = [rng.randint(0, 10 ** 6) for _ in range(batch)] if step == 1 else None
        tokens = sum(max(0, n) for n in new) + rng.randint(0, 70)
        got = ts.paged_reserve(pool, cache, i32(new), tokens,
                               None if first is None else torch.tensor(first, device="cuda"))
        check(got, walk.reserve(new, tokens, first), cache, pool, walk)
        cache.advance(got.granted)
        walk.lens = [a + b for a, b in zip(walk.lens, got.granted.tolist())]
        keep = [rng.choice((-1, -1, 0, rng.randint(0, longest + 100))) for _ in range(batch)]
        ts.paged_release(pool, cache, i32(keep))
        walk.release(keep)
        check(None, None, cache, pool, walk)


def test_a_long_prompt_and_a_short_buffer(ts):
    cache, pool, walk = build(ts, [0, 5, 0, 70], 16, 3000, 3000, 3)
    new = [40000, 1, 0, 3]
    for tokens in (0, 17, 39999, 40010):
        got = ts.paged_reserve(pool, cache, i32(new), tokens)
        check(got, walk.reserve(new, tokens), cache, pool, walk)    # (the pages of the round before are kept)


def test_a_pool_that_runs_dry(ts):
    # 3 pages: sequence 0 takes two, 1 needs none, 2 more than are left, 3 would fit but comes behind, 4 needs none
    cache, pool, walk = build(ts, [0, 3, 0, 0, 20], 16, 8, 3, 1)
    new = [32, 5, 40, 1, 2]
    got = ts.paged_reserve(pool, cache, i32(new), 80)
    check(got, walk.reserve(new, 80), cache, pool, walk)
    assert got.granted.tolist() == [32, 5, 0, 0, 2] and int(pool.n_free) == 1
    assert got.slots[37:77].eq(-1).all() and got.sequences[37:77].eq(2).all()


def test_the_end_of_the_table(ts):
    cache, pool, walk = build(ts, [30, 31, 32, 0], 16, 2, 9, 2)
    for new in ([2, 2, 1, 33], [0, 1, 0, 32]):
        got = ts.paged_reserve(pool, cache, i32(new), 40)
        check(got, walk.reserve(new, 40), cache, pool, walk)
    assert got.granted.tolist() == [0, 1, 0, 32]


def test_entries_that_name_a_page_are_kept_and_holes_are_filled(ts):
    cache, pool, walk = build(ts, [10, 40], 16, 6, 12, 4)
    for t, b, p, v in ((cache.page_table, 0, 2, 3), (cache.page_table, 1, 2, -1), (cache.page_table, 1, 4, 99)):
        t[b, p] = v                                             # 99 is no page of this pool
        walk.table[b][p] = v
    new = [50, 45]
    got = ts.paged_reserve(pool, cache, i32(new), 95)
    check(got, walk.reserve(new, 95), cache, pool, walk)
    assert int(cache.page_table[0, 2]) == 3
    ts.paged_release(pool, cache, i32([10, -5]))
    walk.release([10, -5])
    check(None, None, cache, pool, walk)


def test_more_pages_than_the_pool_has_room_for(ts):
    i = {"dtype": torch.int32, "device": "cuda"}
    pages = torch.zeros(8, 1, 16, 16, dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3]], **i)      # shared, which is not allowed
    cache = ts.PagedKVCache(pages, pages.clone(), table, torch.tensor([64, 64, 64], **i))
    behind = torch.full((12,), 55, **i)
    pool = ts.PagePool(behind[:8], torch.tensor([0], **i))
    ts.paged_release(pool, cache, torch.zeros(3, **i))
    assert int(pool.n_free) == 8 and behind[8:].eq(55).all()                   # nothing behind the pool is written
    for n in (-5, 100):
        pool.n_free.fill_(n)                                                    # a count that cannot be is bounded
        ts.paged_reserve(pool, cache, i32([1, 1, 1]), 3)


def test_captured_cycle_and_8_bit_cache(ts):
    cache = ts.PagedKVCache8.allocate(4, 1, 16, 64, page_size=16)
    cache.page_table.fill_(-1)
    pool = ts.PagePool.allocate(16)
    new, keep = i32([20, 1, 3, 40]), i32([0, 0, 0, 0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ts.paged_reserve(pool, cache, new, 64)
        cache.advance(got.granted)
    g.replay()
    walk = Walk(range(15, -1, -1), 16, [[-1] * 4 for _ in range(4)], [0] * 4, 16, 16)
    want = walk.reserve([20, 1, 3, 40], 64)
    walk.lens = [20, 1, 3, 40]
    check(got, want, cache, pool, walk)
    assert got.slots[:3].tolist() == [0, 1, 2]                                 # page 0 comes first
    ts.paged_release(pool, cache, keep)
    walk.release([0] * 4)
    check(None, None, cache, pool, walk)


def test_refusals(ts):
    cache, pool, _ = build(ts, [1, 2], 16, 4, 4, 1)
    one = i32([1, 1])
    with pytest.raises(ValueError):
        ts.paged_reserve(pool, cache, one[:1], 2)
    with pytest.raises(ValueError):
        ts.paged_reserve(pool, cache, one.long(), 2)
    with pytest.raises(ValueError):
        ts.paged_reserve(pool, cache, one, -1)
    with pytest.raises(ValueError):
        ts.paged_reserve(pool, cache, one, 2, positions=one)
    with pytest.raises(RuntimeError):
        ts.paged_reserve(pool, cache, one.cpu(), 2)
    with pytest.raises(ValueError):
        ts.paged_release(pool, cache, one.float())
    with pytest.raises(ValueError):
        ts.PagePool(pool.free.long(), pool.n_free)
    with pytest.raises(ValueError):
        ts.PagePool(pool.free, pool.free)
    shared = ts.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table[:1].expand(2, 4), cache.seq_lens)
    with pytest.raises(ValueError):
        ts.paged_reserve(pool, shared, one, 2)
    empty = ts.PagedKVCache(cache.k_pages, cache.v_pages, cache.page_table[:0], cache.seq_lens[:0])
    got = ts.paged_reserve(pool, empty, one[:0], 3)
    assert got.offsets.tolist() == [0] and got.slots.tolist() == [-1] * 3 and got.granted.numel() == 0
    ts.paged_release(pool, empty, one[:0])
