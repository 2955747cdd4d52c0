"""The packed-batch cache's bookkeeping and refusals that need no GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

import capi


def test_pool_generation_changes_with_the_free_list():
    lib = capi.lib()
    lib.memopt_pool_generation.restype = ctypes.c_int64
    now = lib.memopt_pool_generation
    lib.memopt_pool_reset()
    seen = [now()]
    for init in ((6, 16, 2, 64), (7, 16, 2, 64), (0, 16, 2, 64), (6, 16, 2, 64)):
        lib.memopt_pool_init(*init)
        assert now() not in seen
        seen.append(now())
    assert lib.memopt_pool_init(6, 16, 2, 64) == 0 and lib.memopt_pool_allocate_block() == 0
    assert lib.memopt_pool_free_block(0) == 0 and now() == seen[-1]  # the same free-list
    lib.memopt_pool_reset()
    assert now() not in seen


class FakePool:
    """memopt_C's pool as far as a cache's constructor uses it, on the CPU."""

    def __init__(self):
        self.kind, self.free, self.generation, self.inits = None, [], 0, 0

    def init_pool(self, num_blocks, block_size, num_heads, head_dim, kv_format="fp16"):
        kind = (num_blocks, block_size, num_heads, head_dim, kv_format)
        if kind != self.kind:
            self.kind, self.free = kind, list(range(num_blocks))
            self.generation += 1

    def pool_format(self):
        if self.kind is None:
            raise RuntimeError("pool not initialized")
        return self.kind[4]

    def get_pool_tensors(self):
        nb, bs, h, d, fmt = self.kind
        k = torch.empty((nb, h, bs, d // 2) if fmt == "int4" else (nb, bs, h, d))
        return k, k

    def pool_generation(self):
        return self.generation

    def free_blocks_count(self):
        return len(self.free)

    def allocate_block(self):
        return self.free.pop(0) if self.free else -1

    def free_block(self, page):
        self.free.append(page)


@pytest.fixture
def pool(monkeypatch):
    import sys

    import memopt  # noqa: F401  its modules keep the real memopt_C

    fake = FakePool()
    monkeypatch.setitem(sys.modules, "memopt_C", fake)
    return fake


def cache_of(num_blocks, heads=2, kv_format="fp16"):
    from memopt import PackedKVCache

    return PackedKVCache(num_blocks, heads, 64, 16, max_seqs=2, max_seq_len=64, kv_format=kv_format, device="cpu")


@pytest.mark.parametrize("kv_format", ["fp16", "int4"])
def test_caches_share_a_pool_without_sharing_pages(pool, kv_format):
    pool.init_pool(20, 16, 2, 64, kv_format)
    a, b = cache_of(12, kv_format=kv_format), cache_of(8, kv_format=kv_format)
    assert pool.generation == 1 and pool.free == []
    rings = [c.table.free_pages[:c.table.free_count()].tolist() for c in (a, b)]
    assert rings == [list(range(12)), list(range(12, 20))]
    assert a.table.free_pages.numel() == 20  # a page is told from another by the pool's number of pages
    for heads, fmt in ((2, kv_format), (4, kv_format), (2, "fp16" if kv_format == "int4" else "int4")):
        with pytest.raises(RuntimeError, match="another PackedKVCache"):
            cache_of(1, heads, fmt)
    assert pool.generation == 1
    a.close()
    a.close()
    assert pool.free == list(range(12))
    with pytest.raises(RuntimeError, match="closed"):
        a.finish([0])
    del b
    assert pool.free == list(range(20))
    c = cache_of(30, kv_format=kv_format)  # nobody lives in the pool: a larger one
    assert pool.generation == 2 and c.table.free_count() == 30


def test_a_cache_notices_that_its_pool_is_gone(pool):
    a = cache_of(5)
    pool.init_pool(6, 16, 2, 64)
    for call in (lambda: a.admit([0], [1]), lambda: a.extend([0]), lambda: a.finish([0]), lambda: a.evict(None, 0.5)):
        with pytest.raises(RuntimeError, match="initialised anew"):
            call()
    a.close()
    assert pool.free == list(range(6))
    pool.free = pool.free[2:]  # somebody holds two
    with pytest.raises(RuntimeError, match="free pages"):
        cache_of(6)


def test_table_pages_are_checked():
    from memopt import DevicePageTable

    table = DevicePageTable(9, 16, 2, 64, device="cpu", pages=[7, 3, 4])
    assert table.free_pages.tolist() == [7, 3, 4] + [-1] * 6 and table.free_count() == 3
    for bad in ([0, 0], [-1], [9]):
        with pytest.raises(ValueError, match="pages"):
            DevicePageTable(9, 16, 2, 64, device="cpu", pages=bad)


P, I, I64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
SOME = 0x1000  # a 16-byte aligned address that no call may touch


def reserve_rows(tables=SOME, lens=SOME, off=SOME, R=4, MB=8, ring=SOME, NB=32, state=SOME, rows=SOME, new=SOME, B=2,
                 BS=16, most=64, replace=0, cu=SOME, slots=SOME, pos=SOME, bt=SOME, bl=SOME, al=SOME):
    return capi.lib().memopt_reserve_rows(P(tables), P(lens), P(off), I(R), I(MB), P(ring), I(NB), P(state), P(rows),
                                          P(new), I(B), I(BS), I64(most), I(replace), P(cu), P(slots), P(pos), P(bt),
                                          P(bl), P(al), P(0))


@pytest.mark.parametrize("change,status", [
    (dict(tables=0), -1), (dict(lens=0), -1), (dict(off=0), -1), (dict(ring=0), -1), (dict(state=0), -1),
    (dict(rows=0), -1), (dict(new=0), -1), (dict(cu=0), -1), (dict(slots=0), -1), (dict(pos=0), -1), (dict(bt=0), -1),
    (dict(bl=0), -1), (dict(al=0), -1), (dict(slots=SOME + 4), -1), (dict(pos=SOME + 8), -1), (dict(most=-1), -1), (dict(B=-1), -1),
    (dict(R=0), -1), (dict(MB=0), -1), (dict(NB=0), -1), (dict(BS=0), -1), (dict(B=8193), -3),
    (dict(R=2 ** 18 + 1), -3), (dict(NB=2 ** 27), -3), (dict(MB=2 ** 27), -3), (dict(most=2 ** 31), -3)])
def test_reserve_rows_refuses(change, status):
    assert reserve_rows(**change) == reserve_rows(**change, replace=1) == status
    assert capi.lib().memopt_last_error().decode().startswith("reserve_rows:")


def test_attention_ex_of_nothing_and_its_refusals():
    def call(q=SOME, out=SOME, seqs=1, tokens=8, zero=1, qs=512):
        return capi.lib().memopt_packed_attention_ex(P(q), I64(qs), P(SOME), I64(256), P(SOME), I64(256), I(0), P(SOME),
                                                     I(seqs), I64(tokens), I(8), I(4), I(2), I(128), I(0), I(1), I(zero),
                                                     P(out), P(0), ctypes.c_size_t(0), P(0))

    assert call(tokens=0) == call(seqs=0, zero=0) == 0
    for zero in (0, 1):
        assert call(q=0, zero=zero) == call(qs=516, zero=zero) == call(out=0, zero=zero) == -1
    assert call(seqs=0, out=0) == -1


def test_layer_says_that_its_scheduler_is_not_used():
    """forward(kv_cache=) obeys the layer's scheduler; a packed batch has none of its scores and says so."""
    import warnings
    from types import SimpleNamespace

    from memopt import DynamicAttention, MemoryScheduler

    cache = SimpleNamespace(prompt=lambda q, *_: q)
    batch, x = SimpleNamespace(whole=True), torch.randn(3, 128)
    with torch.no_grad():
        with pytest.warns(RuntimeWarning, match="scheduler"):
            DynamicAttention(128, 2, scheduler=MemoryScheduler()).forward_packed(x, cache, batch, 3)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            DynamicAttention(128, 2).forward_packed(x, cache, batch, 3)


@pytest.mark.parametrize("MB", [2 ** 31 - 1, 2 ** 31 - 1024])
def test_tables_near_2_to_the_31_are_refused(MB):
    """A lane's index of an entry runs up to 256 past the row's end."""
    assert reserve_rows(MB=MB, BS=1) == -3
    lib = capi.lib()
    assert lib.memopt_truncate_rows(P(SOME), P(SOME), I(4), I(MB), P(SOME), I(32), P(SOME), P(SOME), P(0), I(2), I(1),
                                    P(0)) == -3


def test_an_eviction_that_fails_keeps_the_positions(pool):
    """A row move that ran out of time leaves the lengths shrunk: the positions still go on from the true length."""
    def shrink_and_fail(scores, tables, lens, ratio, sinks):
        lens.copy_(torch.tensor([3, 0], dtype=torch.int32))
        raise RuntimeError("a bounded device wait ran out")

    cache = cache_of(8)
    cache.table.context_lens.copy_(torch.tensor([9, 4], dtype=torch.int32))
    pool.evict_topk_compact = shrink_and_fail
    with pytest.raises(RuntimeError, match="bounded"):
        cache.evict(torch.zeros(2, 2, 9), 0.5)
    assert (cache.table.position_offsets + cache.table.context_lens).tolist() == [9, 4]


def test_packed_batch_of_six_tensors():
    from memopt import PackedBatch

    t = torch.zeros(2, dtype=torch.int32)
    for whole in ((), (True,)):
        batch = PackedBatch(t, t, t, t, t, t, *whole)
        assert batch.whole == bool(whole) and batch.attend_lens is None


def test_caches_made_by_several_threads(pool):
    """Each takes its own pages; one that finds none any more leaves nothing behind."""
    import threading

    plain, taken = pool.allocate_block, []
    pool.init_pool(40, 16, 2, 64)

    def slow():
        import time

        page = plain()
        time.sleep(1e-4)
        return page

    pool.allocate_block = slow
    threads = [threading.Thread(target=lambda: taken.append(cache_of(10))) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(p for c in taken for p in c.table.free_pages[:10].tolist()) == list(range(40))
    taken.clear()
    assert sorted(pool.free) == list(range(40))
    # Somebody else's allocate_block in between.
    pool.allocate_block = lambda: -1 if len(pool.free) == 37 else plain()
    with pytest.raises(RuntimeError, match="free pages"):
        cache_of(10)
    assert sorted(pool.free) == list(range(40))


def test_a_cache_without_pages_is_refused(pool):
    pool.init_pool(5, 16, 2, 64)
    for n in (0, -1):
        with pytest.raises(ValueError, match="num_blocks"):
            cache_of(n)
    assert pool.generation == 1 and len(pool.free) == 5
