"""The packed-batch cache as a program uses it: several caches in a process,
positions after an eviction, refused batches, arguments of every kind."""
from __future__ import annotations

import ctypes
import gc
import math
import threading

import pytest
import torch

import capi
from test_gpu_packed import DEV, attention_ref, attention_tol, cu_of, half_step, make_qkv, rotary_close, rotary_ref

pytestmark = pytest.mark.gpu


def C():
    import memopt_C

    return memopt_C


def tokens(n, H, KVH, D, seed=0, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, H + 2 * KVH, D, generator=g, device=DEV).to(dtype)
    return tuple(t.contiguous() for t in x.split([H, KVH, KVH], 1))


def cached(cache, row):
    """This row's keys and values in the fp16 pool, [n, KVH, D]."""
    n = int(cache.table.context_lens[row])
    pages = cache.table.block_tables[row, : -(-n // cache.block_size)].long()
    return [c[pages].reshape(-1, cache.num_heads, cache.head_dim)[:n].clone() for c in C().get_pool_tensors()]


def paged_close(out, q, kk, vv, first):
    """Rows of q are the tokens from `first` on of a sequence whose keys and
    values are kk and vv: causal attention, to the paged kernels' tolerance."""
    m, (n, H, D) = kk.shape[0], q.shape
    full = torch.zeros(m, H, D, dtype=torch.float64, device=DEV)
    full[first:first + n] = q.double()
    ref, _ = attention_ref(full, kk.double(), vv.double(), [m], -1, True)
    ref = ref[first:first + n]
    return bool(((out.double() - ref).abs() <= 2e-3 + 1e-2 * ref.abs()).all())


# ---- caches that share the process-wide pool ----------------------------------
def test_two_caches_in_a_process_keep_apart():
    """Two layers, each with its own cache over one pool: neither finds the
    other's keys in its pages."""
    from memopt import PackedKVCache

    H, KVH, D, BS = 4, 2, 64, 16
    gc.collect()
    C().init_pool(60, BS, KVH, D)
    caches = [PackedKVCache(30, KVH, D, BS, max_seqs=3, max_seq_len=320) for _ in range(2)]
    lens = [40, 1, 100]
    kept = [[], []]
    for i, cache in enumerate(caches):
        q, k, v = tokens(sum(lens), H, KVH, D, seed=i)
        cache.prompt(q, k, v, cache.admit([0, 1, 2], lens), max(lens))
        kept[i] += [list(x) for x in zip(k.split(lens), v.split(lens))]
    for step in range(20):
        for i, cache in enumerate(caches):
            q, k, v = tokens(3, H, KVH, D, seed=100 + 2 * step + i)
            out = cache.decode(q, k, v, cache.extend([0, 1, 2]))
            for r in range(3):
                kept[i][r] = [torch.cat([a, b[r:r + 1]]) for a, b in zip(kept[i][r], (k, v))]
                kk, vv = kept[i][r]
                assert paged_close(out[r:r + 1], q[r:r + 1], kk, vv, kk.shape[0] - 1)
    for i, cache in enumerate(caches):
        cache.table.check()
        for r in range(3):
            assert all(torch.equal(a, b) for a, b in zip(cached(cache, r), kept[i][r]))
    used = [set(c.table.block_tables[c.table.block_tables >= 0].tolist()) for c in caches]
    assert not used[0] & used[1]


def test_caches_take_their_pages_from_the_pool():
    """A pool whose pages are taken is neither handed out again nor replaced
    under the cache; a cache that is dropped or closed gives its pages back."""
    from memopt import PackedKVCache, PagedKVCache

    H, KVH, D, BS = 2, 2, 64, 16
    gc.collect()
    C().init_pool(21, BS, KVH, D)
    first = PackedKVCache(21, KVH, D, BS, max_seqs=2, max_seq_len=160)
    assert C().free_blocks_count() == 0
    q, k, v = tokens(30, H, KVH, D)
    first.prompt(q, k, v, first.admit([0], [30]), 30)
    for args in ((21, KVH, D, BS), (1, KVH, D, BS), (40, KVH, D, BS), (21, 4, D, BS), (21, KVH, 128, BS)):
        with pytest.raises(RuntimeError, match="another PackedKVCache"):
            PackedKVCache(*args, max_seqs=2, max_seq_len=160)
    with pytest.raises(RuntimeError, match="another PackedKVCache"):
        PackedKVCache(21, KVH, D, BS, max_seqs=2, max_seq_len=160, kv_format="int4")
    paged = PagedKVCache(21, KVH, D, BS)  # the free-list is the same one
    with pytest.raises(MemoryError):
        paged.table.reserve(paged.add_sequence(), 1)
    kk, vv = cached(first, 0)
    assert torch.equal(kk, k) and torch.equal(vv, v)
    first.close()
    assert C().free_blocks_count() == 21
    with pytest.raises(RuntimeError, match="closed"):
        first.extend([0])
    second = PackedKVCache(10, KVH, D, BS, max_seqs=2, max_seq_len=160)  # a part of the pool
    assert C().free_blocks_count() == 11 and second.table.free_count() == 10
    del second, first
    gc.collect()
    assert C().free_blocks_count() == 21
    # Pages that somebody holds are not the cache's.
    held = [C().allocate_block() for _ in range(5)]
    with pytest.raises(RuntimeError, match="free pages"):
        PackedKVCache(21, KVH, D, BS, max_seqs=2, max_seq_len=160)
    third = PackedKVCache(16, KVH, D, BS, max_seqs=2, max_seq_len=160)
    assert not set(third.table.free_pages[:16].tolist()) & set(held)


def test_a_pool_that_was_replaced_is_noticed():
    from memopt import PackedKVCache

    H, KVH, D, BS = 2, 2, 64, 16
    gc.collect()
    C().init_pool(23, BS, KVH, D)
    cache = PackedKVCache(23, KVH, D, BS, max_seqs=2, max_seq_len=160)
    q, k, v = tokens(30, H, KVH, D)
    batch = cache.admit([0], [30])
    cache.prompt(q, k, v, batch, 30)
    step = cache.extend([0])
    C().init_pool(24, BS, KVH, D)  # as another part of the program may
    assert C().free_blocks_count() == 24
    for call in (lambda: cache.admit([1], [3]), lambda: cache.extend([0]), lambda: cache.finish([0]),
                 lambda: cache.prompt(q, k, v, batch, 30), lambda: cache.decode(q[:1], k[:1], v[:1], step),
                 lambda: cache.evict(torch.rand(2, KVH, 160, device=DEV), 0.5)):
        with pytest.raises(RuntimeError, match="initialised anew"):
            call()
    del cache, call
    gc.collect()
    assert C().free_blocks_count() == 24  # nothing is given back to a pool that it did not come from
    assert not C().get_pool_tensors()[0].any()


# ---- arguments as they come out of a fused projection ----------------------------------
@pytest.mark.parametrize("kv_format,D", [("fp16", 64), ("int4", 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_slices_of_a_projection(kv_format, D, dtype):
    """q, k and v as parts of one tensor, without rotary positions: the same
    results as from copies."""
    from memopt import PackedKVCache

    H, KVH = 4, 2
    results = []
    for copy in (False, True):
        gc.collect()
        cache = PackedKVCache(12, KVH, D, 16, max_seqs=2, max_seq_len=96, kv_format=kv_format)
        g = torch.Generator(device=DEV).manual_seed(7)
        outs = []
        for n in (50, 2, 6):
            parts = torch.randn(n, H + 2 * KVH, D, generator=g, device=DEV).to(dtype).split([H, KVH, KVH], 1)
            if copy:
                parts = [t.contiguous() for t in parts]
            if n == 50:
                outs.append(cache.prompt(*parts, cache.admit([0, 1], [30, 20]), 30))
            else:
                outs.append(cache.decode(*parts, cache.extend([0, 1], n // 2)))
        cache.table.check()
        results.append(outs)
        cache.close()
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ---- positions after an eviction ----------------------------------------------
def evicted(cache, rows, scores, ratio):
    kept, count = cache.evict(scores, ratio)
    return [kept[r, : int(count[r])].tolist() for r in rows]


@pytest.mark.parametrize("sections", [[32], [10, 14, 8]], ids=str)
def test_rotary_positions_after_an_eviction(sections):
    """Kept keys stay turned by the positions that they were written with, so
    the tokens after an eviction go on from the sequence's true length."""
    from memopt import PackedKVCache, RotaryPositions

    H, KVH, D, BS = 4, 2, 64, 16
    rot = RotaryPositions(D, sections=sections)
    cache = PackedKVCache(90, KVH, D, BS, max_seqs=4, max_seq_len=320, rotary=rot)
    lens = {2: 92, 0: 5, 1: 200}
    rows, total = list(lens), sum(lens.values())
    q, k, v = tokens(total, H, KVH, D, seed=1)
    cache.prompt(q, k, v, cache.admit(rows, list(lens.values())), 200)
    true = dict(lens)               # logical length of each row
    at = {r: list(range(n)) for r, n in lens.items()}  # logical positions of the cached tokens
    raw = dict(zip(rows, zip(k.split(list(lens.values())), v.split(list(lens.values())))))

    def turned(x, pos):
        p = torch.tensor(pos, device=DEV, dtype=torch.int32)
        return rotary_ref(x, p.expand(len(sections), -1), rot.inv_freq, rot.sections, False)

    def step(n, seed):
        batch = cache.extend(rows, n)
        q, k, v = tokens(n * len(rows), H, KVH, D, seed=seed)
        out = cache.decode(q, k, v, batch)
        for i, r in enumerate(rows):
            some = slice(i * n, (i + 1) * n)
            pos = list(range(true[r], true[r] + n))
            assert batch.positions[some].tolist() == pos
            raw[r] = tuple(torch.cat([a, b[some]]) for a, b in zip(raw[r], (k, v)))
            at[r], true[r] = at[r] + pos, true[r] + n
            kk, vv = cached(cache, r)
            assert rotary_close(kk, *turned(raw[r][0], at[r])) and torch.equal(vv, raw[r][1])
            assert paged_close(out[some], turned(q[some], pos)[0].half(), kk, vv, kk.shape[0] - n)

    def cut(r, n):  # the last n cached tokens are rejected
        raw[r] = tuple(x[: x.shape[0] - n] for x in raw[r])
        at[r], true[r] = at[r][: len(at[r]) - n], true[r] - n

    step(1, 2)
    for part, ratio in enumerate((0.5, 0.7)):  # twice, so that offsets add up
        g = torch.Generator(device=DEV).manual_seed(part)
        for r, kept in zip(rows, evicted(cache, rows, torch.rand(4, KVH, 256, generator=g, device=DEV), ratio)):
            assert len(kept) < len(at[r]) or len(at[r]) < 7
            raw[r] = tuple(x[kept] for x in raw[r])
            at[r] = [at[r][i] for i in kept]
        for i in range(3):
            step(1, 10 * part + i + 3)
        step(5, 40 + part)
        cache.table.truncate(rows, [len(at[r]) - 4 for r in rows])  # four of five drafts rejected
        for r in rows:
            cut(r, 4)
        step(1, 50 + part)
    # A row that begins anew begins at 0; the others keep their offsets.
    cache.finish([2])
    q, k, v = tokens(30, H, KVH, D, seed=60)
    batch = cache.admit([2], [30])
    assert batch.positions.tolist() == list(range(30))
    cache.prompt(q, k, v, batch, 30)
    true[2], at[2], raw[2] = 30, list(range(30)), (k, v)
    step(2, 61)
    batch = cache.admit([0], [3])  # without finish
    assert batch.positions.tolist() == [0, 1, 2]
    cache.table.check()


def test_positions_after_an_eviction_in_a_graph():
    """A captured step goes on from the true positions after evictions between its replays."""
    from memopt import PackedKVCache

    cache = PackedKVCache(40, 2, 64, 16, max_seqs=3, max_seq_len=160)
    q, k, v = tokens(100, 2, 2, 64)
    cache.prompt(q, k, v, cache.admit([0, 2], [60, 40]), 60)
    rows = torch.tensor([2, 0], dtype=torch.int32, device=DEV)
    cache.extend(rows)  # warm-up
    true = [41, 61]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = cache.extend(rows)
    for ratio in (1.0, 0.5, 0.25):
        if ratio < 1:
            cache.evict(torch.rand(3, 2, 160, device=DEV), ratio)
        for _ in range(3):
            graph.replay()
            assert batch.positions.tolist() == true
            true = [t + 1 for t in true]
    cache.table.check()


def test_a_refused_batch_keeps_the_positions():
    from memopt import PackedKVCache

    cache = PackedKVCache(6, 2, 64, 16, max_seqs=2, max_seq_len=96)
    q, k, v = tokens(64, 2, 2, 64)
    cache.prompt(q, k, v, cache.admit([0], [64]), 64)
    cache.evict(torch.rand(2, 2, 96, device=DEV), 0.5)  # 32 cached, the next token is the 65th
    cache.extend([0], 90)
    with pytest.raises((MemoryError, RuntimeError)):
        cache.table.check()
    cache.extend([0, 0])
    with pytest.raises(RuntimeError, match="twice"):
        cache.table.check()
    assert cache.extend([0, 1], 2).positions.tolist() == [64, 65, 0, 1]
    cache.table.check()


# ---- attention: work that other CTAs have not begun -----------------------------
@pytest.mark.parametrize("H,KVH,split", [(16, 16, False), (2, 1, True)])
def test_attention_with_far_more_ctas_than_items(H, KVH, split):
    """Short sequences in tensors that have room for long ones: nearly all
    CTAs have no item, and every row that has one is computed."""
    D, room = 64, 6000 if split else 40000
    q, k, v = make_qkv([room], H, KVH, D, torch.float16, seed=41)
    need = capi.lib().memopt_packed_attention_workspace_size
    need.restype = capi.SZ
    for lens in ([3], [0, 500, 1, 700], [1] * 30, [2600, 0, 5]):
        cu = cu_of(lens + [0] * (31 - len(lens)))
        asked = need(capi.I(31), capi.I64(room), capi.I(room), capi.I(H), capi.I(KVH), capi.I(D), capi.I(0), capi.I(1))
        assert (asked > 0) == split
        T = sum(lens)
        for causal in (True, False):
            out = torch.full_like(q, float("nan"))
            C().packed_attention(q, k, v, cu, room, -1, causal, out)
            ref, mag = attention_ref(q[:T], k[:T], v[:T], lens, -1, causal)
            assert ((out[:T].double() - ref).abs() <= attention_tol(ref, mag, v, max(lens), torch.float16)).all()
            assert torch.isnan(out[T:].float()).all()


# ---- attention: many small weights --------------------------------------------------
@pytest.mark.parametrize("H,n", [(1, 65536), (64, 12000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_a_sink_and_a_flat_tail(H, n, dtype):
    """One key far above all others, and thousands of others that count only
    together: e^-17.5 = 2^-25.2 each.  All are seen in every row's sum, so the
    result is i w / (1 + i w) for values of 0 (the sink) and 1."""
    D = 64
    q = torch.zeros(n, H, D, device=DEV, dtype=dtype)
    k, v = torch.zeros(n, 1, D, device=DEV, dtype=dtype), torch.ones(n, 1, D, device=DEV, dtype=dtype)
    q[..., 0] = 8.0
    k[0, 0, 0], v[0] = 17.5, 0.0
    out = C().packed_attention(q, k, v, cu_of([n]), n)
    w = torch.arange(n, device=DEV, dtype=torch.float64) * math.exp(-17.5)
    want = (w / (1 + w))[:, None, None]
    # half a step of the result; the weight's own rounding (2 half steps) and the exponential
    # (2^-14, scores below 32); fp16 weights are held as 2^7 of themselves, so that each is off
    # by at most 2^-25 / 2^7 where it is subnormal
    u = half_step(dtype)
    tol = (3 * u + 2.0 ** -14) * want + 1e-7
    if dtype == torch.float16:
        tol = tol + torch.arange(n, device=DEV)[:, None, None] * 2.0 ** -32
    assert ((out.double() - want).abs() <= tol).all()


# ---- refused batches -------------------------------------------------------------
def test_a_refused_admission_changes_nothing():
    """Rows that a refused admit names keep what they held."""
    from memopt import PackedKVCache

    H, KVH, D, BS = 2, 2, 64, 16
    cache = PackedKVCache(10, KVH, D, BS, max_seqs=3, max_seq_len=96)  # six pages a row
    own = sorted(cache.table.free_pages[:10].tolist())
    q, k, v = tokens(50, H, KVH, D, seed=5)
    cache.prompt(q, k, v, cache.admit([0, 2], [30, 20]), 30)
    t = cache.table
    state = lambda: [x.clone() for x in (t.block_tables, t.context_lens, t.free_pages, t.pool_state[:2])]
    before = state()
    calls = [(([0, 1, 2], [96, 60, 1]), MemoryError),            # 6 + 4 + 1 pages of 10
             (([0], [97]), RuntimeError), (([2, 0], [-1, 5], 9), RuntimeError), (([0, 0], [1, 1]), RuntimeError),
             (([0, 3], [1, 1]), RuntimeError), (([0, 2], [4, 5], 8), RuntimeError),
             (([1, 0], [2 ** 31 - 1, 1], 64), RuntimeError)]
    for args, error in calls:
        batch = cache.admit(*args)
        assert (batch.slot_mapping == -1).all() and not batch.cu_seqlens.any()
        assert all(torch.equal(a, b) for a, b in zip(before, state()))
        with pytest.raises(error):
            t.check()
    kk, vv = cached(cache, 0)
    assert torch.equal(kk, k[:30]) and torch.equal(vv, v[:30])
    # What only fits with the rows' own pages is taken: 2 + 2 of them held, 6 free, 10 asked for.
    batch = cache.admit([0, 2], [96, 60])
    t.check()
    assert t.free_count() == 0 and batch.context_lens.tolist() == [96, 60]
    assert sorted(t.block_tables[t.block_tables >= 0].tolist()) == own
    assert batch.cu_seqlens.tolist() == [0, 96, 156] and batch.positions.tolist() == [*range(96), *range(60)]


@pytest.mark.parametrize("rows,high", [(5, 90), (300, 40), (1100, 40)])
def test_admission_gives_the_old_pages_back_first(rows, high):
    """admit is truncate and reserve: the same pages in the same order."""
    from memopt import DevicePageTable

    g = torch.Generator().manual_seed(rows)
    tables = [DevicePageTable(rows * 8, 16, rows + 5, 112) for _ in range(2)]
    for step in range(4):
        pick = torch.randperm(rows + 5, generator=g)[:rows].to(torch.int32).to(DEV)
        new = torch.randint(0, high, (rows,), generator=g, dtype=torch.int32)
        total, new = int(new.sum()) + step, new.to(DEV)
        a = tables[0].replace(pick, new, total)
        tables[1].truncate(pick)
        b = tables[1].reserve(pick, new, total)
        for x, y in zip((a.cu_seqlens, a.slot_mapping, a.positions, a.block_tables, a.context_lens),
                        (b.cu_seqlens, b.slot_mapping, b.positions, b.block_tables, b.context_lens)):
            assert torch.equal(x, y)
        for name in ("block_tables", "context_lens", "free_pages", "pool_state"):
            assert torch.equal(getattr(tables[0], name), getattr(tables[1], name))
        tables[0].check()


def test_a_refused_batch_gives_zeros():
    """No stale memory and no attention without the new token: rows of a
    refused batch, and rows past the last token, are zero."""
    from memopt import DynamicAttention, PackedKVCache

    H, KVH, D, BS = 4, 2, 64, 16
    cache = PackedKVCache(6, KVH, D, BS, max_seqs=2, max_seq_len=96)
    q, k, v = tokens(200, H, KVH, D, seed=6)
    for _ in range(3):  # memory that the allocator hands out again
        stale = torch.full_like(q, 9.0).contiguous()
        del stale
        assert not cache.prompt(q, k, v, cache.admit([0], [200]), 200).any()
    with pytest.raises((MemoryError, RuntimeError)):
        cache.table.check()
    out = cache.prompt(q[:60], k[:60], v[:60], cache.admit([0], [33], 60), 33)
    assert not out[33:].any() and out[:33].any(-1).all()
    for n in (1, 3, 80):
        batch = cache.extend([0, 0], n)
        out = cache.decode(q[:2 * n], k[:2 * n], v[:2 * n], batch)
        assert out.shape[0] == 2 * n and not out.any()
        with pytest.raises(RuntimeError):
            cache.table.check()
    batch = cache.extend([0, 1])
    assert cache.decode(q[:2], k[:2], v[:2], batch).any(-1).all()
    assert batch.attend_lens.tolist() == batch.context_lens.tolist() == [34, 1]
    layer = DynamicAttention(H * D, H).half().to(DEV)
    two = PackedKVCache(6, H, D, BS, max_seqs=2, max_seq_len=96) if cache.close() is None else None
    with torch.no_grad():
        y = layer.forward_packed(torch.randn(200, H * D, device=DEV).half(), two, two.admit([0], [200]), 200)
    assert not y.any()


@pytest.mark.parametrize("H,KVH,D,lens,tail", [(4, 2, 64, [70, 0, 3], 500), (2, 1, 128, [2600], 1), (2, 1, 64, [], 2600),
                                               (20, 20, 128, [1500, 900], 1300), (8, 2, 64, [0, 0], 77), (3, 3, 64, [1], 0)])
def test_rows_behind_the_last_sequence_become_zero(H, KVH, D, lens, tail):
    """zero_rest, in the whole, the two-tile and the split form; other rows as without it."""
    T = sum(lens) + tail
    q, k, v = make_qkv([T], H, KVH, D, torch.bfloat16, seed=8)
    for causal in (True, False):
        plain, out = (torch.full_like(q, 3.0) for _ in range(2))
        C().packed_attention(q, k, v, cu_of(lens), T, -1, causal, plain)
        C().packed_attention(q, k, v, cu_of(lens), T, -1, causal, out, zero_rest=True)
        assert torch.equal(out[:T - tail], plain[:T - tail]) and not out[T - tail:].any()
        assert (plain[T - tail:] == 3.0).all()
    for cu in ([5, 2, 1], [0, -7], [0, 2 ** 31 - 1]):  # values that no table builds: inside the tensors all the same
        C().packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV), T, zero_rest=True)
    torch.cuda.synchronize()


# ---- gradients ---------------------------------------------------------------------
@pytest.mark.parametrize("rotary", [False, True])
def test_inputs_that_require_a_gradient_are_refused(rotary):
    """None is cut off in silence, and a refused call writes nothing."""
    from memopt import DynamicAttention, PackedKVCache, RotaryPositions

    H, D = 2, 64
    cache = PackedKVCache(7, H, D, 16, max_seqs=1, max_seq_len=96, rotary=RotaryPositions(D) if rotary else None)
    layer = DynamicAttention(H * D, H).half().to(DEV)
    x = torch.randn(20, H * D, device=DEV).half().requires_grad_(True)
    q, k, v = tokens(20, H, H, D)
    for pool in C().get_pool_tensors():
        pool.fill_(7.0)
    batch = cache.admit([0], [20])
    with pytest.raises(RuntimeError, match="no gradient"):
        layer.forward_packed(x, cache, batch, 20)
    for i in range(3):
        args = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        with pytest.raises(RuntimeError, match="no gradient"):
            cache.prompt(*args, batch, 20)
    assert all((p == 7.0).all() for p in C().get_pool_tensors())
    with torch.no_grad():
        assert not layer.forward_packed(x, cache, batch, 20).requires_grad
    step = cache.extend([0])
    before = [p.clone() for p in C().get_pool_tensors()]
    with pytest.raises(RuntimeError, match="no gradient"):
        layer.forward_packed(x[:1], cache, step)
    for i in range(3):
        args = [t[:1].clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        with pytest.raises(RuntimeError, match="no gradient"):
            cache.decode(*args, step)
    assert all(torch.equal(a, b) for a, b in zip(before, C().get_pool_tensors()))
    # The layer's own projections: out_proj trains, and the caller is told that the others do not.
    with pytest.warns(RuntimeWarning, match="no gradient"):
        y = layer.forward_packed(x[:1].detach(), cache, step)
    y.float().sum().backward()
    assert layer.out_proj.weight.grad is not None and layer.q_proj.weight.grad is None


# ---- page tables: calls at once, arguments of every kind -----------------------------
def test_page_calls_of_two_host_threads():
    """Batches of different sizes from two threads: neither lowers the shared
    memory that the other's launch asks for."""
    lib, bad = capi.lib(), []

    def work(B, calls):
        with torch.cuda.stream(torch.cuda.Stream()):
            i32 = dict(dtype=torch.int32, device=DEV)
            tables, lens = torch.full((B, 1), -1, **i32), torch.zeros(B, **i32)
            ring, state = torch.arange(B, **i32), torch.tensor([0, B, 0, 0], **i32)
            rows, one = torch.arange(B, **i32), torch.ones(B, **i32)
            out = [torch.empty(B + 4, **i32) for _ in range(3)] + [torch.empty(B, 1, **i32), torch.empty(B, **i32)]
            p, s = capi.ptr, capi.stream()
            I, I64 = ctypes.c_int, ctypes.c_int64
            for _ in range(calls):
                st = lib.memopt_reserve_slots(p(tables), p(lens), I(B), I(1), p(ring), I(B), p(state), p(rows), p(one),
                                              I(B), I(16), I64(B), *(p(t) for t in out), s)
                st2 = lib.memopt_truncate_rows(p(tables), p(lens), I(B), I(1), p(ring), I(B), p(state), p(rows),
                                               capi.P(0), I(B), I(16), s)
                if st or st2:
                    bad.append((B, st, st2))
                    return
            torch.cuda.current_stream().synchronize()
            if state.tolist()[1:] != [B, 0, 0]:
                bad.append((B, state.tolist()))

    threads = [threading.Thread(target=work, args=a) for a in ((8192, 4000), (4000, 4000), (6000, 4000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_page_tensors_that_overlap_are_refused():
    """What a call updates must not be what it reads: each pair is refused."""
    i32 = dict(dtype=torch.int32, device=DEV)
    names = ("block_tables", "context_lens", "free_pages", "pool_state", "rows", "lens")

    def args():
        return {"block_tables": torch.full((4, 4), -1, **i32), "context_lens": torch.zeros(4, **i32),
                "free_pages": torch.arange(8, **i32), "pool_state": torch.tensor([0, 8, 0, 0], **i32),
                "rows": torch.arange(4, **i32), "lens": torch.zeros(4, **i32)}

    def call(a):
        C().reserve_slots(*(a[n] for n in names), 16, 4)
        C().truncate_rows(*(a[n] for n in names), 16)

    call(args())
    a = args()
    a["lens"] = a["rows"] = torch.zeros(4, **i32)  # both are only read (and refused on the device: a row twice)
    call(a)
    for i, one in enumerate(names):
        for two in names[i + 1:]:
            if (one, two) == ("rows", "lens"):
                continue
            buf, a = torch.zeros(40, **i32), args()
            a[one] = buf[: a[one].numel()].view(a[one].shape)
            a[two] = buf[a[one].numel() - 1:][: a[two].numel()].view(a[two].shape)  # one value in common
            for f, n in ((C().reserve_slots, (16, 4)), (C().truncate_rows, (16,))):
                with pytest.raises(RuntimeError, match="overlap"):
                    f(*(a[x] for x in names), *n)
            assert not buf.any()


def test_lists_do_not_wait_for_the_stream():
    """Rows and lengths given as Python numbers or as tensors of the host."""
    from memopt import PackedKVCache

    cache = PackedKVCache(20, 2, 64, 16, max_seqs=3, max_seq_len=96)
    long = torch.tensor([3, 4])
    cache.admit([0, 1], [3, 4])  # warm-up
    cache.table.truncate(long - 3, long - 3)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(1_000_000_000)  # half a second
    batches = [cache.admit([0, 1], [3, 4])] + [cache.extend([i % 3, (i + 1) % 3], 1 + i % 2) for i in range(6)]
    cache.table.truncate([0, 2], [2, 1])
    cache.table.reserve(long - 3, long, 7)
    cache.finish([1])
    done.record()
    assert not done.query()
    torch.cuda.synchronize()
    cache.table.check()
    assert batches[0].positions.tolist() == [0, 1, 2, 0, 1, 2, 3]
    assert cache.table.context_lens.tolist() == [5, 0, 1]


def test_numbers_of_the_host_cannot_be_captured():
    """A graph would replay what the list held once: refused, tensors of the GPU are the way."""
    from memopt import DevicePageTable

    table = DevicePageTable(20, 16, 3, 96)
    rows, one = (torch.arange(2, dtype=torch.int32, device=DEV) + i for i in (0, 1))
    host, graph = rows.long().cpu(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: table.reserve([0, 1], one, 3), lambda: table.reserve(rows, [1, 2]),
                     lambda: table.truncate([0]), lambda: table.reserve(host, one, 3)):
            with pytest.raises(RuntimeError, match="tensors of the GPU"):
                call()
        table.reserve(rows, one.long(), 3)
    graph.replay()
    assert table.context_lens.tolist() == [1, 2, 0]
    table.check()


def test_whole_numbers_past_32_bits_are_refused():
    """They are not cut to 32 bits, which would make another row of them."""
    from memopt import DevicePageTable

    table = DevicePageTable(20, 16, 3, 96)
    far = 2 ** 32
    for dev in (DEV, "cpu"):
        t = lambda *values: torch.tensor(values, device=dev)
        for call in (lambda: table.reserve(t(far), t(1), 1), lambda: table.reserve(t(0), t(far + 1), 9),
                     lambda: table.reserve(t(0), t(-far + 1), 9), lambda: table.truncate(t(far + 1)),
                     lambda: table.truncate(t(0), t(far))):
            call()
            with pytest.raises(RuntimeError):
                table.check()
            assert table.context_lens.tolist() == [0, 0, 0] and table.free_count() == 20
    for bad in (torch.tensor([1.0], device=DEV), torch.tensor([1.5]), torch.tensor([True], device=DEV)):
        with pytest.raises(TypeError, match="whole numbers"):
            table.reserve(bad, [1])
        with pytest.raises(TypeError, match="whole numbers"):
            table.truncate([0], bad)
    table.reserve(torch.tensor([2], dtype=torch.uint8, device=DEV), torch.tensor([3], dtype=torch.int16), 3)
    table.check()
    assert table.context_lens.tolist() == [0, 0, 3]


def test_page_counts_of_very_large_blocks():
    """Lengths and block sizes whose sum passes 2^31 still count their pages."""
    i32 = dict(dtype=torch.int32, device=DEV)
    for bs in (1_500_000_000, 1 << 30):
        tables, lens, ring = torch.zeros(1, 1, **i32), torch.tensor([1_000_000_000], **i32), torch.full((1,), -1, **i32)
        state, row = torch.tensor([0, 0, 0, 0], **i32), torch.zeros(1, **i32)
        C().truncate_rows(tables, lens, ring, state, row, torch.tensor([5], **i32), bs)
        assert state.tolist() == [0, 0, 0, 0] and lens.tolist() == [5] and tables.tolist() == [[0]]
        cu, slots, pos, bt, bl = C().reserve_slots(tables, lens, ring, state, row, torch.tensor([3], **i32), bs, 3)
        assert slots.tolist() == pos.tolist() == [5, 6, 7] and bl.tolist() == [8]
        C().truncate_rows(tables, lens, ring, state, row, None, bs)
        assert state.tolist() == [0, 1, 0, 0] and ring.tolist() == [0] and tables.tolist() == [[-1]]


def test_pinned_numbers_may_change_after_the_call():
    """The copy is taken within the call, whatever memory the numbers lie in."""
    from memopt import DevicePageTable

    for dtype in (torch.int32, torch.int64, torch.int16):
        table = DevicePageTable(20, 16, 3, 96)
        rows, lens = (torch.tensor(x, dtype=dtype).pin_memory() for x in ([0, 2], [5, 20]))
        table.reserve(rows, lens, 25)  # warm-up
        table.truncate(rows)
        torch.cuda.synchronize()
        torch.cuda._sleep(300_000_000)
        batch = table.reserve(rows, lens, 25)
        rows.fill_(1)
        lens.fill_(3)
        assert batch.context_lens.tolist() == [5, 20] and batch.rows.tolist() == [0, 2]
        table.check()
        assert table.context_lens.tolist() == [5, 0, 20]


# ---- together, in graphs and on two streams -----------------------------------------------
@pytest.mark.parametrize("kv_format", ["fp16", "int4"])
def test_admission_prompt_and_steps_in_a_graph(kv_format):
    """Captured once and replayed with other rows, lengths and inputs, refused
    batches among them: what the same calls give one by one."""
    from memopt import PackedKVCache, RotaryPositions

    H, KVH, D, T = 4, 2, 64, 120
    gc.collect()
    C().init_pool(40, 16, KVH, D, kv_format=kv_format)
    rot = RotaryPositions(D, sections=[16, 16])
    one, two = (PackedKVCache(20, KVH, D, 16, max_seqs=4, max_seq_len=112, kv_format=kv_format, rotary=rot) for _ in range(2))
    q, k, v = tokens(T, H, KVH, D, seed=1)
    rows, lens = torch.tensor([0, 2], dtype=torch.int32, device=DEV), torch.tensor([60, 50], dtype=torch.int32, device=DEV)

    def step(cache):
        out = [cache.prompt(q, k, v, cache.admit(rows, lens, T), T)]
        out += [cache.decode(q[:2 * n], k[:2 * n], v[:2 * n], cache.extend(rows, n)) for n in (1, 3)]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(one)  # warm-up: the paged attention's workspace of this stream
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(one)
        for i, (r, n) in enumerate((((0, 2), (60, 50)), ((1, 3), (1, 112)), ((1, 0), (100, 20)), ((2, 2), (5, 5)),
                                    ((2, 3), (0, 70)), ((0, 1), (90, 40)))):
            rows.copy_(torch.tensor(r))
            lens.copy_(torch.tensor(n))
            for x, y in zip((q, k, v), tokens(T, H, KVH, D, seed=10 + i)):
                x.copy_(y)
            if i == 0:
                step(two)  # the warm-up's turn, so that both tables have the same past
            graph.replay()
            want = step(two)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            for name in ("context_lens", "position_offsets"):
                assert torch.equal(getattr(one.table, name), getattr(two.table, name))
            assert torch.equal(one.table.pool_state, two.table.pool_state)
            if r == (2, 2):
                assert not any(x.any() for x in got)
    side.synchronize()
    torch.cuda.current_stream().wait_stream(side)


def test_two_caches_on_two_streams():
    """Prompts and steps of two layers at once: as one after the other."""
    from memopt import PackedKVCache, RotaryPositions

    H, KVH, D, lens = 8, 2, 128, [300, 1, 77]

    def layers():
        gc.collect()
        C().init_pool(120, 16, KVH, D)
        return [PackedKVCache(60, KVH, D, 16, max_seqs=3, max_seq_len=320, rotary=RotaryPositions(D)) for _ in range(2)]

    data = [[tokens(n, H, KVH, D, seed=5 * i + j) for j, n in enumerate((378, 3, 3, 6))] for i in range(2)]

    def run(cache, i):
        out = [cache.prompt(*data[i][0], cache.admit([0, 1, 2], lens), 300)]
        for x in data[i][1:]:
            out.append(cache.decode(*x, cache.extend([0, 1, 2], x[0].shape[0] // 3)))
        return out

    caches = layers()
    want = [run(c, i) for i, c in enumerate(caches)]
    torch.cuda.synchronize()
    del caches
    caches, streams, got = layers(), [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(run(caches[i], i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
        caches[i].table.check()


def test_position_offsets_that_overlap_are_refused():
    i32 = dict(dtype=torch.int32, device=DEV)
    names = ("block_tables", "context_lens", "position_offsets", "free_pages", "pool_state", "rows", "lens")
    for other in names:
        if other == "position_offsets":
            continue
        a = {"block_tables": torch.full((4, 4), -1, **i32), "context_lens": torch.zeros(4, **i32),
             "position_offsets": torch.zeros(4, **i32), "free_pages": torch.arange(8, **i32),
             "pool_state": torch.tensor([0, 8, 0, 0], **i32), "rows": torch.arange(4, **i32),
             "lens": torch.zeros(4, **i32)}
        a["position_offsets"] = a[other].view(-1)[:4]
        with pytest.raises(RuntimeError, match="overlap"):
            C().reserve_rows(*(a[n] for n in names), 16, 4)
    with pytest.raises(RuntimeError, match="position_offsets"):
        a["position_offsets"] = torch.zeros(3, **i32)
        C().reserve_rows(*(a[n] for n in names), 16, 4)
