"""Paged caches without a GPU: the page pool's bookkeeping against a plain model of it, and
the refusals of the bindings and of the C entry points."""

import ctypes
import random

import pytest
import torch

import g4b200 as g4




def _apply(store, groups, page_rows):
    for src, dst, rows in groups:
        assert not set(dst) & set(src) and len(set(dst)) == len(dst)
        new = {(d, r): store.get((s, r)) for s, d, n in zip(src, dst, rows) for r in range(n)}
        store.update(new)


@pytest.mark.parametrize("seed", range(8))
def test_pool_random_walk_keeps_every_sequence(seed):
    rng = random.Random(seed)
    n_pages, page_rows = 40, 8
    pool = g4.PagePool(n_pages, page_rows)
    store, want, low, counter = {}, {}, {}, 0
    for _ in range(400):
        op = rng.choice(["add", "extend", "extend", "extend", "fork", "free", "trim", "compact"])
        if op == "add" and len(want) < 8:
            s = pool.add()
            assert s not in want
            want[s], low[s] = [], 0
        elif op == "extend" and want:
            s = rng.choice(list(want))
            before = (pool.table(s), pool.free_pages)
            n = rng.randint(0, 20)
            try:
                pool.extend(s, n)
            except g4.G4Error as e:
                assert e.code == 6 and (pool.table(s), pool.free_pages) == before
                continue
            _apply(store, pool.take_copies(), page_rows)
            table, rows = pool.table(s)
            for r in range(len(want[s]), len(want[s]) + n):
                counter += 1
                store[(table[r // page_rows], r % page_rows)] = counter
                want[s].append(counter)
            assert rows == len(want[s])
        elif op == "fork" and want and len(want) < 8:
            s = rng.choice(list(want))
            free = pool.free_pages
            c = pool.fork(s)
            assert c not in want and pool.free_pages == free
            want[c], low[c] = list(want[s]), low[s]
        elif op == "free" and want:
            s = rng.choice(list(want))
            pool.free(s)
            del want[s], low[s]
        elif op == "trim" and want:
            s = rng.choice(list(want))
            r = rng.randint(0, len(want[s]))
            pool.trim(s, r)
            low[s] = max(low[s], r // page_rows * page_rows)
        elif op == "compact":
            src, dst, pm = ((ctypes.c_int32 * n_pages)() for _ in range(3))
            n = ctypes.c_int32()
            assert g4.LIB.g4_page_pool_compact(pool.handle, src, dst, pm, ctypes.byref(n)) == 0
            used = n_pages - pool.free_pages
            assert all(a >= used > b for a, b in zip(src[:n.value], dst[:n.value]))
            for a, b in zip(src[:n.value], dst[:n.value]):
                assert pm[a] == b
                store.update({(b, r): store.get((a, r)) for r in range(page_rows)})
        held = set()
        for s, rows in want.items():
            table, n = pool.table(s)
            assert n == len(rows) and len(table) == (n + page_rows - 1) // page_rows
            for r in range(low[s], n):
                assert store[(table[r // page_rows], r % page_rows)] == rows[r]
            assert all(p == -1 for p in table[:low[s] // page_rows])
            held |= {p for p in table if p >= 0}
        assert pool.free_pages == n_pages - len(held)
    for s in list(want):
        pool.free(s)
    assert pool.free_pages == n_pages


def test_pool_shares_whole_pages_and_copies_the_last():
    pool = g4.PagePool(16, 8)
    a = pool.add()
    pool.extend(a, 20)
    b, c = pool.fork(a), pool.fork(a)
    assert pool.free_pages == 13
    for s in (a, b, c):
        pool.extend(s, 1)
    ta, tb, tc = (pool.table(s)[0] for s in (a, b, c))
    assert ta[:2] == tb[:2] == tc[:2] and len({ta[2], tb[2], tc[2]}) == 3
    assert pool.take_copies() == [([2, 2], [3, 4], [4, 4])]  # the last one keeps the page
    assert pool.take_copies() == []


def test_pool_copies_that_depend_run_in_turn():
    pool = g4.PagePool(4, 8)
    a = pool.add()
    pool.extend(a, 4)
    b = pool.fork(a)
    pool.extend(b, 1)          # page 0 -> 1
    c = pool.fork(b)
    pool.extend(c, 1)          # page 1 -> 2: reads what the first copy fills
    assert pool.take_copies() == [([0], [1], [4]), ([1], [2], [5])]


def test_pool_fork_of_whole_pages_copies_nothing():
    pool = g4.PagePool(8, 8)
    a = pool.add()
    pool.extend(a, 16)
    b = pool.fork(a)
    pool.extend(b, 3)
    assert pool.take_copies() == [] and pool.table(b)[0][:2] == pool.table(a)[0]


def test_pool_refusals():
    for args in ((0, 8), (4, 0), (4, 12), (4, -8), (4, 65544), (-1, 8), (2 ** 24 + 1, 8), (2 ** 31 - 1, 8)):
        with pytest.raises(g4.G4Error):
            g4.PagePool(*args)
    pool = g4.PagePool(4, 8)
    s = pool.add()
    for call in (lambda: pool.extend(s, -1), lambda: pool.extend(s + 1, 1), lambda: pool.extend(-1, 1),
                 lambda: pool.fork(7), lambda: pool.free(7), lambda: pool.trim(s, 1), lambda: pool.trim(s, -1),
                 lambda: pool.table(9)):
        with pytest.raises(g4.G4Error) as e:
            call()
        assert e.value.code == 1
    for n in (33, 2**31 - 1):
        with pytest.raises(g4.G4Error) as e:
            pool.extend(s, n)
        assert e.value.code == 6
    pool.extend(s, 32)
    assert pool.free_pages == 0
    with pytest.raises(g4.G4Error) as e:
        pool.extend(s, 1)
    assert e.value.code == 6 and pool.table(s)[1] == 32
    pool.free(s)
    with pytest.raises(g4.G4Error):
        pool.free(s)
    # compaction while copies wait
    s = pool.add()
    pool.extend(s, 4)
    c = pool.fork(s)
    pool.extend(c, 1)
    buf = [(ctypes.c_int32 * 4)() for _ in range(3)]
    n = ctypes.c_int32()
    assert g4.LIB.g4_page_pool_compact(pool.handle, *buf, ctypes.byref(n)) == 1
    assert g4.LIB.g4_page_pool_add(None, ctypes.byref(n)) == 1
    assert g4.LIB.g4_page_pool_last_error(None) == b"null page pool"
    assert g4.LIB.g4_page_pool_table(pool.handle, c, (ctypes.c_int32 * 1)(), -1, ctypes.byref(n)) == 1


def test_table_longer_than_the_pool():
    """A windowed sequence gives pages back and goes on: its table outgrows the pool."""
    pool = g4.PagePool(4, 8)
    s = pool.add()
    for i in range(10):
        pool.extend(s, 8)
        pool.trim(s, 8 * i)
    table, rows = pool.table(s)
    assert rows == 80 and table[:9] == [-1] * 9 and table[9] >= 0


def test_c_entry_points_refuse_a_null_context():
    null = ctypes.c_void_p(0)
    cd, bd = g4.paged._CacheDesc(), g4.paged._BatchDesc()
    assert g4.LIB.g4_paged_attention(null, None, 0, 0, 1, cd, bd, 1.0, 0, None, 0, 0) == 1
    assert g4.LIB.g4_paged_store_qkv(null, None, 0, 0, 1, None, 0, 0, None, 0, 0, None, None, None, None, 1, cd, bd,
                                     None, 0, 0) == 1
    assert g4.LIB.g4_paged_copy(null, cd, 1, None, None, None, 0) == 1
    assert g4.LIB.g4_paged_compact(null, cd, 1, None, None, 0, None, 0, 0, 0, None) == 1


def test_descriptors_refuse_wrong_tensors():
    z = torch.zeros(2, 8, 1, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        g4.PagedCache(z, z)
    with pytest.raises(TypeError, match="torch"):
        g4.PagedCache([1], z)
    with pytest.raises(ValueError, match="CUDA"):
        g4.PagedBatch(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                      torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="no layers"):
        g4.PagedCaches([])


def test_a_batch_gives_each_call_its_own_descriptor(monkeypatch):
    """Two threads with differently padded q over one batch: neither sees the other's token count."""
    monkeypatch.setattr(g4.paged, "_cuda", lambda name, t, *_: t)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    batch = g4.PagedBatch(i32(3, 5), i32(4), i32(3))
    a, b = batch.desc(7), batch.desc(900)
    assert (a.n_tokens, b.n_tokens) == (7, 900)
    for d in (a, b):
        assert (d.max_pages, d.n_seqs, d.table_stride, d.kv_len) == (5, 3, 5, batch.kv_len.data_ptr())


def test_pool_refuses_numbers_past_32_bits():
    """Not their low 32 bits in their place."""
    for args in ((2 ** 32 + 4, 8), (4, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="32 bits"):
            g4.PagePool(*args)
    pool = g4.PagePool(4, 8)
    s = pool.add()
    pool.extend(s, 8)
    big = 2 ** 32
    for call in (lambda: pool.extend(s, big + 1), lambda: pool.extend(big + s, 1), lambda: pool.fork(big + s),
                 lambda: pool.trim(s, big + 8), lambda: pool.trim(big + s, 8), lambda: pool.free(big + s),
                 lambda: pool.table(big + s), lambda: pool.extend(s, -big)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    with pytest.raises(TypeError):
        pool.extend(s, 1.5)
    assert pool.table(s) == ([0], 8) and pool.free_pages == 3


def _no_gpu(monkeypatch):
    """PagePool's calls of the GPU side, replaced: uploads and checks let everything pass."""
    monkeypatch.setattr(g4.paged, "_upload", lambda ctx, x: list(x))
    monkeypatch.setattr(g4.PagePool, "_check_caches", lambda *a: None)
    monkeypatch.setattr(g4.paged, "_check_tables", lambda *a: None)
    monkeypatch.setattr(g4.paged, "_same_device", lambda *a, **kw: None)


def test_copies_that_were_not_launched_still_wait(monkeypatch):
    """A launch that fails loses no copy: a forked sequence would attend over a page that was never
    filled."""
    _no_gpu(monkeypatch)
    pool = g4.PagePool(8, 8)
    a = pool.add()
    pool.extend(a, 4)
    b = pool.fork(a)
    pool.extend(b, 1)
    c = pool.fork(b)
    pool.extend(c, 1)  # reads what the first copy fills: a group of its own
    ran, fail_at = [], 1

    def copy(ctx, caches, *group):
        if len(ran) == fail_at:
            raise g4.G4Error("g4_paged_copy", 2, "a launch that fails")
        ran.append(group)

    monkeypatch.setattr(g4.paged, "paged_copy", copy)
    with pytest.raises(g4.G4Error, match="fails"):
        pool.run_copies(None, None)
    assert ran == [([0], [1], [4])]
    with pytest.raises(g4.G4Error, match="wait"):
        pool.compact(None, None, None)
    d = pool.fork(a)
    pool.extend(d, 1)
    fail_at = -1
    pool.run_copies(None, None)
    assert ran == [([0], [1], [4]), ([1], [2], [5]), ([0], [3], [4])]
    pool.run_copies(None, None)
    assert len(ran) == 3 and pool.take_copies() == []


def test_a_compaction_that_was_not_launched_is_taken_up_again(monkeypatch):
    """The pool has renumbered its pages when the launch fails: nothing goes by the new numbers until
    the pages are where they say."""
    _no_gpu(monkeypatch)
    pool = g4.PagePool(8, 8)
    a, b = pool.add(), pool.add()
    pool.extend(a, 16)
    pool.extend(b, 24)
    pool.free(a)
    calls = []

    def compact(ctx, caches, src, dst, tables, page_map):
        calls.append((src, dst, page_map))
        if len(calls) == 1:
            raise g4.G4Error("g4_paged_compact", 2, "a launch that fails")

    monkeypatch.setattr(g4.paged, "paged_compact", compact)
    with pytest.raises(g4.G4Error, match="fails"):
        pool.compact(None, None, None)
    for call in (lambda: pool.table(b), lambda: pool.batch(None, [b], [1]), lambda: pool.run_copies(None, None),
                 pool.take_copies):
        with pytest.raises(g4.G4Error, match="compact again"):
            call()
    pool.extend(pool.fork(b), 1)
    assert pool.compact(None, None, None) == 2
    assert calls[1] == calls[0] == ([3, 4], [0, 1], [0, 1, 2, 0, 1, 5, 6, 7])
    assert pool.table(b)[0] == [2, 0, 1] and pool.take_copies() == []
    assert pool.compact(None, None, None) == 0


def test_a_table_takes_the_room_of_its_sequence():
    """Not of the pool: a server asks for each sequence's table at every step."""
    import tracemalloc

    pool = g4.PagePool(2 ** 20, 8)
    seqs = [pool.add() for _ in range(4)]
    for s in seqs[1:]:
        pool.extend(s, 8 * 25 - 3)
    tracemalloc.start()
    got = [pool.table(s) for s in seqs]
    peak = tracemalloc.get_traced_memory()[1]
    tracemalloc.stop()
    assert got[0] == ([], 0) and all(len(t) == 25 and r == 197 for t, r in got[1:])
    assert [t[0] for t, _ in got[1:]] == [0, 25, 50]
    assert peak < 2 ** 16
    rows = ctypes.c_int32()
    assert g4.LIB.g4_page_pool_table(pool.handle, seqs[1], None, 0, ctypes.byref(rows)) == 6 and rows.value == 197
    assert g4.LIB.g4_page_pool_table(pool.handle, 99, None, 0, ctypes.byref(rows)) == 1
