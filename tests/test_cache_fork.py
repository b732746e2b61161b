"""Sequences that share their first tokens, and sequences that go back: the cache's bookkeeping."""
import random

import pytest
import torch

from cretif_b200.cache import BlockPool, CacheError, CacheFull, KVRequest, SequenceCache, StateRequest


def test_blocks_with_several_holders():
    pool = BlockPool(4)
    a = pool.take(2)
    pool.share(a)
    pool.share([a[0]])
    assert pool.holders(a[0]) == 3 and pool.holders(a[1]) == 2 and pool.shared_count == 3
    pool.give_back(a)
    assert pool.free_count == 2 and pool.held_count == 2 and pool.shared_count == 1
    pool.give_back([a[1]])
    assert pool.free_count == 3 and pool.take(1) == [a[1]]
    pool.give_back([a[0]])
    pool.give_back([a[0]])
    with pytest.raises(CacheError, match="not held"):
        pool.give_back([a[0]])
    with pytest.raises(CacheError, match="shared"):
        pool.share([a[0]])
    with pytest.raises(CacheError, match="shared"):
        pool.share([9])
    assert pool.shared_count == 0
    pool.check()


def make(max_tokens=1024, window=False, state=False, pool=0):
    reqs = {0: KVRequest(2, 16), 1: KVRequest(2, 16), 2: KVRequest(1, 32, shared_values=True)}
    if window:
        reqs[3] = KVRequest(1, 16, window=100, pool=pool)
    if state:
        reqs[4] = StateRequest((3,))
    return SequenceCache(reqs, max_tokens, torch.float32, "cpu", max_slots=8)


def write(cache, slot, n, value):
    """``n`` more tokens whose keys and values are ``value`` + position."""
    start = cache.length(slot)
    cache.begin_step([(slot, n)])
    for g in cache._kv_groups:
        if g.tokens_per_entry > 1:
            continue
        for pos in range(start, start + n):
            blk = int(g.table_host[slot, pos // 64])
            g.k[:, blk, :, pos % 64] = value + pos
            if g.v is not g.k:
                g.v[:, blk, :, pos % 64] = -(value + pos)
    cache.end_step([(slot, n)])


def read(cache, slot):
    out = []
    for g in cache._kv_groups:
        lo = max(0, cache.length(slot) - g.request.window + 1) if g.request.window else 0
        out.append([float(g.k[0, int(g.table_host[slot, p // 64]), 0, p % 64, 0]) for p in range(lo, cache.length(slot))])
    return out


@pytest.mark.parametrize("length", [1, 63, 64, 65, 128, 200])
def test_forks_share_full_blocks_and_write_apart(length):
    cache = make()
    a = cache.alloc_slot()
    write(cache, a, length, 1000)
    b, c = cache.fork(a, 2)
    g = cache._kv_groups[0]
    full = length // 64
    assert g.table_host[b, :full].tolist() == g.table_host[a, :full].tolist() == g.table_host[c, :full].tolist()
    assert g.pool.held_count == full + (3 if length % 64 else 0)
    assert torch.equal(g.table, torch.from_numpy(g.table_host))
    groups = cache.shared_groups([c, a, b])
    assert groups == ([([0, 1, 2], 64 * full)] if full else [])
    cache.check()
    before = read(cache, a)
    write(cache, b, 70, 2000)
    write(cache, c, 3, 3000)
    assert read(cache, a) == before and cache.length(a) == length
    assert read(cache, b)[0][:length] == before[0] and read(cache, b)[0][length:] == [2000.0 + length + i for i in range(70)]
    write(cache, a, 1, 9000)
    assert read(cache, c)[0] == before[0] + [3000.0 + length + i for i in range(3)]
    cache.check()
    cache.free_slot(a)                                     # the others keep what they share
    assert read(cache, b)[0][:length] == before[0]
    cache.free_slot(b)
    cache.free_slot(c)
    assert all(g.pool.held_count == 0 and g.pool.shared_count == 0 for g in cache._kv_groups)
    cache.check()


def test_forks_of_forks_and_groups_of_a_batch():
    cache = make(2048)
    a, x = cache.alloc_slot(), cache.alloc_slot()
    write(cache, a, 130, 0)
    write(cache, x, 200, 0)
    b = cache.fork(a)[0]
    write(cache, b, 130, 0)
    c = cache.fork(b)[0]
    y = cache.fork(x)[0]
    assert cache.shared_groups([b, c]) == [([0, 1], 256)]
    assert cache.shared_groups([a, b, c]) == [([0, 1, 2], 128)]
    assert sorted(cache.shared_groups([y, a, x, b])) == [([0, 2], 192), ([1, 3], 128)]
    assert cache.shared_groups([a, x]) == [] and cache.shared_groups([a]) == []
    cache.check()


def test_states_and_windows_are_carried_over():
    cache = make(1024, window=True, state=True)
    a = cache.alloc_slot()
    write(cache, a, 300, 5)
    cache.state_view(4)[a] = torch.tensor([1.0, 2.0, 3.0])
    b, c = cache.fork(a, 2)
    assert cache.state_view(4)[b].tolist() == cache.state_view(4)[c].tolist() == [1.0, 2.0, 3.0]
    assert read(cache, b) == read(cache, a)
    write(cache, b, 100, 7)
    write(cache, a, 40, 9)
    assert read(cache, c)[3 - 1] == [5.0 + p for p in range(201, 300)]
    cache.check()
    for s in (a, b, c):
        cache.free_slot(s)
    cache.check()


def test_a_fork_that_does_not_fit_changes_nothing():
    cache = make(256)                                      # four blocks
    a = cache.alloc_slot()
    write(cache, a, 130, 0)                                # three of them
    with pytest.raises(CacheFull, match="blocks"):
        cache.fork(a, 2)
    with pytest.raises(CacheFull, match="slots"):
        cache.fork(a, 8)
    with pytest.raises(CacheError, match="not in use"):
        cache.fork(5)
    with pytest.raises(ValueError):
        cache.fork(a, 0)
    cache.check()
    assert cache.slots.free_count == 7 and cache._kv_groups[0].pool.held_count == 3
    b = cache.fork(a)[0]
    assert cache.length(b) == 130
    cache.check()


@pytest.mark.parametrize("length", [0, 1, 64, 100, 128, 130, 190, 199, 200])
def test_going_back(length):
    cache = make()
    a = cache.alloc_slot()
    write(cache, a, 200, 100)
    cache.truncate(a, length)
    assert cache.length(a) == length and read(cache, a)[0] == [100.0 + p for p in range(length)]
    write(cache, a, 100, 500)
    assert read(cache, a)[0] == [100.0 + p for p in range(length)] + [500.0 + p for p in range(length, length + 100)]
    cache.check()
    cache.free_slot(a)
    cache.check()


@pytest.mark.parametrize("length", [0, 1, 64, 100, 128, 130, 192, 199])
def test_going_back_into_shared_blocks(length):
    """What other sequences hold is never written: the last block is copied, blocks behind are let go."""
    cache = make()
    a = cache.alloc_slot()
    write(cache, a, 200, 100)
    b, c = cache.fork(a, 2)
    before = read(cache, a)
    cache.truncate(b, length)
    cache.check()
    write(cache, b, 100, 700)
    assert read(cache, a) == before == read(cache, c)
    assert read(cache, b)[0] == [100.0 + p for p in range(length)] + [700.0 + p for p in range(length, length + 100)]
    cache.check()
    for s in (a, b, c):
        cache.free_slot(s)
    cache.check()
    assert all(g.pool.held_count == 0 for g in cache._kv_groups)


def test_going_back_is_refused_where_the_past_is_gone():
    cache = make(state=True)
    a = cache.alloc_slot()
    write(cache, a, 10, 0)
    with pytest.raises(CacheError, match="states"):
        cache.truncate(a, 5)
    cache.truncate(a, 10)
    cache = make(window=True)
    a = cache.alloc_slot()
    write(cache, a, 300, 0)                                # the window keeps positions from 192 on
    cache.truncate(a, 299)
    with pytest.raises(CacheError, match="given back"):
        cache.truncate(a, 150)
    for bad in (-1, 300):
        with pytest.raises(CacheError, match="cut"):
            cache.truncate(a, bad)
    cache.check()
    cache = make(window=True, pool=8)
    a = cache.alloc_slot()
    write(cache, a, 30, 0)
    with pytest.raises(CacheError, match="pooled"):
        cache.truncate(a, 20)
    cache = make(128)
    a = cache.alloc_slot()
    write(cache, a, 128, 0)
    b = cache.fork(a)[0]
    with pytest.raises(CacheFull):
        cache.truncate(b, 100)                             # no block is left for the copy
    assert cache.length(b) == 128
    cache.check()


@pytest.mark.parametrize("window", [False, True])
@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_steps_forks_cuts_and_frees(seed, window):
    rng = random.Random(seed)
    cache = make(1024, window=window)
    held = {}                                              # slot -> the values its tokens were written with
    for turn in range(120):
        live = sorted(held)
        what = rng.choice(["new", "write", "write", "fork", "cut", "free", "reserve"])
        s = rng.choice(live) if live else None
        try:
            if what == "new" or s is None:
                held[cache.alloc_slot()] = []
            elif what == "write":
                n, at = rng.randint(1, 90), len(held[s])
                write(cache, s, n, 1000.0 * turn)
                held[s] = held[s] + [1000.0 * turn + p for p in range(at, at + n)]
            elif what == "fork":
                for new in cache.fork(s, rng.randint(1, 3)):
                    held[new] = list(held[s])
            elif what == "cut":
                n = rng.randint(0, len(held[s]))
                cache.truncate(s, n)
                held[s] = held[s][:n]
            elif what == "reserve":
                cache.reserve(s, min(1024, len(held[s]) + rng.randint(0, 200)))
            else:
                cache.free_slot(s)
                del held[s]
        except CacheError:                                 # (no room, or a window's keys are gone: nothing has changed)
            pass
        cache.check()
        for b in held:
            assert cache.length(b) == len(held[b])
            for g, got in zip(cache._kv_groups, read(cache, b)):
                assert got == held[b][len(held[b]) - len(got):]
                if b not in g.dirty:                       # (what is goes up before the next step)
                    assert torch.equal(g.table[b], torch.from_numpy(g.table_host[b]))
        slots = rng.sample(sorted(held), len(held))
        for members, p in cache.shared_groups(slots) if len(slots) > 1 else []:
            assert len(members) > 1 and 0 < p <= min(len(held[slots[m]]) for m in members)
            assert all(held[slots[m]][:p] == held[slots[members[0]]][:p] for m in members)
