"""Which forked sequences a step groups: those that spare the most reading."""
import random

import torch

from cretif_b200.cache import KVRequest, SequenceCache


def make(max_tokens=64 * 400, slots=40):
    return SequenceCache({0: KVRequest(1, 1)}, max_tokens, torch.float32, "cpu", max_slots=slots)


def grow(cache, slot, n):
    cache.begin_step([(slot, n)])
    cache.end_step([(slot, n)])


def test_an_early_fork_does_not_take_the_sharing_from_the_others():
    cache = make()
    a = cache.alloc_slot()
    grow(cache, a, 130)
    early = cache.fork(a)[0]                                # shares 128 tokens
    grow(cache, a, 8000)
    rest = cache.fork(a, 30)
    slots = [early, a] + rest
    assert cache.shared_groups(slots) == [(list(range(1, 32)), 8128)]
    assert cache.shared_groups([early, a]) == [([0, 1], 128)]
    cache.check()


def test_several_prompts_behind_one_block():
    """A system prompt's block that all share, and what is behind it: the groups of the prompts."""
    cache = make()
    a = cache.alloc_slot()
    grow(cache, a, 64)
    prompts = [a] + cache.fork(a, 3)
    for i, p in enumerate(prompts):
        grow(cache, p, 640 if i < 2 else 5)
    answers = [[p] + cache.fork(p, 4) for p in prompts[:2]]
    slots = answers[0] + prompts[2:] + answers[1]
    assert cache.shared_groups(slots) == [([0, 1, 2, 3, 4], 704), ([7, 8, 9, 10, 11], 704)]
    # where the rest is long enough only for few, all together spare more
    assert cache.shared_groups(prompts) == [([0, 1, 2, 3], 64)]


def spared(groups):
    return sum((len(m) - 1) * p for m, p in groups)


def brute(rows, members, at):
    """The most that any grouping spares, by trying the tree of common beginnings."""
    n = at
    while all(r[n] == rows[members[0]][n] >= 0 for r in (rows[m] for m in members)):
        n += 1
    best = (len(members) - 1) * n
    parts = {}
    for m in members:
        parts.setdefault(rows[m][n], []).append(m)
    return max(best, sum(brute(rows, p, n) for b, p in parts.items() if b >= 0 and len(p) > 1))


def test_any_tree_of_forks():
    rng = random.Random(5)
    for _ in range(40):
        cache = make()
        first = cache.alloc_slot()
        grow(cache, first, 64 * rng.randint(1, 4))
        slots = [first]
        while len(slots) < 14:
            s = rng.choice(slots)
            if rng.random() < 0.5:
                grow(cache, s, rng.randint(1, 200))
            else:
                slots += cache.fork(s, rng.randint(1, 3))
        rng.shuffle(slots)
        groups = cache.shared_groups(slots)
        seen = [m for members, _ in groups for m in members]
        assert len(seen) == len(set(seen))
        table = cache._kv_groups[0].table_host
        for members, p in groups:
            heads = {tuple(table[slots[m], :p // 64].tolist()) for m in members}
            assert len(heads) == 1 and -1 not in heads.pop()
            assert all(cache.length(slots[m]) >= p for m in members)
        rows = [table[s].tolist() + [-1] for s in slots]
        by_first = {}
        for i, r in enumerate(rows):
            by_first.setdefault(r[0], []).append(i)
        want = sum(64 * brute(rows, m, 0) for m in by_first.values() if len(m) > 1)
        assert spared(groups) == want


def test_a_chain_of_forks():
    cache = make(slots=200, max_tokens=64 * 1000)
    s = cache.alloc_slot()
    slots = [s]
    for _ in range(150):
        grow(cache, s, 64)
        s = cache.fork(s)[0]
        slots.append(s)
    groups = cache.shared_groups(slots)
    assert groups and spared(groups) > 0
    cache.check()
