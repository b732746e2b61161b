"""The cache's own check: it finds what is wrong, in time that grows with the blocks, not with their square."""
import time

import pytest
import torch

from cretif_b200.cache import CacheError, KVRequest, SequenceCache


def test_many_blocks():
    n = 24000
    cache = SequenceCache({0: KVRequest(1, 1)}, 64 * n, torch.float32, "cpu", max_slots=4)
    a = cache.alloc_slot()
    cache.reserve(a, 64 * n // 2)
    start = time.perf_counter()
    cache.check()
    apart = time.perf_counter() - start
    cache.begin_step([(a, 64 * n // 2)])
    cache.end_step([(a, 64 * n // 2)])
    cache.fork(a, 3)
    start = time.perf_counter()
    cache.check()
    took = time.perf_counter() - start
    # (twice the blocks held by four: four times the entries; counting each by walking all is sixteen times)
    assert took < 1.0 and apart < 1.0


def test_what_is_wrong_is_found():
    cache = SequenceCache({0: KVRequest(1, 4)}, 1024, torch.float32, "cpu", max_slots=4)
    a = cache.alloc_slot()
    cache.begin_step([(a, 200)])
    cache.end_step([(a, 200)])
    b = cache.fork(a)[0]
    cache.check()
    g = cache._kv_groups[0]
    row = g.table_host[b].copy()
    g.table_host[b, 0] = g.table_host[b, 1]                # one block once too often, another too seldom
    with pytest.raises(CacheError, match="mapped by"):
        cache.check()
    g.table_host[b] = row
    g.table_host[b, 3] = -1                                # a block that nobody maps
    with pytest.raises(CacheError, match="are mapped"):
        cache.check()
    g.table_host[b] = row
    cache.check()
