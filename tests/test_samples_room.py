"""What a batch of several answers a prompt was promised is there: the cache's blocks, and those of pooled entries."""
import pytest
import torch

from cretif_b200.cache import KVRequest, SequenceCache
from test_generation_loop import ScriptedBackend, loop


@pytest.mark.parametrize("pool", [4, 16, 128])
@pytest.mark.parametrize("max_tokens, max_slots", [(512, None), (1024, None), (2560, 10)])
def test_the_most_answers_that_fit(pool, max_tokens, max_slots):
    fork_only = 0
    for n in list(range(64, max_tokens, 192)) + [130, 190, 250, 448]:
        for answer in (2, 10, 70):
            most = 0
            for samples in range(1, 41):
                cache = SequenceCache({0: KVRequest(1, 2, window=100, pool=pool), 1: KVRequest(1, 2)}, max_tokens,
                                      torch.float32, "cpu", max_slots=max_slots)
                g = loop(ScriptedBackend({}), capacity=cache.max_tokens, max_len=cache.max_len)
                try:
                    g.plan_batches([n], answer, samples)
                except ValueError:
                    break
                if samples > cache.max_slots:
                    break
                most = samples
            if most < 2:
                continue
            fork_only += 1
            reserve = g._reserve_len(n, answer)
            a = cache.alloc_slot()
            cache.reserve(a, reserve)
            cache.begin_step([(a, n)])
            cache.end_step([(a, n)])
            slots = [a] + cache.fork(a, most - 1)
            for s in slots:
                cache.reserve(s, reserve)
            for _ in range(reserve - n):
                cache.begin_step([(s, 1) for s in slots])
                cache.end_step([(s, 1) for s in slots])
            cache.check()
    assert fork_only > 5


def test_answers_of_one_token_need_no_room():
    g = loop(ScriptedBackend({}), capacity=192)
    assert g.plan_batches([130], 1, samples=16) == [list(range(16))]
    with pytest.raises(ValueError, match="cache holds"):
        g.plan_batches([130], 2, samples=16)
