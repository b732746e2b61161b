"""Several answers a prompt: the loop's decisions, with a scripted backend on the CPU."""
import pytest

from test_generation_loop import ScriptedBackend, loop


class Sampling(ScriptedBackend):
    def start_batch(self, request_ids, prompts, reserve_lens, samples=1):
        super().start_batch(request_ids, prompts, reserve_lens)
        self.log[-1] += (samples, tuple(tuple(p) for p in prompts))


def test_requests_of_a_prompt_stay_together_and_in_order():
    be = Sampling({i: [10 + i] * 5 for i in range(6)})
    res = loop(be, max_batch=4).run([[1], [2, 2], [3]], max_tokens=2, samples=2)
    assert [r.tokens for r in res] == [[10 + i] * 2 for i in range(6)]
    assert [r.prompt_len for r in res] == [1, 1, 2, 2, 1, 1]
    starts = [e for e in be.log if e[0] == "start"]
    assert [e[1] for e in starts] == [(0, 1, 2, 3), (4, 5)] and all(e[3] == 2 for e in starts)
    assert starts[0][4] == ((1,), (1,), (2, 2), (2, 2))


def test_room_is_counted_with_the_prompts_blocks_once():
    g = loop(Sampling({}), capacity=512)
    # 130 + 29 positions: three blocks, of which two are the prompt's and held once
    assert g.plan_batches([130, 130], 30, samples=3) == [[0, 1, 2], [3, 4, 5]]        # 3 + 2 each
    assert g.plan_batches([130], 30, samples=6) == [[0, 1, 2, 3, 4, 5]]               # 3 + 5
    with pytest.raises(ValueError, match="cache holds"):
        g.plan_batches([130], 30, samples=7)
    assert g.plan_batches([10, 10], 10) == [[0, 1]]


def test_refusals():
    for samples in (0, -1, 65):
        with pytest.raises(ValueError, match="answers a prompt"):
            loop(Sampling({})).run([[1]], max_tokens=2, samples=samples)
    assert [r.finish_reason for r in loop(Sampling({})).run([[1], [2]], max_tokens=0, samples=2)] == ["length"] * 4
