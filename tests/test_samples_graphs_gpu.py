"""Answers to one prompt that end one after the other: how often a decode step is captured, and what it gives."""
import pytest
import torch

import tiny

pytestmark = pytest.mark.gpu


def engine(model_dirs, name, **kw):
    from cretif_b200.engine import Engine
    return Engine(model_dirs[name], dtype="bfloat16", max_tokens=8192, **kw)


@pytest.fixture
def captures(monkeypatch):
    import sys
    import cretif_b200.engine  # noqa: F401
    generate, seen = sys.modules["cretif_b200.engine.generate"], []
    real = generate.capturing
    monkeypatch.setattr(generate, "capturing", lambda *a: (seen.append(1), real(*a))[1])
    return seen


def run(eng, n, samples, **kw):
    """``samples`` answers that end at different lengths; how many lengths there were."""
    prompt = tiny.tokens("C", n, 3)
    out = [r.tokens for r in eng.generate([prompt], max_tokens=120, temperature=1.5, seed=4,
                                          stop_ids=list(range(0, eng.vocab_size, 25)), samples=samples, **kw)]
    assert len({len(t) for t in out}) >= min(samples, 12) // 2
    return out


def test_steps_that_gain_nothing_share_the_graphs_of_all_others(model_dirs, captures):
    """A short prompt's answers take the ordinary kernels: batches of a size share a graph, whatever is
    shared, from prompt to prompt and beside copies of the prompt."""
    from cretif_b200.parts import attention
    eng = engine(model_dirs, "C")
    heads = eng.model.shared_heads()
    assert heads and not any(attention.shared_pays([(list(range(16)), 128)], [1] * 16, [150] * 16, *h) for h in heads)
    run(eng, 150, 16)
    first = len(captures)
    assert 0 < first <= 16
    run(eng, 150, 16)
    assert len(captures) == first
    run(eng, 215, 16)                                       # (the same contexts in buckets, other blocks shared)
    eng.generate([tiny.tokens("C", 150, 3)] * 16, max_tokens=4, temperature=1.5, seed=4, stop_ids=[])
    again = len(captures)
    run(eng, 280, 16)
    assert len(captures) - again <= 2                       # (batch sizes that did not come before)
    (runner,) = {b.runner for b in eng._backends.values()}
    assert all(k[2] == () for k in runner.graphs)


def test_forked_steps_that_gain_nothing_share_captured_steps(model_dirs):
    eng = engine(model_dirs, "C")
    outs = []
    for n in (130, 200):                                    # two blocks in common, then three
        a = eng.alloc_slot()
        eng.step([(a, tiny.tokens("C", n, 1))])
        b = eng.fork_slot(a)[0]
        for _ in range(3):
            outs.append(eng.step([(a, [5]), (b, [6])]))
        eng.free_slot(a), eng.free_slot(b)
    alone = [eng.alloc_slot() for _ in range(2)]
    for s in alone:
        eng.step([(s, tiny.tokens("C", 130, 1))])
    eng.step([(alone[0], [5]), (alone[1], [6])])
    assert len([k for k in eng._graphs if k[0] == (1, 1)]) == 1
    assert all(torch.isfinite(o).all() for o in outs)
