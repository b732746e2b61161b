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


def test_graphs_of_shared_prefixes_are_kept(model_dirs, captures, monkeypatch):
    """Where steps share, a make-up that comes again finds its graph; the latest used are kept."""
    import sys
    from cretif_b200.parts import attention
    generate = sys.modules["cretif_b200.engine.generate"]
    monkeypatch.setattr(attention, "SHARED_MIN_BYTES", 0)   # (a capture costs nothing, all gain)
    eng = engine(model_dirs, "C")
    want = run(eng, 150, 24)
    first = len(captures)
    assert first > 10
    assert run(eng, 150, 24) == want and len(captures) == first
    (runner,) = {b.runner for b in eng._backends.values()}
    assert len([k for k in runner.graphs if k[2]]) > 10
    monkeypatch.setattr(generate, "MAX_SHARED_GRAPHS", 5)
    eng.generate([tiny.tokens("C", 150, 3)], max_tokens=4, temperature=1.5, seed=4, stop_ids=[], samples=24)
    largest = max(len(k[2][0][0]) for k in runner.graphs if k[2])
    assert largest == 24
    for n in range(6):                                      # other make-ups push out the rest, not the one in use
        eng.generate([tiny.tokens("C", 215 + 64 * n, 3)], max_tokens=3, temperature=1.5, seed=4, stop_ids=[], samples=2)
        eng.generate([tiny.tokens("C", 150, 3)], max_tokens=3, temperature=1.5, seed=4, stop_ids=[], samples=24)
    kept = [k for k in runner.graphs if k[2]]
    assert len(kept) <= 24 + 6 and any(len(k[2][0][0]) == 24 for k in kept)


def test_a_make_up_runs_as_the_ordinary_step_until_a_graph_pays(model_dirs, captures, monkeypatch):
    """What comes of a call does not depend on which graphs are there, or on whether there are any."""
    from cretif_b200.csrc import ops
    from cretif_b200.engine import engine as module
    from cretif_b200.parts import attention
    eng = engine(model_dirs, "C")
    prompt = tiny.tokens("C", 150, 3)
    heads = eng.model.shared_heads()
    layers = sum(heads.values())
    ((nh, nkv, hd),) = heads
    spared = layers * attention.shared_spares([(list(range(6)), 128)], nkv, hd)
    monkeypatch.setattr(attention, "shared_pays", lambda *a: True)
    monkeypatch.setattr(module, "SHARED_CAPTURE", 10 * spared / attention.SHARED_MIN_BYTES)
    steps, real = [], ops.attn_shared
    monkeypatch.setattr(ops, "attn_shared", lambda *a, **k: (steps.append(1), real(*a, **k))[1])

    def go(**kw):
        return [r.tokens for r in eng.generate([prompt], max_tokens=30, temperature=1.5, seed=4, stop_ids=[], samples=6, **kw)]
    first = go()
    (runner,) = {b.runner for b in eng._backends.values()}
    assert sorted(bool(k[2]) for k in runner.graphs) == [False, True]
    n = len(captures)
    assert go() == first and len(captures) == n             # (the same kernels step for step, no capture)
    del steps[:]
    assert go(use_graph=False) == first
    assert len(steps) == (29 - 10) * layers                 # the first token is the prompt's, ten steps wait


def test_a_plan_is_made_once_for_steps_of_a_make_up(model_dirs, monkeypatch):
    """Steps with drafts that are not captured, and the layers of each, use the plan of the first."""
    from cretif_b200.csrc import ops
    from cretif_b200.engine import engine as module
    made = []
    real = ops.shared_prefix_plan
    monkeypatch.setattr(ops, "shared_prefix_plan", lambda *a: (made.append(real(*a)), made[-1])[1])
    eng = engine(model_dirs, "C", step_graphs=False)
    a = eng.alloc_slot()
    eng.step([(a, tiny.tokens("C", 150, 1))])
    b = eng.fork_slot(a)[0]
    outs = []
    for i in range(4):
        outs.append(eng.step([(a, [5, 7]), (b, [6])], "all"))
        eng.truncate_slot(a, 150), eng.truncate_slot(b, 150)
    assert len(made) == 1 and all(torch.equal(outs[0], o) for o in outs)
    for n in (1, 2):                                        # the other way round, and another number of drafts
        eng.step([(a, [5] * n), (b, [6, 8, 1])])
    assert len(made) == 3
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    eng.truncate_slot(a, 150), eng.truncate_slot(b, 150)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):                         # kept plans serve other streams
        got = eng.step([(a, [5, 7]), (b, [6])], "all")
    torch.cuda.synchronize()
    assert torch.equal(got, outs[0]) and len(made) == 3
    for n in range(1, module.MAX_SHARED_PLANS + 9):
        eng.truncate_slot(a, 150), eng.truncate_slot(b, 150)
        eng.step([(a, [5] * (1 + n % 9)), (b, [6] * (2 + n // 9))])
    assert len(eng._shared_plans) == module.MAX_SHARED_PLANS


@pytest.mark.parametrize("block_tokens", [32, 128])
def test_blocks_of_another_size_are_shared_in_the_cache_alone(model_dirs, monkeypatch, block_tokens):
    """The attention over shared prefixes takes blocks of 64: forks on others step as all sequences do."""
    from cretif_b200.csrc import ops
    from cretif_b200.parts import attention
    monkeypatch.setattr(attention, "shared_pays", lambda *a: True)
    monkeypatch.setattr(ops, "attn_shared", None)
    eng = engine(model_dirs, "C", block_tokens=block_tokens)
    prompt = tiny.tokens("C", 300, 3)
    opts = dict(max_tokens=12, temperature=1.5, seed=4, stop_ids=[])
    got = [r.tokens for r in eng.generate([prompt], samples=4, **opts)]
    assert got == [r.tokens for r in eng.generate([prompt] * 4, **opts)]
    a = eng.alloc_slot()
    eng.step([(a, prompt)])
    b = eng.fork_slot(a)[0]
    for _ in range(3):
        eng.step([(a, [5, 6]), (b, [7])])
    assert eng.cache.shared_groups([a, b]) == [([0, 1], 300 // block_tokens * block_tokens)]
    assert all(k[1] == "last" for k in eng._graphs)


def test_shapes_that_never_come_again_are_forgotten(model_dirs):
    """Steps with drafts are of ever new shapes: how many of them an engine remembers is bounded."""
    eng = engine(model_dirs, "C")
    a, b = eng.alloc_slot(), eng.alloc_slot()
    eng._seen.update({("a shape", i): 1 for i in range(4096)})
    eng.step([(a, [1, 2, 3]), (b, [4])])
    assert len(eng._seen) == 1
    eng.step([(a, [1, 2, 3]), (b, [4])])
    assert len(eng._graphs) == 1
    eng._seen.update({("a shape", i): 1 for i in range(4095)})
    for n in range(1, 12):
        eng.step([(a, [1] * n), (b, [4] * 9)])
        assert len(eng._seen) <= 4096
