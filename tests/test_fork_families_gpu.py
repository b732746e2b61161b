"""Forked sequences and several answers a prompt in every registered architecture: recurrent states, convolutions'
last inputs, pooled entries, sinks, chunks, shared latents and borrowed caches go on from where the prompt ended."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

FAMILIES = ["rigozen", "losorax", "virorax", "mipurax", "gibipel", "pudorax"]
# families of whose attention some is over all keys, with no bias and values like the keys
SHARING = {("mipurax", "B"), ("pudorax", "B")}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    made = {}

    def get(family, name):
        if (family, name) not in made:
            test = importlib.import_module(f"test_{family}_gpu")
            tiny = importlib.import_module(f"{family}_tiny")
            made[family, name] = (test._write(tmp_path_factory, f"forks_{name}", tiny.CONFIGS[name], tiny.SEEDS[name]),
                                  test, tiny)
        return made[family, name]
    return get


@pytest.fixture
def always_shared(monkeypatch):
    from cretif_b200.csrc import ops
    from cretif_b200.parts import attention
    monkeypatch.setattr(attention, "SHARED_MIN_BYTES", 0)
    seen, real = [], ops.attn_shared
    monkeypatch.setattr(ops, "attn_shared", lambda *a, **k: (seen.append(a[8]), real(*a, **k))[1])
    return seen


def steps(eng, slots, tiny, name, prompt):
    """Single tokens, several, and a fork that ends; what every step gives, and what every sequence was fed."""
    out, texts = [], [list(prompt) for _ in slots]
    for i, news in enumerate([(1, 1, 1), (1, 1, 1), (1, 1, 1), (3, 1, 2), (1, 1, 1), (0, 4, 4), (0, 1, 1), (0, 20, 1)]):
        entries = []
        for b, n in enumerate(news):
            if n:
                toks = tiny.tokens(name, n, 100 + 10 * i + b)
                texts[b] += toks
                entries.append((slots[b], toks))
        out.append(eng.step(entries, "all").clone())
    return out, texts


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "D"])
@pytest.mark.parametrize("family", FAMILIES)
def test_forks_go_on_where_the_prompt_ended(models, always_shared, family, name, dtype):
    from cretif_b200.engine import Engine
    folder, test, tiny = models(family, name)
    eng = Engine(folder, dtype=dtype, max_tokens=4096)
    n = 150
    prompt = tiny.tokens(name, n, 5)
    apart = []
    for _ in range(3):                                      # the same, each with a prompt of its own
        s = eng.alloc_slot()
        eng.step([(s, prompt)])
        apart.append(s)
    want, texts = steps(eng, apart, tiny, name, prompt)
    for s in apart:
        eng.free_slot(s)
    assert not always_shared
    a = eng.alloc_slot()
    eng.step([(a, prompt)])
    forked = [a] + eng.fork_slot(a, 2)
    eng.cache.check()
    got, _ = steps(eng, forked, tiny, name, prompt)
    eng.cache.check()
    if dtype == "bfloat16" and (family, name) in SHARING:
        assert always_shared
    if not always_shared:
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    else:
        # both are the same sums in another order, and roundings of them: against the plain model each
        plain = importlib.import_module(f"plain_{family}")
        cfg, w = plain.read_model_folder(folder)
        rows = [plain.forward(cfg, w, t).numpy()[n:] for t in texts]
        check = getattr(test, "close_routed", test.close)
        for which in (got, want):
            mine = [[] for _ in range(3)]
            for i, news in enumerate([(1, 1, 1)] * 3 + [(3, 1, 2), (1, 1, 1), (0, 4, 4), (0, 1, 1), (0, 20, 1)]):
                at = 0
                for b, k in enumerate(news):
                    mine[b].append(which[i][at:at + k])
                    at += k
            for b in range(3):
                assert check(torch.cat(mine[b]).float().cpu().numpy(), rows[b], dtype)
    # the first may go on, and be forked again, behind what the others did
    again = eng.fork_slot(forked[1])
    x = eng.step([(forked[1], [3])])
    y = eng.step([(again[0], [3])])
    assert torch.equal(x, y)
    for s in forked + again:
        eng.free_slot(s)
    eng.cache.check()
    eng.check_fault()


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("family", FAMILIES)
def test_several_answers_are_those_of_copies(models, family, name):
    from cretif_b200.engine import Engine
    folder, _, tiny = models(family, name)
    prompts = [tiny.tokens(name, n, 6) for n in (130, 64, 9)]
    eng = Engine(folder, dtype="float32", max_tokens=4096)
    opts = dict(max_tokens=12, temperature=0.9, top_k=20, seed=3, stop_ids=[])
    want = eng.generate([p for p in prompts for _ in range(3)], **opts)
    for use_graph in (True, False):
        got = eng.generate(prompts, samples=3, use_graph=use_graph, **opts)
        assert [r.tokens for r in got] == [r.tokens for r in want]
    # answers of one token are drawn from the prompt's logits, and need no room of their own
    one = {**opts, "max_tokens": 1}
    tight = Engine(folder, dtype="float32", max_tokens=192)
    got = tight.generate(prompts[:1], samples=16, **one)
    want = eng.generate(prompts[:1] * 16, **one)
    assert [r.tokens for r in got] == [r.tokens for r in want]
    assert not eng.cache.slots.live() and not tight.cache.slots.live()
    for e in (eng, tight):
        e.cache.check()


@pytest.mark.parametrize("family", FAMILIES)
def test_only_what_can_go_back_is_cut(models, family):
    from cretif_b200.cache import CacheError
    from cretif_b200.engine import Engine
    folder, _, tiny = models(family, "B")
    eng = Engine(folder, dtype="float32", max_tokens=4096)
    a, b = eng.alloc_slot(), eng.alloc_slot()
    toks = tiny.tokens("B", 100, 1)
    eng.step([(a, toks), (b, toks[:97])])
    if eng.cache.has_states() or eng.cache._pool_of:
        with pytest.raises(CacheError, match="cannot go back"):
            eng.truncate_slot(a, 97)
        assert eng.cache.length(a) == 100
    else:
        eng.truncate_slot(a, 97)
        assert torch.equal(eng.step([(a, [4, 2])]), eng.step([(b, [4, 2])]))
    eng.cache.check()
