"""Several answers to one prompt, and drafts that are taken back, through the engine: against the plain
implementation, and the operators together as a program uses them."""
import numpy as np
import pytest
import torch

import plain_llama
import tiny
from replay_cuts import rel_err

pytestmark = pytest.mark.gpu

# (the bounds of the engine's other tests: activations and cached keys in 8 bits of mantissa, and 32-bit)
TOL = {"float32": 1e-4, "bfloat16": 2e-2}


@pytest.fixture
def always_shared(monkeypatch):
    """Single tokens take the attention over shared prefixes however little it spares."""
    from cretif_b200.parts import attention
    monkeypatch.setattr(attention, "SHARED_MIN_BYTES", 0)


@pytest.fixture
def calls(monkeypatch):
    from cretif_b200.csrc import ops
    seen = []
    real = ops.attn_shared
    monkeypatch.setattr(ops, "attn_shared", lambda *a, **k: (seen.append(a[8]), real(*a, **k))[1])
    return seen


def engine(model_dirs, name, dtype, **kw):
    from cretif_b200.engine import Engine
    return Engine(model_dirs[name], dtype=dtype, max_tokens=4096, **kw)


def plain(plain_models, name, toks):
    cfg, w = plain_models[name]
    return plain_llama.forward(cfg, w, list(toks)).numpy()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["A", "B", "C", "W"])
def test_forks_give_what_whole_prompts_give(model_dirs, plain_models, always_shared, calls, name, dtype):
    """A prompt run once and forked; single tokens, drafts, forks of forks, an answer that ends."""
    eng = engine(model_dirs, name, dtype)
    n = {"A": 70}.get(name, 150)
    prompt = tiny.tokens(name, n, 1)
    a = eng.alloc_slot()
    eng.step([(a, prompt)])
    slots = [a] + eng.fork_slot(a, 3)
    texts = {s: list(prompt) for s in slots}

    def step(news):
        entries = [(s, tiny.tokens(name, k, 100 + 7 * s + len(texts[s]))) for s, k in news]
        got = eng.step(entries, "all").float().cpu().numpy()
        at = 0
        for s, toks in entries:
            texts[s] += toks
            want = plain(plain_models, name, texts[s])[-len(toks):]
            assert rel_err(got[at:at + len(toks)], want) <= TOL[dtype], (name, s, len(texts[s]))
            at += len(toks)
        eng.cache.check()
    for _ in range(3):
        step([(s, 1) for s in slots])
    step([(slots[2], 3), (slots[0], 1), (slots[1], 5)])
    more = eng.fork_slot(slots[1])
    texts[more[0]] = list(texts[slots[1]])
    eng.free_slot(slots[0])
    for _ in range(2):
        step([(s, 1) for s in more + slots[1:]])
    step([(s, 4) for s in more + slots[1:]])
    if dtype == "bfloat16" and name != "W":
        # one layer's calls: single tokens twice and their capture (then they are replayed), two steps of drafts
        assert len(calls) >= 5
        assert all(p.T >= 3 for p in calls)
    if dtype == "float32":
        assert not calls
    for s in more + slots[1:]:
        eng.free_slot(s)
    eng.cache.check()


def test_little_in_common_takes_the_ordinary_kernels(model_dirs, calls):
    eng = engine(model_dirs, "B", "bfloat16")
    a = eng.alloc_slot()
    eng.step([(a, tiny.tokens("B", 130, 1))])
    b = eng.fork_slot(a)[0]
    eng.step([(a, [5]), (b, [6])])
    assert not calls
    eng.step([(a, [5, 7]), (b, [6])])
    assert calls
    del calls[:]
    eng.step([(a, [5] * 17), (b, [6])])                     # a prompt's chunk
    c = eng.alloc_slot()
    eng.step([(c, [1, 2, 3]), (a, [4])])                    # nothing in common
    assert not calls


def test_captured_steps_of_forks(model_dirs, always_shared):
    """The third step of a shape is replayed from a graph; other forks of the same shape, and steps of
    sequences that share nothing, are not mistaken for it."""
    prompt = tiny.tokens("C", 200, 3)
    outs = []
    for graphs in (True, False):
        eng = engine(model_dirs, "C", "bfloat16", step_graphs=graphs)
        got = []
        for round_ in range(2):
            a = eng.alloc_slot()
            eng.step([(a, prompt[:180 + 20 * round_])])
            slots = [a] + eng.fork_slot(a, 2)
            alone = eng.alloc_slot()
            eng.step([(alone, prompt[:90])])
            for i in range(5):
                got.append(eng.step([(s, [11 + i + s % 3]) for s in slots]))
                got.append(eng.step([(s, [11 + i + s % 3, 4]) for s in (slots[0], slots[1], alone)], "all"))
            for s in slots + [alone]:
                eng.free_slot(s)
        outs.append([g.cpu() for g in got])
    for x, y in zip(*outs):
        assert torch.equal(x, y)


def test_plans_follow_the_answers_lengths(model_dirs, always_shared, calls):
    """A plan cuts own keys by how many there are: steps of the same shape get another one as they grow."""
    eng = engine(model_dirs, "C", "bfloat16")
    a = eng.alloc_slot()
    eng.step([(a, tiny.tokens("C", 64, 3))])
    b = eng.fork_slot(a)[0]
    for _ in range(3):
        eng.step([(s, [5, 6]) for s in (a, b)])
    few = {id(p) for p in calls}
    eng.step([(s, tiny.tokens("C", 600, 3)) for s in (a, b)])
    del calls[:]
    eng.step([(s, [5, 6]) for s in (a, b)])
    assert calls and not few & {id(p) for p in calls}
    for s in (a, b):
        eng.free_slot(s)
    for use_graph in (True, False):
        del calls[:]
        eng.generate([tiny.tokens("C", 64, 3)], max_tokens=600, stop_ids=[], samples=2, use_graph=use_graph)
        assert len({id(p) for p in calls}) == 2             # up to 512 tokens of their own, and beyond


def draft(rng, right, wrong, vocab):
    """Drafts of which some are the model's next tokens and some are not."""
    return [t if rng.random() < 0.7 else int(rng.integers(0, vocab)) for t in right] + [int(t) for t in wrong]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafts_verified_and_taken_back_greedy(model_dirs, plain_models, dtype):
    """Three answers to a prompt, each stepped with drafts, verified, cut back to what stands: in float32 the
    tokens are the plain model's greedy ones, in bfloat16 the best or within the bound of it."""
    from cretif_b200.sampling import DraftVerifier, SamplingParams
    name, K, total = "B", 4, 24
    cfg, w = plain_models[name]
    eng = engine(model_dirs, name, dtype)
    V = eng.vocab_size
    verifier = DraftVerifier(SamplingParams(0.0), V)
    rng = np.random.default_rng(7)
    prompt = tiny.tokens(name, 100, 5)
    a = eng.alloc_slot()
    eng.step([(a, prompt)])
    slots = [a] + eng.fork_slot(a, 2)
    # the answers begin apart
    texts = [list(prompt) + [3 + 5 * i] for i in range(3)]
    start = [len(t) for t in texts]
    goal = [plain_llama.greedy(cfg, w, t, total + K + 1) for t in texts]
    rounds = 0
    while any(len(t) - s < total for t, s in zip(texts, start)):
        rounds += 1
        live = [i for i in range(3) if len(texts[i]) - start[i] < total]
        drafts = np.full((len(live), K), -7, dtype=np.int32)
        entries, cu = [], [0]
        for r, i in enumerate(live):
            n = int(rng.integers(0, K + 1))
            at = len(texts[i]) - start[i]
            d = draft(rng, goal[i][at:at + n], [], V)
            drafts[r, :n] = d
            entries.append((slots[i], [texts[i][-1]] + d))
            cu.append(cu[-1] + 1 + n)
        logits = eng.step(entries, "all")
        dev = dict(device="cuda", dtype=torch.int32)
        accepted, tokens = torch.empty(len(live), **dev), torch.empty((len(live), K + 1), **dev)
        u = torch.rand((len(live), K), device="cuda")
        verifier(logits, torch.tensor(cu, **dev), torch.from_numpy(drafts).cuda(), u, u[:, 0].contiguous(), accepted, tokens)
        for r, i in enumerate(live):
            n = int(accepted[r])
            got = tokens[r, :n + 1].tolist()
            assert got[:n] == entries[r][1][1:n + 1] and all(t == -1 for t in tokens[r, n + 1:].tolist())
            texts[i] += got
            eng.truncate_slot(slots[i], len(texts[i]) - 1)
        eng.cache.check()
        eng.check_fault()
    assert rounds < total                                   # some drafts stood
    for i in range(3):
        got = texts[i][start[i]:]
        if dtype == "float32":
            assert got[:total] == goal[i][:total]
        else:
            rows = plain_llama.forward(cfg, w, texts[i][:-1], storage=torch.bfloat16).numpy()[start[i] - 1:]
            bound = 4e-2 * float(np.abs(rows).max())
            for row, t in zip(rows, got):
                assert row.max() - row[t] <= bound


def test_sampled_drafts_from_a_smaller_model(model_dirs):
    """Drafts drawn from another model's logits at a temperature, verified with given numbers: the verifier's
    answer is the definition's on the very logits, and the sequences go on from what stands."""
    from test_verify_drafts_gpu import by_definition
    from cretif_b200.sampling import DraftVerifier, Sampler, SamplingParams
    big, small = engine(model_dirs, "B", "bfloat16"), engine(model_dirs, "B", "float32")
    V, K, B = big.vocab_size, 3, 4
    params = SamplingParams(0.9, 20, seed=11)
    sampler, verifier = Sampler(params, V), DraftVerifier(params, V)
    prompt = tiny.tokens("B", 64, 9)
    slots = {}
    for eng in (big, small):
        a = eng.alloc_slot()
        eng.step([(a, prompt)])
        slots[eng] = [a] + eng.fork_slot(a, B - 1)
    last = [[7 + i] for i in range(B)]
    gen = torch.Generator().manual_seed(3)
    dev = dict(device="cuda", dtype=torch.int32)
    draws = torch.zeros(B, **dev)
    total = 0
    for _ in range(6):
        drafts, q = torch.empty((B, K), **dev), torch.empty((B, K, V), device="cuda")
        feed = [list(x) for x in last]
        before = [small.cache.length(s) for s in slots[small]]
        for j in range(K):
            q[:, j] = small.step([(s, f) for s, f in zip(slots[small], feed)])
            out = torch.empty(B, **dev)
            sampler(q[:, j].contiguous(), out, torch.arange(B, device="cuda"), draws)
            drafts[:, j] = out
            feed = [[t] for t in out.tolist()]
        logits = big.step([(s, x[-1:] + d) for s, x, d in zip(slots[big], last, drafts.tolist())], "all")
        cu = (torch.arange(B + 1) * (K + 1)).int().cuda()
        u = ((torch.randint(0, 1 << 24, (B, K + 1), generator=gen).float() + 0.5) / (1 << 24)).cuda()
        accepted, tokens = torch.empty(B, **dev), torch.empty((B, K + 1), **dev)
        verifier(logits, cu, drafts, u[:, :K], u[:, K].contiguous(), accepted, tokens, draft_logits=q)
        want = by_definition(logits, cu, drafts, u[:, :K], u[:, K], 0.9, 20, q)
        assert torch.equal(accepted.cpu(), want[0]) and torch.equal(tokens.cpu(), want[1])
        for i in range(B):
            n = int(accepted[i])
            total += n
            # the model has seen its last token and the drafts that stand, the small one all but the last draft
            have = big.cache.length(slots[big][i]) - K + n
            big.truncate_slot(slots[big][i], have)
            small.truncate_slot(slots[small][i], min(small.cache.length(slots[small][i]), before[i] + len(last[i]) + n))
            fresh = int(tokens[i, n])
            last[i] = ([int(drafts[i, K - 1])] if n == K else []) + [fresh]
            missing = have + 1 - small.cache.length(slots[small][i])
            assert missing == len(last[i])
        for eng in (big, small):
            eng.cache.check()
            eng.check_fault()
    assert total > 6                                        # the models are alike: many drafts stand


def test_generate_beside_forks(model_dirs):
    """Generation takes no notice of sequences that are forked beside it, and of blocks that were."""
    eng = engine(model_dirs, "B", "bfloat16")
    prompts = [tiny.tokens("B", 90, 4), tiny.tokens("B", 20, 5)]
    want = [r.tokens for r in eng.generate(prompts, max_tokens=12, stop_ids=[])]
    a = eng.alloc_slot()
    eng.step([(a, tiny.tokens("B", 130, 1))])
    forks = eng.fork_slot(a, 2)
    eng.step([(s, [4, 5]) for s in forks])
    assert [r.tokens for r in eng.generate(prompts, max_tokens=12, stop_ids=[])] == want
    for s in [a] + forks:
        eng.free_slot(s)
    assert [r.tokens for r in eng.generate(prompts, max_tokens=12, stop_ids=[])] == want
    eng.cache.check()


@pytest.mark.parametrize("name", ["A", "B", "C", "W"])
def test_several_answers_a_prompt(model_dirs, plain_models, always_shared, name):
    """float32: each greedy answer is the plain model's, each sampled one what its request gives alone.
    bfloat16: the best tokens or within the bound; the prompts' blocks are held once."""
    prompts = [tiny.tokens(name, n, 6) for n in (70, 9, 66)]
    cfg, w = plain_models[name]
    eng = engine(model_dirs, name, "float32")
    res = eng.generate(prompts, max_tokens=6, stop_ids=[], samples=3)
    assert len(res) == 9
    for i, r in enumerate(res):
        assert r.tokens == plain_llama.greedy(cfg, w, prompts[i // 3], 6) and r.prompt_len == len(prompts[i // 3])
    one = eng.generate([p for p in prompts for _ in range(3)], max_tokens=20, temperature=0.8, top_k=30, seed=5, stop_ids=[])
    many = eng.generate(prompts, max_tokens=20, temperature=0.8, top_k=30, seed=5, stop_ids=[], samples=3)
    assert [r.tokens for r in many] == [r.tokens for r in one]
    assert len({tuple(r.tokens) for r in many[:3]}) > 1     # numbers of their own
    stop = many[1].tokens[3]
    cut = eng.generate(prompts, max_tokens=20, temperature=0.8, top_k=30, seed=5, stop_ids=[stop], samples=3)
    for c, r in zip(cut, many):
        assert c.tokens == (r.tokens[:r.tokens.index(stop) + 1] if stop in r.tokens else r.tokens)
    eng.cache.check()
    assert not eng.cache.slots.live()
    eng = engine(model_dirs, name, "bfloat16")
    for use_graph in (True, False):
        res = eng.generate(prompts, max_tokens=8, stop_ids=[], samples=4, use_graph=use_graph)
        for i, r in enumerate(res):
            rows = plain_llama.forward(cfg, w, prompts[i // 4] + r.tokens[:-1], storage=torch.bfloat16).numpy()
            rows = rows[len(prompts[i // 4]) - 1:]
            bound = 4e-2 * float(np.abs(rows).max())
            assert all(row.max() - row[t] <= bound for row, t in zip(rows, r.tokens))
    eng.cache.check()
    assert not eng.cache.slots.live()


def test_answers_that_fit_only_because_they_share(model_dirs):
    from cretif_b200.engine import Engine
    eng = Engine(model_dirs["B"], dtype="bfloat16", max_tokens=512)      # eight blocks
    prompt = tiny.tokens("B", 200, 2)
    res = eng.generate([prompt], max_tokens=30, stop_ids=[], samples=5)  # four blocks and one for each of four more
    assert len(res) == 5 and all(len(r.tokens) == 30 for r in res)
    with pytest.raises(ValueError, match="cache holds"):
        eng.generate([prompt], max_tokens=30, stop_ids=[], samples=6)
    with pytest.raises(ValueError, match="answers a prompt"):
        eng.generate([prompt], max_tokens=30, stop_ids=[], samples=65)
    with pytest.raises(ValueError, match="answers a prompt"):
        eng.generate([prompt], max_tokens=30, stop_ids=[], samples=0)
    eng.cache.check()
    assert not eng.cache.slots.live()


def test_refusals(model_dirs):
    from cretif_b200.cache import CacheError
    eng = engine(model_dirs, "B", "bfloat16")
    with pytest.raises(CacheError):
        eng.fork_slot(0)
    a = eng.alloc_slot()
    b = eng.fork_slot(a)[0]                                 # an empty sequence has nothing to share
    assert eng.cache.length(b) == 0 and eng.cache.shared_groups([a, b]) == []
    eng.step([(a, [1, 2, 3]), (b, [1, 2])])
    for bad in (-1, 4):
        with pytest.raises(CacheError):
            eng.truncate_slot(a, bad)
    eng.truncate_slot(a, 0)
    eng.step([(a, [1, 2, 3])])
    eng.cache.check()
