"""Verification of drafted tokens against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cretif_b200.csrc import ops
    ops.lib()
    return ops


@pytest.fixture(autouse=True)
def no_fault(ops):
    yield
    assert int(ops.fault_word("cuda").item()) == 0


def row_probabilities(x, temperature, top_k):
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x).double()
    V = x.numel()
    keep = torch.ones(V, dtype=torch.bool)
    if 0 < top_k < V:
        keep[:] = False
        keep[torch.sort(x, descending=True, stable=True).indices[:top_k]] = True
    e = torch.where(x == x.max(), torch.ones_like(x), torch.exp((x - x.max()) / temperature))
    e = torch.where(keep, e, torch.zeros_like(e))
    return e / e.sum()


def by_definition(logits, cu, drafts, accept_u, next_u, temperature, top_k, draft_logits=None):
    logits, drafts, accept_u, next_u = logits.cpu(), drafts.cpu(), accept_u.cpu().double(), next_u.cpu().double()
    draft_logits = None if draft_logits is None else draft_logits.cpu()
    cu = cu.tolist()
    B, K = drafts.shape
    V = logits.shape[1]
    tokens, accepted = torch.full((B, K + 1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        n = cu[b + 1] - cu[b] - 1
        j, rest = 0, None
        while True:
            x = logits[cu[b] + j]
            if temperature <= 0:
                x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
                best = int((x == x.max()).nonzero()[0])
                if j < n and int(drafts[b, j]) == best:
                    j += 1
                    continue
                token = best
                break
            p = row_probabilities(x, temperature, top_k)
            if j == n:
                rest = p
                break
            d = int(drafts[b, j])
            if draft_logits is not None:
                q = row_probabilities(draft_logits[b, j], temperature, top_k)
            else:
                q = torch.zeros(V, dtype=torch.float64)
                if 0 <= d < V:
                    q[d] = 1.0
            if 0 <= d < V and accept_u[b, j] * q[d] < p[d]:
                j += 1
                continue
            rest = (p - q).clamp_min(0.0)
            if not rest.sum() > 0:
                rest = p
            break
        if rest is not None:
            run = torch.cumsum(rest, 0)
            token = int((run <= next_u[b] * run[-1]).sum())
        accepted[b] = j
        tokens[b, :j] = drafts[b, :j]
        tokens[b, j] = token
    return accepted, tokens


def make(B, K, V, counts, seed, temperature, top_k, like=0.8, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n + 1)
    logits = spread * torch.randn((cu[-1], V), generator=gen)
    rows = torch.tensor([[min(cu[b] + j, cu[b + 1] - 1) for j in range(K)] for b in range(B)],
                        dtype=torch.long).view(B, K)
    draft_logits = logits[rows] + like * torch.randn((B, K, V), generator=gen)
    if temperature > 0 and K:
        p = torch.stack([row_probabilities(r, temperature, top_k) for r in draft_logits.view(-1, V)])
        drafts = torch.multinomial(p, 1, generator=gen).view(B, K).int()
    else:
        drafts = draft_logits.argmax(-1).int()
    u = (torch.randint(0, 1 << 24, (B, K + 1), generator=gen).float() + 0.5) / (1 << 24)
    return dict(logits=logits.cuda(), cu=torch.tensor(cu, dtype=torch.int32).cuda(), drafts=drafts.cuda(),
                draft_logits=draft_logits.cuda(), accept_u=u[:, :K].cuda(), next_u=u[:, K].contiguous().cuda())


def verify(ops, s, temperature, top_k, draft_logits=None, fault=None):
    B, K = s["drafts"].shape
    accepted = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tokens = torch.full((B, K + 1), -9, dtype=torch.int32, device="cuda")
    ops.verify_drafts(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], accepted, tokens, temperature,
                      top_k, draft_logits, fault)
    return accepted, tokens


def check(ops, s, temperature, top_k, proposed=True):
    q = s["draft_logits"] if proposed else None
    accepted, tokens = verify(ops, s, temperature, top_k, q)
    want_a, want_t = by_definition(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], temperature, top_k, q)
    assert torch.equal(accepted.cpu(), want_a)
    assert torch.equal(tokens.cpu(), want_t)
    return want_a


@pytest.mark.parametrize("proposed", [True, False])
@pytest.mark.parametrize("temperature, top_k", [(0.0, 0), (0.8, 0), (1.0, 40), (0.3, 1), (1.7, 1000), (0.05, 7)])
@pytest.mark.parametrize("V", [49152, 1001, 1024, 151])
def test_options(ops, V, temperature, top_k, proposed):
    if top_k > V:
        top_k = V
    s = make(5, 4, V, [4, 0, 3, 4, 1], seed=V + top_k, temperature=temperature, top_k=top_k)
    check(ops, s, temperature, top_k, proposed)


@pytest.mark.parametrize("V", [1, 2, 3, 31, 33, 4095, 4097, 50001, 131075])
@pytest.mark.parametrize("top_k", [0, 2])
def test_vocabularies(ops, V, top_k):
    check(ops, make(3, 2, V, [2, 1, 2], seed=V, temperature=0.9, top_k=top_k), 0.9, top_k)
    check(ops, make(3, 2, V, [2, 1, 2], seed=V, temperature=0.0, top_k=0), 0.0, 0)


@pytest.mark.parametrize("B, K", [(1, 1), (1, 12), (2, 0), (70, 3), (300, 1)])
def test_batches(ops, B, K):
    counts = [(b * 7 + K) % (K + 1) for b in range(B)]
    accepted = check(ops, make(B, K, 997, counts, seed=B, temperature=1.0, top_k=0, like=0.3), 1.0, 0)
    if B > 50:
        assert (accepted > 0).any() and (accepted < torch.tensor(counts)).any()


@pytest.mark.parametrize("proposed", [True, False])
@pytest.mark.parametrize("like", [0.02, 0.5])
def test_many_long_rows(ops, like, proposed):
    """Enough rows that the later places wait for the first ones' verdicts: sequences that go on past
    them, that end among them, and that have fewer drafts."""
    B, K, V = 72, 5, 49152
    counts = [(b * 5) % (K + 1) for b in range(B)]
    s = make(B, K, V, counts, seed=int(100 * like), temperature=0.9, top_k=0, like=like)
    accepted = check(ops, s, 0.9, 0, proposed)
    if proposed and like < 0.1:
        assert (accepted >= 3).any()
    s["cu"] = s["cu"].clone()
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    s["drafts"] = s["drafts"].clone()
    s["drafts"][5, 1] = V
    got = verify(ops, s, 0.9, 0, s["draft_logits"] if proposed else None, fault)
    want = by_definition(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], 0.9, 0,
                         s["draft_logits"] if proposed else None)
    rows = [b for b in range(B) if b != 5]
    assert all(torch.equal(g.cpu()[rows], w[rows]) for g, w in zip(got, want))
    assert int(fault.item()) in (0, 1) and int(got[0][5]) <= 1


def test_a_draft_like_the_model_always_stands(ops):
    s = make(16, 4, 2048, [4] * 16, seed=3, temperature=0.7, top_k=0, like=0.0)
    accepted = check(ops, s, 0.7, 0)
    assert (accepted == 4).all()


@pytest.mark.parametrize("V", [151, 5001, 49153])
def test_nothing_left_of_rows_that_are_alike(ops, V):
    # (rows of an odd length begin on other boundaries, so that 32-bit sums of the same numbers differ)
    s = make(6, 3, V, [3, 2, 3, 1, 3, 3], seed=40, temperature=0.8, top_k=0, like=0.0)
    cu = s["cu"].tolist()
    for b in range(6):
        bad = 7 * b + 1                                    # what neither row allows is not a draft that stands
        s["drafts"][b, b % 2] = bad
        s["logits"][cu[b]:cu[b + 1], bad] = float("-inf")
        s["draft_logits"][b, :, bad] = float("-inf")
        s["drafts"][b, 1 - b % 2] = bad + 1
    accepted = check(ops, s, 0.8, 0)
    assert accepted.tolist() == [min(b % 2, n) for b, n in enumerate([3, 2, 3, 1, 3, 3])]


def test_equal_logits_are_kept_by_id(ops):
    """Ties at the top-k border keep the lowest ids; a flat row is uniform."""
    s = make(4, 2, 4096, [2, 2, 1, 0], seed=4, temperature=1.0, top_k=9)
    s["logits"] = (s["logits"] * 1.5).round()
    s["draft_logits"] = (s["draft_logits"] * 1.5).round()
    check(ops, s, 1.0, 9)
    check(ops, s, 1.0, 700)
    s["logits"].zero_()
    s["draft_logits"].fill_(-0.0)
    check(ops, s, 1.0, 9)
    check(ops, s, 1.0, 0, proposed=False)
    check(ops, s, 0.0, 0)


def test_masked_infinite_and_broken_logits(ops):
    s = make(8, 3, 5000, [3] * 8, seed=5, temperature=0.8, top_k=0)
    lowest = torch.finfo(torch.float32).min
    x = s["logits"].view(8, 4, 5000)
    x[0, :, 100:] = float("-inf")
    x[1, :, ::2] = lowest
    x[2, 0] = float("-inf")
    x[3, 1, 77] = float("inf")
    x[3, 1, 99] = float("inf")
    x[4, :, 5] = float("nan")
    x[5, 0] = lowest
    s["draft_logits"][0, :, 50:] = float("-inf")
    s["draft_logits"][6, 0] = float("-inf")
    for t, k in ((0.8, 0), (0.8, 20), (0.0, 0)):
        for proposed in (True, False):
            check(ops, s, t, k, proposed)


def test_the_ends_of_the_unit_interval(ops):
    s = make(6, 2, 3000, [2] * 6, seed=6, temperature=1.0, top_k=0)
    below = 1.0 - 2.0 ** -24
    for a in (0.0, below):
        for n in (0.0, below):
            s["accept_u"] = torch.full_like(s["accept_u"], a)
            s["next_u"] = torch.full_like(s["next_u"], n)
            for k in (0, 50):
                check(ops, s, 1.0, k)


def test_strides(ops):
    s = make(5, 3, 1003, [3, 2, 3, 0, 1], seed=7, temperature=0.8, top_k=0)
    want = verify(ops, s, 0.8, 0, s["draft_logits"])
    wide = torch.full((s["logits"].shape[0], 1009), float("nan"), device="cuda")
    wide[:, 3:1006] = s["logits"]
    q = torch.full((5, 4, 1010), float("nan"), device="cuda")
    q[:, :3, 5:1008] = s["draft_logits"]
    d = torch.full((5, 7), -5, dtype=torch.int32, device="cuda")
    d[:, 2:5] = s["drafts"]
    u = torch.full((5, 9), 7.0, device="cuda")
    u[:, :3] = s["accept_u"]
    t = {**s, "logits": wide[:, 3:1006], "drafts": d[:, 2:5], "accept_u": u[:, :3]}
    got = verify(ops, t, 0.8, 0, q[:, :3, 5:1008])
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_rows_that_lie_over_each_other(ops):
    """One row of logits for every place (expanded tensors) is read as such."""
    s = make(4, 3, 777, [3, 3, 2, 0], seed=13, temperature=0.8, top_k=0)
    row, q = s["logits"][:1], s["draft_logits"][:1, :1]
    t = {**s, "logits": row.expand(s["logits"].shape), "draft_logits": q.expand(4, 3, 777)}
    same = {**s, "logits": t["logits"].contiguous(), "draft_logits": t["draft_logits"].contiguous()}
    for k in (0, 20):
        want = verify(ops, same, 0.8, k, same["draft_logits"])
        got = verify(ops, t, 0.8, k, t["draft_logits"])
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(ops.KernelError):
        ops.verify_drafts(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"],
                          torch.empty(4, dtype=torch.int32, device="cuda"),
                          torch.empty((1, 4), dtype=torch.int32, device="cuda").expand(4, 4), 0.8)


def test_broken_input_sets_the_fault_word(ops):
    s = make(3, 2, 500, [2, 2, 2], seed=8, temperature=0.8, top_k=0)
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (-1, 500, 2 ** 31 - 1):
        for temperature in (0.8, 0.0):
            t = {**s, "drafts": s["drafts"].clone()}
            t["drafts"][1, 0] = bad
            fault.zero_()
            accepted, tokens = verify(ops, t, temperature, 0, s["draft_logits"], fault)
            assert int(fault.item()) == 1 and int(accepted[1]) == 0 and 0 <= int(tokens[1, 0]) < 500
    for rows in ([0, 0, 3, 6], [0, 3, 7, 9], [0, 3, 6, 10], [-1, 2, 5, 8], [0, 3, 2, 5]):
        fault.zero_()
        accepted, tokens = verify(ops, {**s, "cu": torch.tensor(rows, dtype=torch.int32).cuda()}, 0.8, 0,
                                  s["draft_logits"], fault)
        assert int(fault.item()) == 1
        assert any((t == -1).all() for t in tokens)


def test_how_often_ids_are_drawn(ops):
    """Accepted or replaced, the first token is distributed as the model's: over 40,000 sequences every
    id's share is within six standard deviations of its probability."""
    V, N = 12, 40000
    gen = torch.Generator().manual_seed(9)
    p, q = torch.randn(V, generator=gen) * 1.3, torch.randn(V, generator=gen) * 1.3
    drafts = torch.multinomial(torch.softmax(q.double() / 0.9, 0), N, replacement=True, generator=gen)
    s = dict(logits=p.cuda().repeat(2 * N, 1), cu=(2 * torch.arange(N + 1)).int().cuda(), drafts=drafts.int().view(N, 1).cuda(),
             accept_u=torch.rand((N, 1), generator=gen).cuda(), next_u=torch.rand(N, generator=gen).cuda())
    _, tokens = verify(ops, s, 0.9, 0, q.cuda().expand(N, 1, V))
    share = torch.bincount(tokens[:, 0].long().cpu(), minlength=V).double() / N
    want = torch.softmax(p.double() / 0.9, 0)
    assert ((share - want).abs() <= 6 * (want * (1 - want) / N).sqrt()).all()


def test_captured_on_another_stream(ops):
    s = make(6, 3, 4000, [3, 1, 2, 3, 0, 3], seed=10, temperature=0.8, top_k=30)
    want = verify(ops, s, 0.8, 30, s["draft_logits"])
    accepted, tokens = torch.empty_like(want[0]), torch.empty_like(want[1])

    def go():
        ops.verify_drafts(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], accepted, tokens, 0.8, 30,
                          s["draft_logits"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    for _ in range(3):
        accepted.fill_(-9), tokens.fill_(-9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(accepted, want[0]) and torch.equal(tokens, want[1])


def test_the_most_sequences_and_drafts(ops):
    B = 65535
    gen = torch.Generator().manual_seed(31)
    logits = torch.randn((B + 1, 2), generator=gen)
    p0 = torch.softmax(logits.double() / 0.7, dim=-1)[:, 0]
    u = torch.rand(B + 1, generator=gen)
    u = torch.where((u.double() - p0).abs() < 1e-3, torch.zeros_like(u), u)     # (away from the border)

    def step(n):
        return dict(logits=logits[:n].cuda(), cu=torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                    drafts=torch.zeros((n, 0), dtype=torch.int32, device="cuda"),
                    accept_u=torch.zeros((n, 0), device="cuda"), next_u=u[:n].cuda())
    for temperature, top_k, want in ((0.7, 0, u.double() >= p0), (0.7, 1, logits[:, 1] > logits[:, 0]),
                                     (0.0, 0, logits[:, 1] > logits[:, 0])):
        accepted, tokens = verify(ops, step(B), temperature, top_k)
        assert torch.equal(tokens.cpu()[:, 0], want[:B].int()) and not accepted.any()
        with pytest.raises(ops.KernelError):
            verify(ops, step(B + 1), temperature, top_k)
    for K, fits in ((8191, True), (8192, False)):
        logits = torch.tensor([0.0, 40.0, 1.0]).repeat(K + 1, 1)
        drafts = torch.ones((1, K), dtype=torch.int32)
        drafts[0, 8000] = 0
        s = dict(logits=logits.cuda(), cu=torch.tensor([0, K + 1], dtype=torch.int32, device="cuda"),
                 drafts=drafts.cuda(), accept_u=torch.full((1, K), 0.5, device="cuda"),
                 next_u=torch.full((1,), 0.5, device="cuda"))
        for temperature, top_k in ((1.0, 0), (1.0, 2), (0.0, 0)):
            if not fits and not top_k and temperature:
                with pytest.raises(ops.KernelError):
                    verify(ops, s, temperature, top_k)
                continue
            accepted, tokens = verify(ops, s, temperature, top_k)
            assert accepted.tolist() == [8000]
            assert (tokens[0, :8001] == 1).all() and (tokens[0, 8001:] == -1).all()


def test_verifier_class(ops):
    from cretif_b200.sampling import DraftVerifier, SamplingParams
    s = make(4, 3, 300, [3, 2, 3, 3], seed=11, temperature=0.6, top_k=25)
    want = verify(ops, s, 0.6, 25, s["draft_logits"])
    accepted, tokens = torch.empty_like(want[0]), torch.empty_like(want[1])
    v = DraftVerifier(SamplingParams(0.6, 25), 300)
    assert v(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], accepted, tokens,
             draft_logits=s["draft_logits"]) is tokens
    assert torch.equal(accepted, want[0]) and torch.equal(tokens, want[1])
    with pytest.raises(ValueError):
        v(s["logits"][:, :299], s["cu"], s["drafts"], s["accept_u"], s["next_u"], accepted, tokens)
    with pytest.raises(ValueError):
        DraftVerifier(SamplingParams(0.6, -1), 300)


def test_refusals(ops):
    s = make(3, 2, 5000, [2, 2, 2], seed=12, temperature=0.8, top_k=0)
    good = dict(logits=s["logits"], cu_rows=s["cu"], drafts=s["drafts"], accept_u=s["accept_u"], next_u=s["next_u"],
                accepted=torch.empty(3, dtype=torch.int32, device="cuda"),
                tokens=torch.empty((3, 3), dtype=torch.int32, device="cuda"), temperature=0.8, top_k=0,
                draft_logits=s["draft_logits"])
    ops.verify_drafts(**good)
    bad = [dict(logits=s["logits"].bfloat16()), dict(logits=s["logits"].t()), dict(logits=s["logits"][0]),
           dict(cu_rows=s["cu"][:3]), dict(cu_rows=s["cu"].long()), dict(drafts=s["drafts"].long()),
           dict(drafts=s["drafts"][:2]), dict(accept_u=s["accept_u"][:, :1]), dict(accept_u=s["accept_u"].double()),
           dict(next_u=s["next_u"][:2]), dict(accepted=good["accepted"][:2]), dict(tokens=good["tokens"][:, :2]),
           dict(tokens=good["tokens"].long()), dict(temperature=float("nan")), dict(top_k=-1), dict(top_k=1025),
           dict(draft_logits=s["draft_logits"][:, :1]), dict(draft_logits=s["draft_logits"].bfloat16()),
           dict(draft_logits=s["draft_logits"].transpose(1, 2).contiguous().transpose(1, 2)),
           dict(logits=s["logits"].cpu()), dict(next_u=s["next_u"].cpu()), dict(logits=s["logits"][:0])]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.verify_drafts(**{**good, **change})
    torch.cuda.synchronize()
