"""Verification of drafts where little decides: rows that are nearly alike, numbers next to a border."""
import pytest
import torch

from test_verify_drafts_gpu import by_definition, make, row_probabilities, verify

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


def nearly_alike(B, V, seed, least, most):
    """One draft a sequence, refused; the rows differ in 24 ids, so that from ``least`` to ``most`` of the
    probability is left to draw from.  Every second row's model likes those ids less than the draft's, which leaves
    a little of every other id."""
    gen = torch.Generator().manual_seed(seed)
    logits = 2.0 * torch.randn((2 * B, V), generator=gen)
    draft_logits = logits[::2].clone()
    drafts = torch.zeros((B, 1), dtype=torch.int32)
    for b in range(B):
        ids = torch.randperm(V, generator=gen)[:24]
        mass = float(torch.softmax(logits[2 * b].double(), 0)[ids].sum())
        want = least * (most / least) ** (b / max(1, B - 1))
        step = min(0.5, 2 * want / mass)
        sign = torch.ones(24) if b % 2 else torch.tensor([1.0, -1.0]).repeat(12)
        draft_logits[b, ids] += (step * sign).float()
        drafts[b, 0] = ids[0]
        # (so that one of the ids is refused whatever the step, and little comes of it)
        logits[2 * b, ids[0]] = draft_logits[b, ids[0]] = -6.0 - 4.0 * torch.rand((), generator=gen)
        draft_logits[b, ids[0]] += 0.01
    u = torch.full((B, 2), 1.0 - 2.0 ** -24)
    u[:, 1] = (torch.randint(0, 1 << 24, (B,), generator=gen).float() + 0.5) / (1 << 24)
    u[0, 1], u[1, 1] = 0.0, 1.0 - 2.0 ** -24
    return dict(logits=logits.cuda(), cu=(2 * torch.arange(B + 1)).int().cuda(), drafts=drafts.cuda(),
                draft_logits=draft_logits[:, None].contiguous().cuda(), accept_u=u[:, :1].cuda(),
                next_u=u[:, 1].contiguous().cuda())


@pytest.mark.parametrize("B, V", [(16, 20000), (200, 20000), (16, 49153), (24, 1000)])
@pytest.mark.parametrize("least, most", [(4e-9, 4e-7), (1e-7, 1e-4), (1e-4, 1e-1)])
def test_rows_that_are_nearly_alike(ops, B, V, least, most):
    """Every id is one that the definition may give when the 64-bit sums are off by 1e-12 of a row's."""
    s = nearly_alike(B, V, 5 + B, least, most)
    accepted, tokens = verify(ops, s, 0.9, 0, s["draft_logits"])
    off, drawn = 1e-12, 0
    for b in range(B):
        p = row_probabilities(s["logits"][2 * b].cpu(), 0.9, 0)
        q = row_probabilities(s["draft_logits"][b, 0].cpu(), 0.9, 0)
        rest = (p - q).clamp_min(0.0)
        d, at = int(s["drafts"][b, 0]), 0
        if float(s["accept_u"][b, 0]) * float(q[d]) < float(p[d]):     # (where all other ids got dearer by more)
            rest, at = row_probabilities(s["logits"][2 * b + 1].cpu(), 0.9, 0), 1
        drawn += at == 0
        assert int(accepted[b]) == at
        run = torch.cumsum(rest, 0)
        got = int(tokens[b, at])
        goal = float(s["next_u"][b]) * float(run[-1])
        assert 0 <= got < V and float(run[-1]) > 1e3 * off
        assert float(run[got]) >= goal - off and float(run[got] - rest[got]) <= goal + off, (b, got, float(run[-1]))
        assert float(rest[got]) > -off and tokens[b].tolist() == ([d, got] if at else [got, -1])
    assert drawn >= B // 2


def test_the_same_answers_again(ops):
    """Nothing that is drawn depends on which CTA of a sequence's answers first."""
    s = nearly_alike(64, 20000, 77, 4e-9, 1e-2)
    first = verify(ops, s, 0.9, 0, s["draft_logits"])
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, verify(ops, s, 0.9, 0, s["draft_logits"])))


def at_the_border(B, K, V, seed, temperature, proposed):
    """Every draft's number is within three steps of a 32-bit number of the one at which it no longer stands."""
    gen = torch.Generator().manual_seed(seed)
    logits = 2.5 * torch.randn((B * (K + 1), V), generator=gen)
    draft_logits = logits.view(B, K + 1, V)[:, :K] + 0.5 * torch.randn((B, K, V), generator=gen)
    drafts, u = torch.zeros((B, K), dtype=torch.int32), torch.zeros((B, K))
    for b in range(B):
        for j in range(K):
            p = row_probabilities(logits[b * (K + 1) + j], temperature, 0)
            if proposed:
                q = row_probabilities(draft_logits[b, j], temperature, 0)
                x = int(torch.where(p < 0.95 * q, q, torch.zeros_like(q)).argmax())
                border = p[x] / q[x]
            else:
                x = int(p.argmax())
                border = p[x]
            drafts[b, j] = x
            at = border.float()
            # a third of them just below: they stand, and the next draft is judged
            steps = [-3, -2, -1, 1, 0, 2, -1, 3][int(torch.randint(0, 8, (1,), generator=gen))]
            for _ in range(abs(steps)):
                at = torch.nextafter(at, torch.tensor(2.0 if steps > 0 else -1.0))
            u[b, j] = at
            assert abs(float(at) / float(border) - 1) > 1e-12    # (64-bit sums tell them)
    nu = (torch.randint(0, 1 << 24, (B,), generator=gen).float() + 0.5) / (1 << 24)
    return dict(logits=logits.cuda(), cu=((K + 1) * torch.arange(B + 1)).int().cuda(), drafts=drafts.cuda(),
                draft_logits=draft_logits.contiguous().cuda(), accept_u=u.cuda(), next_u=nu.cuda())


@pytest.mark.parametrize("proposed", [True, False])
@pytest.mark.parametrize("B, K, V, temperature", [(40, 3, 49152, 0.7), (24, 3, 32003, 1.0), (3, 5, 49152, 1.7),
                                                  (200, 2, 1001, 0.3), (16, 3, 151, 1.0)])
def test_numbers_at_the_border(ops, B, K, V, temperature, proposed):
    """A draft is judged as the definition has it however close its number lies."""
    s = at_the_border(B, K, V, B + V, temperature, proposed)
    q = s["draft_logits"] if proposed else None
    accepted, tokens = verify(ops, s, temperature, 0, q)
    want = by_definition(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], temperature, 0, q)
    wrong = int((accepted.cpu() != want[0]).sum())
    assert wrong == 0, f"{wrong} of {B} judged otherwise"
    assert torch.equal(tokens.cpu(), want[1])
    assert len(set(accepted.tolist())) > 1


def test_a_border_behind_a_border_and_infinite_rows(ops):
    """Rows whose largest entries are infinite are uniform over them; a number that is the border itself, exactly,
    does not stand."""
    B, K, V = 4, 2, 4099
    gen = torch.Generator().manual_seed(9)
    logits = torch.randn((B * (K + 1), V), generator=gen)
    draft_logits = torch.randn((B, K, V), generator=gen)
    logits[:, [5, 17, 100, 4000]] = float("inf")
    draft_logits[:, :, [5, 17]] = float("inf")
    drafts = torch.full((B, K), 17, dtype=torch.int32)
    u = torch.full((B, K), 0.5)                            # p = 1/4, q = 1/2
    u[1] = 0.5 - 2.0 ** -25
    u[2, 1] = 0.5 - 2.0 ** -25
    u[3, 0] = 0.5 - 2.0 ** -25
    s = dict(logits=logits.cuda(), cu=((K + 1) * torch.arange(B + 1)).int().cuda(), drafts=drafts.cuda(),
             draft_logits=draft_logits.cuda(), accept_u=u.cuda(), next_u=torch.tensor([0.1, 0.3, 0.6, 0.9]).cuda())
    accepted, tokens = verify(ops, s, 1.0, 0, s["draft_logits"])
    assert accepted.tolist() == [0, 2, 0, 1]
    want = by_definition(s["logits"], s["cu"], s["drafts"], s["accept_u"], s["next_u"], 1.0, 0, s["draft_logits"])
    assert torch.equal(accepted.cpu(), want[0]) and torch.equal(tokens.cpu(), want[1])


@pytest.mark.parametrize("temperature", [0.8, 0.0])
def test_a_top_k_beyond_the_vocabulary_is_none(ops, temperature):
    s = make(6, 3, 2000, [3, 2, 3, 1, 3, 3], seed=21, temperature=temperature, top_k=0)
    want = verify(ops, s, temperature, 0, s["draft_logits"])
    for top_k in (2000, 2001, 2 ** 31, 2 ** 32 + 2, 2 ** 40):
        got = verify(ops, s, temperature, top_k, s["draft_logits"])
        assert all(torch.equal(a, b) for a, b in zip(want, got)), top_k


@pytest.mark.parametrize("proposed", [True, False])
@pytest.mark.parametrize("temperature, top_k", [(0.9, 0), (0.9, 30), (0.0, 0)])
def test_a_draft_outside_the_vocabulary(ops, temperature, top_k, proposed):
    """At a place that is judged it does not stand and sets the fault word, exactly; behind the last draft, or behind
    one that does not stand, it is not looked at."""
    B, K, V = 24, 5, 3001
    counts = [K - b % 3 for b in range(B)]
    s = make(B, K, V, counts, seed=17, temperature=temperature, top_k=top_k, like=0.05)
    if temperature <= 0:                                   # (drafts that are the arg max, some of them)
        cu = s["cu"].tolist()
        best = s["logits"].argmax(-1).int()
        for b in range(B):
            for j in range(counts[b]):
                if (b + j) % 4:
                    s["drafts"][b, j] = best[cu[b] + j]
    q = s["draft_logits"] if proposed else None
    accepted, tokens = (t.cpu() for t in verify(ops, s, temperature, top_k, q))
    judged = behind = 0
    fault = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (V, -1, 2 ** 31 - 1):
        for b in range(B):
            for j in range(K):
                if (b + j + bad) % 3:
                    continue
                t = {**s, "drafts": s["drafts"].clone()}
                t["drafts"][b, j] = bad
                fault.zero_()
                got_a, got_t = (x.cpu() for x in verify(ops, t, temperature, top_k, q, fault))
                others = [i for i in range(B) if i != b]
                assert torch.equal(got_a[others], accepted[others]) and torch.equal(got_t[others], tokens[others])
                if j < counts[b] and j <= int(accepted[b]):
                    assert int(fault.item()) == 1 and int(got_a[b]) == j
                    assert got_t[b, :j].tolist() == s["drafts"][b, :j].tolist() and 0 <= int(got_t[b, j]) < V
                    assert (got_t[b, j + 1:] == -1).all()
                    judged += 1
                else:
                    assert int(fault.item()) == 0
                    assert int(got_a[b]) == int(accepted[b]) and torch.equal(got_t[b], tokens[b])
                    behind += 1
    assert judged > 10 and behind > 10
