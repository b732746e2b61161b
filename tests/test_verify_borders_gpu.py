"""Verification of drafts where little decides: rows that are nearly alike, numbers next to a border."""
import pytest
import torch

from test_verify_drafts_gpu import by_definition, row_probabilities, verify

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
