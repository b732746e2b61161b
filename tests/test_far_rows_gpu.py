"""Rows that lie more than 2^31 numbers apart: the operators give what they give on rows that lie together."""
import pytest
import torch

from shared_prefix_tools import Step
from test_verify_drafts_gpu import make, verify

pytestmark = pytest.mark.gpu

APART = (1 << 31) + 64


@pytest.fixture(scope="module")
def ops():
    from cretif_b200.csrc import ops
    ops.lib()
    return ops


@pytest.fixture(scope="module")
def far():
    """One storage of 8.6 GB, of which the tests take views; released behind them."""
    base = torch.empty(APART + (1 << 20), dtype=torch.float32, device="cuda")
    yield base
    del base
    torch.cuda.empty_cache()


def spread(base, t, at, apart=APART):
    """``t`` [2, n], its second row ``apart`` numbers behind the first, ``at`` numbers into the storage."""
    view = base.view(t.dtype).as_strided(t.shape, (apart, 1), at)
    view.copy_(t)
    return view


@pytest.mark.parametrize("temperature, top_k", [(0.0, 0), (0.8, 0), (0.8, 9)])
def test_verification(ops, far, temperature, top_k):
    V = 5000
    s = make(2, 1, V, [0, 0], seed=3, temperature=temperature, top_k=top_k)
    two = {**s, "logits": spread(far, s["logits"], 0)}      # two sequences of no drafts, a row each
    # sequences of one draft each: their places lie apart in turn
    one = make(2, 1, V, [1, 1], seed=4, temperature=temperature, top_k=top_k)
    apart = {**one, "drafts": spread(far, one["drafts"], 100_000), "accept_u": spread(far, one["accept_u"], 200_000)}
    for a, b in ((s, two), (one, apart)):
        want = verify(ops, a, temperature, top_k, a["draft_logits"])
        accepted = torch.full((2,), -9, dtype=torch.int32, device="cuda")
        tokens = spread(far, torch.full((2, 2), -9, dtype=torch.int32, device="cuda"), 300_000)
        ops.verify_drafts(b["logits"], b["cu"], b["drafts"], b["accept_u"], b["next_u"], accepted, tokens, temperature,
                          top_k, b["draft_logits"])
        assert torch.equal(accepted, want[0]) and torch.equal(tokens, want[1])
    assert int(ops.fault_word("cuda").item()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("prefix", [64, 1024])
def test_attention(ops, far, dtype, prefix):
    s = Step([([0, 1], prefix)], [70, 3], [1, 1], 4, 2, 64, dtype, seed=5)
    want = s.check(ops)[:2]
    apart = APART                                          # (in bfloat16 the storage holds twice as many)
    s.q = spread(far, s.q.contiguous(), 0, apart)
    out = spread(far, torch.full_like(want, 7.0), 100_000, apart)
    got = s.run(ops, out=out)
    assert torch.equal(got, want)
    # (tables of two slots: the sequences' own are brought there)
    rows = s.table[s.seq_slot.long()].contiguous()
    s.table, s.seq_slot = spread(far, rows, 300_000, apart), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    assert torch.equal(s.run(ops, out=out), want)
    assert int(ops.fault_word("cuda").item()) == 0


def test_one_row_may_have_any_stride(ops):
    """A tensor of one row carries whatever stride its making gave it."""
    s = make(1, 0, 999, [0], seed=6, temperature=0.8, top_k=0)
    want = verify(ops, s, 0.8, 0)
    row = s["logits"].as_strided((1, 999), (3_000_000_000, 1))
    assert all(torch.equal(a, b) for a, b in zip(want, verify(ops, {**s, "logits": row}, 0.8, 0)))
