"""A long prefix of two sequences beside many that share nothing: outputs, and the memory that a call takes."""
import pytest
import torch

from shared_prefix_tools import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cretif_b200.csrc import ops
    ops.lib()
    return ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("new, own", [(1, 5), (1, 1100), (4, 30)])
@pytest.mark.parametrize("heads", [(8, 2, 64), (16, 2, 128)], ids=str)
def test_two_of_many(ops, heads, new, own, dtype):
    B = 12
    s = Step([([7, 3], 2560), ([0, 5, 9], 384)], own=[own + b for b in range(B)], news=[1 + b % new for b in range(B)],
             nh=heads[0], nkv=heads[1], hd=heads[2], dtype=dtype, seed=new + own)
    s.check(ops)
    assert int(ops.fault_word("cuda").item()) == 0


def test_memory_of_a_call(ops):
    nh, nkv, hd, B, new = 32, 1, 128, 64, 16
    s = Step([([0, 1], 9984)], own=[3 + b for b in range(B)], news=[new] * B, nh=nh, nkv=nkv, hd=hd,
             dtype=torch.bfloat16, seed=2)
    plan = s.plan(ops)
    out = torch.empty((s.T, nh * hd), dtype=torch.bfloat16, device="cuda")
    s.run(ops, plan, out=out)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    s.run(ops, plan, out=out)
    torch.cuda.synchronize()
    took = torch.cuda.max_memory_allocated() - before
    # two sequences' 16 tokens with a piece for every 64 keys at the very most
    assert took <= 2 * new * (9984 // 64 + 1) * nh * (hd + 2) * 4 + (1 << 20)
