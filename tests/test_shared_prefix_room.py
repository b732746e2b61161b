"""The room that a call's pieces take: as many as its tokens have, however few of them share a long prefix."""
import pytest
import torch

from cretif_b200.csrc import ops


@pytest.mark.parametrize("nh, nkv, hd", [(32, 1, 128), (32, 8, 128), (32, 8, 64), (9, 3, 64)])
@pytest.mark.parametrize("B, new", [(64, 16), (256, 16), (64, 1)])
def test_strangers_beside_a_long_prefix_cost_nothing(nh, nkv, hd, B, new):
    long, dtype = 30016, torch.bfloat16
    groups = [([0, 1], long)]
    starts = [long + 5, long + 70] + [40 + b % 50 for b in range(B - 2)]
    plan = ops.shared_prefix_plan(groups, [new] * B, starts, nh, nkv, hd, dtype, "cpu")
    alone = ops.shared_prefix_plan(groups, [new] * 2, starts[:2], nh, nkv, hd, dtype, "cpu")
    splits = plan.launch[3]
    # the two sequences' pieces (not more than by themselves have any: 148 SMs), and own ones where they are cut
    most = 2 * new * 300 + (B * new * splits if splits > 1 else 0)
    assert plan.pieces <= most and alone.pieces <= 2 * new * 300 + 2 * new * 8
    assert plan.pieces * nh * (hd + 2) * 4 <= 170 << 20


def test_the_pieces_lie_one_behind_the_other():
    groups, news = [([4, 1], 1280), ([0, 3], 320)], [2, 1, 3, 1, 2]
    starts = [330, 1300, 9, 320, 1290]
    for dtype in (torch.bfloat16, torch.float32):
        plan = ops.shared_prefix_plan(groups, news, starts, 8, 2, 64, dtype, "cpu")
        n_pre, n_own, _, splits, n_rows, T = plan.launch[:6]
        data = plan.data.tolist()
        own = [data[8 * i:8 * i + 8] for i in range(n_pre, n_pre + n_own)]
        rows = data[8 * (n_pre + n_own):][:n_rows]
        rows_first = data[8 * (n_pre + n_own) + n_rows:][:n_rows]
        first = data[8 * (n_pre + n_own) + 2 * n_rows:]
        kept = 0 if dtype == torch.bfloat16 and splits == 1 else splits
        assert len(first) == T + 1 and first[0] == 0 and first[-1] == plan.pieces
        assert [first[t] for t in rows] == rows_first
        cu = [0, 2, 3, 6, 7, 9]
        for seq, tok0, row0, n, prefix, pieces, least, at in own:
            assert tok0 == cu[seq] and at == first[tok0]
            assert all(first[t + 1] - first[t] == pieces + kept for t in range(cu[seq], cu[seq + 1]))
        for i in range(n_pre):
            base, row0, n, seq, b0, b1, piece, _ = data[8 * i:8 * i + 8]
            for r in range(row0, row0 + n):
                t = rows[base + r // 4]
                assert first[t] + piece < first[t + 1] - kept
