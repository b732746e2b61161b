"""The host side of a shared-prefix plan: every row meets every key it sees exactly once."""
import pytest
import torch

from cretif_b200.csrc import ops


def walk(groups, news, starts, nh, nkv, tile_rows, own_rows, ctas, whole=False):
    pre, own, splits, pieces, rows, tok_pieces, prefix = ops._shared_items(
        groups, news, starts, nh, nkv, 64, tile_rows, own_rows, ctas, whole)
    g = nh // nkv
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    tok_seq = [b for b in range(len(news)) for _ in range(news[b])]
    seen = {}
    for i in range(0, len(pre), 8):
        base, row0, n, member, b0, b1, piece, _ = pre[i:i + 8]
        assert 0 < n <= tile_rows and b0 < b1
        for r in range(row0, row0 + n):
            t = rows[base + r // g]
            assert piece < tok_pieces[t] <= pieces - splits
            assert prefix[tok_seq[t]] == prefix[member]
            for blk in range(b0, b1):
                key = (t, r % g, blk)
                assert key not in seen
                seen[key] = piece
    for t, b in enumerate(tok_seq):
        assert cu[b] <= t < cu[b + 1]
        for h in range(g):
            for blk in range(0 if whole else prefix[b] // 64):
                assert (t, h, blk) in seen
    assert len(seen) == (0 if whole else g * sum(prefix[b] // 64 * news[b] for b in range(len(news))))
    mine = set()
    for i in range(0, len(own), 8):
        b, tok0, row0, n, shared, mine_pieces, least, _ = own[i:i + 8]
        assert 0 < n <= own_rows and tok0 == cu[b] and shared == (0 if whole else prefix[b]) and least == prefix[b]
        assert all(tok_pieces[t] == mine_pieces for t in range(cu[b], cu[b + 1]))
        for r in range(row0, row0 + n):
            assert (b, r) not in mine
            mine.add((b, r))
    assert len(mine) == g * sum(news)
    return pre, own, splits, pieces


@pytest.mark.parametrize("tile_rows, own_rows", [(32, 32), (128, 16)])
@pytest.mark.parametrize("ctas", [1, 7, 296])
def test_every_row_meets_every_key_once(tile_rows, own_rows, ctas):
    walk([([0, 3, 1], 640), ([2, 5], 64)], [1, 4, 2, 1, 1, 9], [700, 640, 64, 641, 9, 100], 12, 4, tile_rows, own_rows,
         ctas)
    walk([(list(range(50)), 1024)], [1 + b % 3 for b in range(50)], [1024 + b for b in range(50)], 9, 3, tile_rows,
         own_rows, ctas)
    walk([], [1, 2], [0, 5], 4, 1, tile_rows, own_rows, ctas)
    walk([([0, 2], 128), ([1], 64)], [1, 2, 1], [128, 70, 140], 4, 1, tile_rows, own_rows, ctas, whole=True)
    walk([([0], 0), ([1], 64)], [1, 2], [0, 64], 4, 1, tile_rows, own_rows, ctas)


def test_items_fill_the_chip_without_going_far_beyond_it():
    for batch, blocks in ((2, 3), (8, 31), (64, 125), (64, 469)):
        pre, *_ = walk([(list(range(batch)), 64 * blocks)], [1] * batch, [64 * blocks] * batch, 9, 3, 32, 32, 296)
        tiles = -(-batch * 3 // 32)
        assert len(pre) // 8 * 3 <= max(296, 3 * tiles)


def test_refusals():
    plan = ops.shared_prefix_plan
    ok = dict(groups=[([0, 1], 64)], news=[1, 1], starts=[64, 70], nh=4, nkv=2, hd=64, dtype=torch.bfloat16,
              device="cpu")
    assert plan(**ok).T == 2
    for change in (dict(groups=[([0, 1], 65)]), dict(groups=[([0, 1], -64)]), dict(groups=[([0, 2], 64)]),
                   dict(groups=[([0, -1], 64)]), dict(groups=[([0], 64), ([0, 1], 64)]), dict(groups=[([0, 0], 64)]),
                   dict(groups=[([0, 1], 128)]), dict(news=[1, 0]), dict(news=[]), dict(starts=[64]),
                   dict(starts=[64, -1]), dict(nh=3), dict(nkv=0), dict(hd=72), dict(hd=144), dict(hd=0),
                   dict(dtype=torch.float16)):
        with pytest.raises(ops.KernelError):
            plan(**{**ok, **change})


def test_cpu_tensors_are_refused():
    plan = ops.shared_prefix_plan([([0, 1], 64)], [1, 1], [64, 70], 4, 2, 64, torch.float32, "cpu")
    z = torch.zeros
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.attn_shared(z(2, 256), z(2, 256), z(4, 2, 64, 64), z(4, 2, 64, 64), z(2, 4, dtype=torch.int32),
                        z(2, dtype=torch.int32), z(3, dtype=torch.int32), z(2, dtype=torch.int32), plan, 0.125, 64,
                        z(1, dtype=torch.int32))


def test_numbers_in_any_kind_of_sequence():
    want = ops.shared_prefix_plan([([0, 1], 512)], [1, 3], [512, 600], 4, 2, 64, torch.bfloat16, "cpu")
    for kind in (tuple, iter, torch.tensor):
        got = ops.shared_prefix_plan(iter([(kind([0, 1]), torch.tensor(512))]), kind([1, 3]), kind([512, 600]), 4, 2,
                                     64, torch.bfloat16, "cpu")
        assert torch.equal(got.data, want.data) and got.launch == want.launch
