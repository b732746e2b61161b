"""Which kernel a step of forked sequences takes, against what both were measured to take."""
import pytest

from cretif_b200.parts import attention

# heads, key/value heads, head size, sequences on a prefix, its tokens, own tokens, new ones, us shared, us ordinary
MEASURED = [
    (16, 2, 128, 8, 64, 60, 1, 4.7, 12.9),
    (16, 2, 128, 32, 64, 60, 1, 6.2, 16.4),
    (16, 2, 128, 32, 256, 60, 1, 8.2, 17.9),
    (16, 2, 128, 32, 2048, 60, 1, 14.2, 28.5),
    (32, 32, 64, 32, 64, 60, 1, 10.0, 17.4),
    (32, 32, 64, 8, 2048, 60, 1, 10.6, 26.2),
    (32, 32, 64, 64, 8000, 150, 1, 33.8, 500.0),
    (9, 3, 64, 32, 2048, 60, 1, 8.4, 11.6),
    (9, 3, 64, 8, 256, 60, 1, 5.5, 4.5),
    (9, 3, 64, 8, 512, 60, 1, 6.7, 4.9),
    (9, 3, 64, 2, 1024, 60, 1, 6.9, 4.6),
    (16, 2, 128, 4, 512, 60, 1, 11.4, 7.3),
    (16, 2, 128, 4, 1024, 60, 1, 12.1, 8.1),
    (32, 32, 64, 2, 512, 60, 1, 8.2, 5.7),
    (16, 2, 128, 2, 512, 60, 1, 9.8, 7.0),
    (9, 3, 64, 8, 2048, 60, 4, 10.2, 22.9),
    (9, 3, 64, 2, 64, 60, 4, 4.3, 5.7),
    (32, 32, 64, 32, 512, 60, 4, 17.2, 84.2),
    (16, 2, 128, 32, 512, 60, 4, 19.3, 53.9),
    (16, 2, 128, 2, 2048, 60, 4, 18.0, 35.5),
    (32, 2, 64, 2, 64, 30, 1, 3.5, 18.0),
    (20, 2, 32, 8, 64, 30, 1, 3.2, 12.6),
    (20, 2, 32, 2, 512, 1000, 1, 9.8, 57.5),
    (24, 2, 128, 2, 4096, 4000, 1, 18.5, 827.5),
    (16, 16, 128, 3, 448, 30, 16, 15.0, 11.3),
    (16, 16, 128, 6, 320, 10, 8, 12.8, 10.0),
    (32, 8, 128, 4, 320, 60, 3, 12.4, 10.1),
    (16, 1, 128, 6, 384, 30, 16, 16.9, 12.0),
]


@pytest.mark.parametrize("row", MEASURED, ids=str)
def test_the_faster_one_is_taken(row):
    nh, nkv, hd, B, prefix, own, new, shared, ordinary = row
    assert max(shared, ordinary) > 1.2 * min(shared, ordinary)      # (what is tabled is clear)
    got = attention.shared_pays([(list(range(B)), prefix)], [new] * B, [prefix + own] * B, nh, nkv, hd)
    assert got == (shared < ordinary)


@pytest.mark.parametrize("nh, nkv, hd, members, prefix, own", [
    (16, 16, 128, 3, 4800, 5657),        # 91 and 146
    (32, 32, 64, 2, 15040, 12018),       # 50 and 67
    (32, 32, 64, 3, 576, 1728),          # 18 and 26
])
def test_long_own_keys_go_to_the_ordinary_kernel(nh, nkv, hd, members, prefix, own):
    B = members + 4
    starts = [prefix + own // 2 if b < members else own for b in range(B)]
    assert not attention.shared_pays([(list(range(members)), prefix)], [1] * B, starts, nh, nkv, hd)
    # while the answers are short, it pays
    short = [prefix + 5] * members
    if prefix > 1000:
        assert attention.shared_pays([(list(range(members)), prefix)], [1] * members, short, nh, nkv, hd)


def test_nothing_to_spare_is_nothing_gained():
    assert not attention.shared_pays([([0], 4096)], [1, 1], [4096, 10], 9, 3, 64)
    assert not attention.shared_pays([([0], 4096), ([1], 640)], [1, 1], [4096, 700], 16, 2, 128)
