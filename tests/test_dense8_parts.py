"""How the product of few tiles deals the blocks of k out to the CTAs that share a tile."""
from __future__ import annotations

import ctypes as C

import pytest


CLUSTERS = {2: 74, 4: 33, 8: 15}  # that run at once on a B200


def parts(native, tiles, blocks):
    first = (C.c_uint32 * 9)()
    n = native.tcc_test_product_parts(tiles, blocks, (C.c_uint32 * 3)(*CLUSTERS.values()), first)
    return list(first[:n + 1])


@pytest.mark.parametrize("tiles", [1, 8, 15, 16, 18, 33, 34, 37, 74, 75, 1000])
def test_parts_are_even_groups_of_four_blocks(native, tiles):
    most = max([p for p, count in CLUSTERS.items() if tiles <= count], default=1)
    for blocks in list(range(1, 300)) + [1023, 1024, 1025, 65537, 1 << 24]:
        first = parts(native, tiles, blocks)
        n = len(first) - 1
        assert n <= most and (n == most or blocks < 8 * n)  # all the CTAs that there are SMs and four blocks each for
        assert first[0] == 0 and first[-1] == blocks and all(f % 4 == 0 for f in first[:-1])
        sizes = [b - a for a, b in zip(first, first[1:])]
        assert n == 1 or min(sizes) >= 4
        assert max(sizes) <= -(-(-(-blocks // 4)) // n) * 4  # no more than an even share of the groups


def test_one_more_block_keeps_the_shares(native):
    """33 blocks over eight CTAs are one more for one of them, not 20 and 13 over two."""
    assert parts(native, 8, 32) == [0, 4, 8, 12, 16, 20, 24, 28, 32]
    assert parts(native, 8, 33) == [0, 4, 8, 12, 16, 20, 24, 28, 33]
    assert max(b - a for a, b in zip(parts(native, 8, 65), parts(native, 8, 65)[1:])) <= 12
