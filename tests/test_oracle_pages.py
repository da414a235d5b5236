"""The oracle of the 4-bit codes and of the page pool, pinned to values worked out by hand (no GPU)."""
import math

import pytest
import torch

from oracle import pages as P


def row(*values):
    return torch.tensor(list(values) + [0.0] * (32 - len(values)))


def test_codes():
    codes = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    x = P.decode(codes, torch.full((256, 1), 128, dtype=torch.uint8))
    assert x[0x71, 0] == 1.0 and x[0x71, 1] == 12.0 and x[0xF9, 0] == -1.0 and x[0xF9, 1] == -12.0 and x[0x2A, 0] == -2.0
    assert torch.isnan(P.decode(codes[:1].repeat(1, 2), torch.tensor([[127, 255]], dtype=torch.uint8))).all()


@pytest.mark.parametrize("largest,scale", [(6.0, 0), (7.0, 0), (7.03125, 1), (12.0, 1), (14.0, 1), (3.5, -1), (3.0, -1), (1.0, -2), (1.75, -2), (1.7578125, -1)])
def test_scales(largest, scale):
    assert P.exponents(row(0.1, -largest).bfloat16()).item() == scale


def test_limits_of_scales():
    assert P.exponents(row(65504.0).half()).item() == 13 and P.exponents(row(torch.finfo(torch.bfloat16).max).bfloat16()).item() == 125
    assert P.exponents(row(0.0).bfloat16()).item() == -125 and P.exponents(row(2.0**-133).bfloat16()).item() == -125
    assert P.exponents(row(2.0**-24).half()).item() == -26


def test_rounding():
    x = row(6.0, 0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 2.6, 3.5, 3.4, 5.0, 5.1, -0.75, -2.5, -0.2, 6.5).half()
    got, scale = P.encode(x)
    assert got[:17].tolist() == [6, 0, 0.5, 1, 0.5, 1, 2, 2, 3, 4, 3, 4, 6, -1, -2, 0, 6] and scale.tolist() == [127]
    got, scale = P.encode(torch.cat((x, row(math.inf).half())))
    assert torch.isnan(got).all() and scale.tolist() == [255, 255]


def test_pool():
    pool = P.Pool([[7, -1, -1], [-1] * 3, [-1] * 3], [3, 0, 0], [5, 1, 4, 9, -1], 4, 4)
    starts, positions, slots, granted = pool.extend([2, 4, 1], 8)
    assert starts == [0, 2, 6, 7] and positions == [3, 4, 0, 1, 2, 3, 0, 0] and granted == [True] * 3
    assert slots == [31, 36, 16, 17, 18, 19, 4, -1] and pool.table == [[7, 9, -1], [4, -1, -1], [1, -1, -1]] and pool.left == 1
    pool.truncate([3, 0, 0])
    assert pool.lengths == [3, 0, 0] and pool.left == 4 and pool.free == [5, 1, 4, 9, -1] and pool.table == [[7, -1, -1], [-1] * 3, [-1] * 3]
    # four pages for the second one of which three columns hold; five for the third and fourth, of which there are four
    pool = P.Pool([[-1] * 3] * 4, [0] * 4, list(range(4)), 4, 4)
    starts, positions, slots, granted = pool.extend([4, 13, 9, 5], 100)
    assert granted == [True, False, True, False] and pool.left == 0 and pool.lengths == [4, 0, 9, 0]
    # a sequence that needs no page is served behind one that lacks them; tokens beyond max_tokens are not
    pool = P.Pool([[0, -1], [-1, -1], [1, -1], [2, -1]], [2, 0, 1, 3], [3], 0, 4)
    starts, positions, slots, granted = pool.extend([1, 1, 2, 1], 4)
    assert granted == [True, False, True, False] and starts == [0, 1, 2, 4, 4] and slots == [2, -1, 5, 6] and pool.lengths == [3, 0, 3, 3]
