"""Beams whose totals lie at the end of f32, on the GPU."""
import math

import pytest

from gpu_util import need_gpu, torch
from test_gpu_beam_totals import select

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOWEST = torch.finfo(torch.bfloat16).min


def test_a_total_that_rounds_to_minus_infinity_is_none():
    """Two steps over rows whose mask is the type's lowest value: twice that is a finite f64, but no score."""
    need_gpu()
    x = torch.full((4, 2), LOWEST, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 0.0
    low = float(torch.tensor(LOWEST))
    got = select(x, [0.0] + [-math.inf] * 3, [0] * 4, 4, 1)
    assert got == ([0.0, low, -math.inf, -math.inf], [0, 1, 1, 1], [0, 0, 2, 3], [0, 1, 1, 1])
    got = select(x, got[0], [0] * 4, 4, -1)
    assert got == ([0.0, low, low, -math.inf], [0, 0, 0, 1], [0, 0, 1, 3], [0, 1, 0, 0])
    got = select(x, got[0], got[1], 4, 0)
    assert got[0] == [0.0, low, low, low] and got[2] == [0, 0, 1, 2] and got[3] == [0, 1, 0, 0]
    # of each row all totals but one are too low
    x[:] = LOWEST
    x[:, 0] = 3e38
    got = select(x, [low] * 4, [0] * 4, 4, -1)
    assert got[0] == [low] * 4 and got[2] == [0, 1, 2, 3] and got[3] == [0] * 4
    y = torch.full((4, 4), LOWEST, dtype=torch.bfloat16, device=DEV)
    y[:, 2] = 3e38
    got = select(y[:1].contiguous(), [low], [0], 1, 2)
    assert got == ([low], [1], [0], [2])


def test_the_lowest_total_that_is_a_score():
    """f32's lowest number, and what rounds to it, are scores; half a step of f32 further down rounds to -infinity."""
    need_gpu()
    top = -3.4028234663852886e38                      # f32's lowest number; its step is 2^104
    x = torch.full((3, 1), 0.0, dtype=torch.bfloat16, device=DEV)
    got = select(x, [top] * 3, [0] * 3, 3, -1)        # one token: its probability is 1
    assert got == ([top] * 3, [0] * 3, [0, 1, 2], [0] * 3)
    for below, is_score in ((-2.0 ** 101, True), (-2.0 ** 102, True), (-2.0 ** 103, False), (-2.0 ** 104, False)):
        x = torch.full((2, 2), below, dtype=torch.bfloat16, device=DEV)
        x[:, 0] = 0.0
        got = select(x, [top, -math.inf], [0, 0], 2, -1)
        want = ([top, top], [0, 0], [0, 0], [0, 1]) if is_score else ([top, -math.inf], [0, 1], [0, 1], [0, 0])
        assert got == want, below
