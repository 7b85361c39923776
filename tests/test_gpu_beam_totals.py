"""The order of beams whose totals lie close, on the GPU."""
import math

import pytest

import candidates_model as cm
from gpu_util import need_gpu, say, torch
from moa_amd import ops
from test_gpu_beams import logits_of, run_select
from test_gpu_paged import i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


def select(logits, scores, finished, beams, eos):
    """(scores, finished, parents, tokens) of a call whose results are its next inputs too."""
    s, f = torch.tensor(scores, dtype=torch.float32, device=DEV), i32(finished)
    p, t = torch.full_like(f, -9), torch.full_like(f, -9)
    ops.beam_select(logits, s, f, s, f, p, t, beams=beams, eos=eos)
    assert ops.device_errors() == 0
    return s.tolist(), f.tolist(), p.tolist(), t.tolist()


# places of 7 to 263 small logits beside a row's largest: in its 16 bytes, its thread's, its wave's and its workgroup's
TAILS = {"chunk": [0, 0, 0], "thread": [0, 1, 0], "wave": [0, 0, 31], "block": [0, 0, 255], "both": [0, 1, 100]}


@pytest.mark.parametrize("beams,vocab", [(2, 5000), (2, 262144), (24, 262144)])
@pytest.mark.parametrize("depth", [16.75, 17.0, 18.5, 25.0])
@pytest.mark.parametrize("tail", TAILS)
def test_small_probabilities_decide_between_equal_beams(tail, depth, beams, vocab):
    """All rows but the last hold the same largest logit and beside it a tail of small ones, so the last row's candidate is the best.
    One small exponential is e^-16.75 = 0.89 * 2^-24 at most, nothing beside 1 in f32, and all of a tail together make totals
    that differ by 9e-11 at least. An exponential is off by at most 2^-22 of itself for each unit of its depth and six more, so
    by 2^-17: no tail comes near none. The totals, near 0, are f64."""
    need_gpu()
    say(f"a tail of the {tail} at -{depth}, {beams} beams of {vocab}")
    _, threads, lanes = TAILS[tail]
    at = [i for i in range(1, 8)]
    if threads:  # the same thread's chunks, whether a thread has two or four
        at += [2048 * k + i for k in (1, 2, 3) for i in range(8) if 2048 * k + i < vocab]
    at += [8 * (1 + i) for i in range(lanes) if 8 * (1 + i) < vocab]
    x = torch.full((beams, vocab), -math.inf, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 0.0
    x[:beams - 1, at] = -depth
    assert (torch.exp(x[0].double()).sum() - 1).item() > 9e-11
    scores, finished, parents, tokens = select(x, [-1.0] * beams, [0] * beams, beams, -1)
    assert parents == [beams - 1] + list(range(beams - 1)) and tokens == [0] * beams and finished == [0] * beams
    run_select(x, [-1.0] * beams, [0] * beams, beams, -1)


@pytest.mark.parametrize("shift", [-30.0, 0.0, 1000.0])
def test_beams_of_equal_rows_in_another_order(shift):
    """The same logits at other places give the same sums up to the exponentials' own error: rows whose totals differ by more come in order."""
    need_gpu()
    say(f"permuted rows, largest logit {shift}")
    g = torch.Generator(device=DEV).manual_seed(2)
    row = (torch.randn(50000, generator=g, device=DEV) * 3).to(torch.bfloat16)
    x = torch.stack([row[torch.randperm(50000, generator=g, device=DEV)] for _ in range(6)])
    x = torch.cat([x[:, :7], torch.full_like(x[:, :1], 20.0), x[:, 7:]], 1)
    x = (x.float() + shift).to(torch.bfloat16)
    scores = [-1.0 - 2.0 ** -15 * i for i in range(6)]  # apart by four times the bound of a logarithm
    got = select(x, scores[::-1], [0] * 6, 6, -1)
    assert got[2] == [5, 4, 3, 2, 1, 0] and got[3] == [7] * 6


@pytest.mark.parametrize("score", [-1e30, -3e38, math.inf])
def test_a_rows_logits_keep_their_order_where_totals_are_equal(score):
    """Beside such a score a logit is nothing: totals are equal, and a row's candidates come in the order of its logits."""
    need_gpu()
    x = logits_of(4, 700, 5)
    got = select(x, [score] * 4, [0] * 4, 4, -1)
    order = torch.argsort(x[0].float(), descending=True, stable=True)[:4].tolist()
    assert got[2] == [0] * 4 and got[3] == order and got[0] == [torch.tensor(score, dtype=torch.float32).item()] * 4


def test_scores_of_beams_that_wait():
    """-1e9 for the rows that wait, as some programs write it, in place of -infinity: f64 totals still tell their candidates apart."""
    need_gpu()
    run_select(logits_of(8, 3000, 8), [0.0, -1e9, -1e9, -1e9] * 2, [0] * 8, 4, -1)
    run_select(logits_of(8, 2, 8), [0.0, -1e9, -1e9, -1e9] * 2, [0] * 8, 4, -1)
    assert cm.select(logits_of(4, 2, 8), [0.0, -1e9, -1e9, -1e9], [0] * 4, 4, -1)[2][2] > 0
