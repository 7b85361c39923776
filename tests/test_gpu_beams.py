"""Beam search over the paged cache on the GPU: the selection against a float64 evaluation, the reordering of the sequences against
a plain model, and steps of them together."""
import math

import pytest

import candidates_model as cm
import paged_model as pm
from gpu_util import need_gpu, torch
from moa_amd import _lib, ops
from test_gpu_paged import Setup, i32, raw

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run_select(logits, scores, finished, beams, eos):
    n = logits.shape[0]
    s, f = torch.tensor(scores, dtype=torch.float32, device=DEV), i32(finished)
    so, fo, p, t = torch.full_like(s, 9.0), torch.full_like(f, 9), torch.full_like(f, -9), torch.full_like(f, -9)
    ops.beam_select(logits, s, f, so, fo, p, t, beams=beams, eos=eos)
    assert ops.device_errors() == 0
    want = cm.select(logits, s.tolist(), finished, beams, eos)
    assert p.tolist() == want[2] and t.tolist() == want[3] and fo.tolist() == want[1]
    check_scores(so, want[0])
    ops.beam_select(logits, s, f, s, f, p, t, beams=beams, eos=eos)  # in place
    assert torch.equal(s, so) and torch.equal(f, fo) and n == s.numel()


def check_scores(got, want):
    """A score is rounded once: 2^-24 of it. The log of the sum: its terms are f32 exponentials of rounded arguments, 2^-23 of a
    term plus 2^-24 of an argument below 2^5 for all that count, its sums of at most 64 terms a lane and 8 across add
    2^-18 in all: the logarithm moves by at most 2^-17."""
    for a, b in zip(got.tolist(), want):
        assert a == b or abs(a - b) <= 2.0 ** -17 + 2.0 ** -24 * abs(b), (a, b)


def logits_of(rows, vocab, seed=0, spread=4.0, stride=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn((rows, stride or vocab), generator=g, device=DEV) * spread).to(torch.bfloat16)
    return x[:, :vocab]


def scores_of(rows, seed=0):
    r = cm.rng(seed)
    return [-8.0 * r.random() for _ in range(rows)]


@pytest.mark.parametrize("vocab", [1, 3, 8, 63, 64, 65, 1000, 4096, 32003, 100001, 262144, 1 << 20])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 5), (2, 64)])
def test_select_takes_the_best(groups, beams, vocab):
    need_gpu()
    if vocab > 200000 and beams == 64:
        groups = 1
    n = groups * beams
    r = cm.rng(vocab + beams)
    finished = [int(r.random() < 0.2) for _ in range(n)]
    run_select(logits_of(n, vocab, vocab), scores_of(n, beams), finished, beams, r.randrange(-1, vocab))


@pytest.mark.parametrize("stride", [999, 1000, 1003, 1016])
def test_select_of_rows_that_lie_apart(stride):
    need_gpu()
    x = logits_of(24, 999, 3, stride=stride)
    if stride > 999:
        torch.as_strided(x, (24, stride - 999), (stride, 1), 999).fill_(1000.0)  # not the rows'
    run_select(x, scores_of(24), [0] * 24, 8, 5)


def test_select_of_many_rows():
    need_gpu()
    run_select(logits_of(1200, 3001, 4), scores_of(1200), [0] * 1200, 12, 7)
    run_select(logits_of(64, 70000, 5), scores_of(64), [1] * 63 + [0], 16, 7)


def test_select_from_one_living_beam():
    """The first step: all but one beam of a group at -infinity."""
    need_gpu()
    run_select(logits_of(12, 5000, 6), [0.0, -math.inf, -math.inf, -math.inf] * 3, [0] * 12, 4, 2)


@pytest.mark.parametrize("vocab", [70, 9000])
def test_select_of_ties(vocab):
    """Equal logits and equal beams: the lowest row, then the lowest token."""
    need_gpu()
    x = torch.zeros((8, vocab), dtype=torch.bfloat16, device=DEV)
    x[:, 1::3] = -0.0
    run_select(x, [-1.0] * 8, [0] * 8, 8, -1)
    x = logits_of(1, vocab, 7).repeat(6, 1)
    run_select(x, [-2.0] * 6, [0] * 6, 6, -1)
    x = torch.full((4, vocab), -3.0, dtype=torch.bfloat16, device=DEV)
    x[:, vocab - 5:] = 1.0
    run_select(x, [-2.0, -1.0, -2.0, -1.0], [0] * 4, 4, -1)


@pytest.mark.parametrize("vocab", [40, 20000])
@pytest.mark.parametrize("beams", [2, 6, 33])
def test_select_of_masked_logits(beams, vocab):
    """Rows whose mask leaves fewer tokens than beams, or none; masks of -infinity and of the type's lowest value; NaN and +infinity."""
    need_gpu()
    n = 4 * beams
    x = logits_of(n, vocab, beams)
    lowest = torch.finfo(torch.bfloat16).min
    keep = x[:, [3, vocab - 1]].clone()
    x[:beams] = -math.inf                       # group 0: one beam has two tokens, the others none
    x[1, [3, vocab - 1]] = keep[1]
    x[beams:2 * beams] = lowest                 # group 1: the lowest value is a number
    x[beams, [3, vocab - 1]] = keep[beams]
    x[2 * beams, 7] = float("nan")              # group 2: rows of no candidates beside good ones
    x[2 * beams + 1, 8] = math.inf
    x[3 * beams:, ::2] = -math.inf
    x[4 * beams - 1] = float("nan")
    run_select(x, scores_of(n), [0] * n, beams, 3)
    run_select(x[2 * beams:2 * beams + 2].contiguous(), [-1.0, -2.0], [0, 0], 2, 3)  # nothing at all


def test_select_of_finished_beams():
    need_gpu()
    x = logits_of(8, 300, 9)
    run_select(x, scores_of(8), [1] * 8, 8, 4)
    run_select(x, scores_of(8), [1, 0] * 4, 4, 4)
    run_select(x, scores_of(8), [1, 0] * 4, 4, -1)
    run_select(x, [-math.inf] * 8, [1, 0] * 4, 4, 4)
    run_select(x, [float("nan")] + [-1.0] * 7, [0] * 8, 4, 4)
    x[:, 4] = 30.0  # the end is every beam's best
    run_select(x, scores_of(8), [0] * 8, 4, 4)


# --------------------------------------------------------------------------------------------- reorder

def beams_of(groups, beams, slots, fmt="bf16", heads=2, dim=64, layers=2, layout="nhd", ragged=False, spare=3, seed=0, tail=None):
    """A Setup whose groups share the full pages of a prompt, each sequence with a tail of its own."""
    r = cm.rng(seed)
    prompts = [r.randrange(0, 5) * slots for _ in range(groups)]
    tails = [r.randrange(1, 2 * slots + 3) if tail is None else tail for _ in range(groups)]
    lens = []
    for p, n in zip(prompts, tails):
        lens += [p + (r.randrange(0, n + 1) if ragged else n) for _ in range(beams)]
    st = Setup(lens, slots, heads, dim, fmt, layers=layers, layout=layout, spare=spare, seed=seed, columns=max(1, 5 + 4))
    for g, p in enumerate(prompts):
        for b in range(1, beams):
            for i in range(p // slots):
                st.state.refs[st.state.table[g * beams + b][i]] -= 1
                st.state.table[g * beams + b][i] = st.state.table[g * beams][i]
                st.state.refs[st.state.table[g * beams][i]] += 1
    st.table.copy_(i32(st.state.table))
    st.refs.copy_(i32(st.state.refs))
    return st


def parents_of(groups, beams, seed):
    r = cm.rng(seed)
    return [g * beams + min(r.randrange(beams), r.randrange(beams)) for g in range(groups) for _ in range(beams)]


def run_reorder(st, parents, beams):
    k, v = raw(st.k).clone(), raw(st.v).clone()
    before = [list(row) for row in st.table.tolist()]
    moves = cm.reorder(st.state, parents, beams)
    ops.paged_cache_reorder(st.cache, i32(parents), beams)
    assert ops.device_errors() == (_lib.DEVERR_PAGED if moves is None else 0)
    for a, b, used in moves or []:
        k[:, b, :used], v[:, b, :used] = k[:, a, :used].clone(), v[:, a, :used].clone()
    st.check_state()
    assert torch.equal(raw(st.k), k) and torch.equal(raw(st.v), v)
    for s, row in enumerate(st.table.tolist()):  # entries behind the pages in use keep what they held
        n = pm.pages_of(st.state.lens[s], st.slots)
        assert row[n:] == before[s][n:]
    return moves


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("slots", [1, 5, 16, 64])
def test_reorder_shares_and_copies(layout, fmt, slots):
    need_gpu()
    for seed, ragged in ((1, False), (2, True)):
        st = beams_of(4, 5, slots, fmt, layout=layout, ragged=ragged, spare=20, seed=seed)
        moves = run_reorder(st, parents_of(4, 5, seed), 5)
        assert moves if slots > 1 else moves == []


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (17, 128), (3, 64)])
@pytest.mark.parametrize("beams", [1, 2, 7, 64])
def test_reorder_of_head_layouts(beams, heads, dim):
    need_gpu()
    st = beams_of(3, beams, 16, heads=heads, dim=dim, seed=beams, tail=20)
    run_reorder(st, parents_of(3, beams, 5), beams)


def test_reorder_needs_no_free_page_for_beams_of_one_length():
    need_gpu()
    st = beams_of(3, 6, 16, spare=0, seed=3, tail=9)
    assert run_reorder(st, [g * 6 + 2 for g in range(3) for _ in range(6)], 6)
    assert run_reorder(st, [g * 6 + (5, 0, 3, 3, 1, 0)[b] for g in range(3) for b in range(6)], 6)
    assert run_reorder(st, [(s // 6 * 6 + (s + 1) % 6) for s in range(18)], 6) == []  # a rotation copies nothing
    assert run_reorder(st, list(range(18)), 6) == []


def test_reorder_with_too_few_pages_changes_nothing():
    need_gpu()
    st = Setup([24, 32, 32, 5], 16, 2, 64, spare=1)  # the sequences that are dropped have no partly filled page
    assert run_reorder(st, [0, 0, 0, 3], 4) is None
    st = Setup([24, 32, 32, 5], 16, 2, 64, spare=2)
    assert len(run_reorder(st, [0, 0, 0, 3], 4)) == 2


@pytest.mark.parametrize("parents", [[0, 1, 2, 4, 4, 5], [-1, 0, 0, 3, 3, 3], [0, 0, 0, 3, 3, 6], [2 ** 31 - 1, 0, 0, 3, 3, 3],
                                     [0, 0, 0, 2, 3, 3]])
def test_reorder_of_parents_outside_their_group_changes_nothing(parents):
    need_gpu()
    st = beams_of(2, 3, 16, seed=4)
    want = cm.reorder(st.state, parents, 3)
    if want is None:
        run_reorder(st, parents, 3)
        return
    st = beams_of(2, 3, 16, seed=4)
    run_reorder(st, parents, 3)


@pytest.mark.parametrize("what", ["length", "negative", "page"])
def test_reorder_of_a_broken_group_changes_nothing(what):
    need_gpu()
    st = beams_of(2, 4, 16, seed=5, tail=10)
    s = 5
    if what == "page":
        st.table[s, st.state.lens[s] // 16] = 1 << 20
    else:
        st.lens[s] = -1 if what == "negative" else 9 * 16 + 1
    saved = [t.clone() for t in (st.table, st.lens, st.refs, raw(st.k), raw(st.v))]
    ops.paged_cache_reorder(st.cache, i32([0, 1, 2, 3, 5, 5, 5, 7]), 4)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    for t, x in zip((st.table, st.lens, st.refs, raw(st.k), raw(st.v)), saved):
        assert torch.equal(t, x)


def test_reorder_moves_an_entry_outside_the_pool_uncounted():
    need_gpu()
    st = Setup([40, 40], 16, 2, 64)
    st.table[0, 0] = -3
    ops.paged_cache_reorder(st.cache, i32([0, 0]), 2)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert st.table[1, 0] == -3 and st.table[1, 1] == st.table[0, 1] and st.lens.tolist() == [40, 40]
    refs = st.refs.tolist()
    assert refs[st.state.table[1][0]] == 0 and refs[st.state.table[0][1]] == 2 and refs[st.state.table[0][2]] == 1


@pytest.mark.parametrize("groups,beams", [(400, 3), (1100, 1), (40, 64), (300, 8)])
def test_reorder_of_many_groups(groups, beams):
    need_gpu()
    st = beams_of(groups, beams, 8, heads=1, layers=1, ragged=True, spare=groups * beams, seed=6)
    run_reorder(st, parents_of(groups, beams, 6), beams)
    run_reorder(st, parents_of(groups, beams, 7), beams)


def test_reorder_of_some_sequences_leaves_the_others():
    need_gpu()
    st = beams_of(4, 3, 16, seed=8)
    parents = parents_of(2, 3, 3)
    k = raw(st.k).clone()
    moves = cm.reorder(st.state, parents, 3)
    ops.paged_cache_reorder(st.cache, i32(parents), 3)
    st.check_state()
    for a, b, used in moves:
        k[:, b, :used] = k[:, a, :used].clone()
    assert torch.equal(raw(st.k), k)
    ops.paged_cache_reorder(st.cache, i32([]), 3)
    st.check_state()
    assert ops.device_errors() == 0


@pytest.mark.parametrize("seed", range(6))
def test_runs_of_reorders(seed):
    need_gpu()
    r = cm.rng(seed)
    beams, slots = r.choice([2, 3, 4, 8]), r.choice([1, 4, 16])
    st = beams_of(3, beams, slots, r.choice(["bf16", "e4m3"]), ragged=r.random() < 0.5, spare=12, seed=seed)
    for i in range(6):
        run_reorder(st, parents_of(3, beams, 10 * seed + i), beams)
        new = [r.randrange(0, 3)] * (3 * beams)
        fits = st.state.reserve(new)
        ops.paged_cache_reserve(st.cache, i32(new))
        assert (ops.device_errors() == 0) == fits
        st.check_state()


# ------------------------------------------------------------------------------------- steps of them together

def beam_steps(graph):
    """A beam search of two prompts: reserve, append and attend a token of every beam, select among the candidates of logits
    that are a function of the attention's output, reorder. Each sequence's rows are followed in plain form."""
    need_gpu()
    groups, beams, heads, dim, slots, vocab, layers = 2, 4, 2, 64, 4, 700, 2
    S = groups * beams
    st = beams_of(groups, beams, slots, heads=heads, dim=dim, layers=layers, spare=60, seed=11, tail=3)
    g = torch.Generator(device=DEV).manual_seed(1)
    head = torch.randn((2 * heads * dim, vocab), generator=g, device=DEV) * 0.5
    k, v = (torch.empty((layers, S, heads, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q, out = (torch.empty((S, 2 * heads, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    logits = torch.empty((S, vocab), dtype=torch.bfloat16, device=DEV)
    scores = torch.tensor([0.0] + [-math.inf] * (beams - 1), device=DEV).repeat(groups)
    finished, parents, tokens = i32([0] * S), i32([0] * S), i32([0] * S)
    new, rs = i32([1] * S), i32(list(range(S + 1)))

    def rows(s, tensor, layer):
        n = st.state.lens[s]
        t = torch.arange(n, device=DEV)
        return tensor[layer, torch.tensor(st.state.table[s], device=DEV)[t // slots], t % slots]

    def step():
        ops.paged_cache_reserve(st.cache, new)
        for layer in range(layers):
            ops.paged_cache_append(st.cache, k[layer], v[layer], rs, layer=layer)
            ops.paged_attention(q, st.cache, rs, out, layer=layer, scale=0.2, max_rows=1)
        logits.copy_(torch.matmul(out.view(S, -1).float(), head))
        ops.beam_select(logits, scores, finished, scores, finished, parents, tokens, beams=beams, eos=3)
        ops.paged_cache_reorder(st.cache, parents, beams)

    def inputs():
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))

    run = step
    if graph:
        ops.init()
        inputs()
        state = (st.table, st.lens, st.refs, st.k, st.v, scores, finished)
        saved = [t.clone() for t in state]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
        for t, x in zip(state, saved):
            t.copy_(x)
        run = captured.replay
    held = [[[rows(s, t, layer).clone() for layer in range(layers)] for t in (st.k, st.v)] for s in range(S)]
    for _ in range(6):
        inputs()
        before, was = scores.tolist(), finished.tolist()
        run()
        assert ops.device_errors() == 0
        want = cm.select(logits, before, was, beams, 3)
        assert parents.tolist() == want[2] and tokens.tolist() == want[3] and finished.tolist() == want[1]
        check_scores(scores, want[0])
        assert st.state.reserve([1] * S)
        assert cm.reorder(st.state, want[2], beams) is not None
        st.check_state()
        for s in range(S):
            for t, new_rows in enumerate((k, v)):
                for layer in range(layers):
                    held[s][t][layer] = torch.cat([held[s][t][layer], new_rows[layer, s:s + 1]])
        held = [[[x for x in t] for t in held[p]] for p in want[2]]
        for s in range(S):
            for t, tensor in enumerate((st.k, st.v)):
                for layer in range(layers):
                    assert torch.equal(rows(s, tensor, layer), held[s][t][layer]), (s, t, layer)


def test_beam_steps():
    beam_steps(graph=False)


def test_a_captured_beam_step_replays():
    beam_steps(graph=True)


def test_calls_repeat_their_bits():
    need_gpu()
    x, s = logits_of(40, 50000, 2), torch.tensor(scores_of(40), device=DEV)
    f = i32([0] * 40)
    first = None
    for _ in range(3):
        o = torch.empty_like(s), torch.empty_like(f), torch.empty_like(f), torch.empty_like(f)
        ops.beam_select(x, s, f, *o, beams=10, eos=1)
        first = first or o
        assert all(torch.equal(a, b) for a, b in zip(o, first))


def test_the_front_end_refuses():
    need_gpu()
    x, s, f = logits_of(6, 100), torch.zeros(6, device=DEV), i32([0] * 6)
    p, t = f.clone(), f.clone()
    st = Setup([30, 40, 20], 16, 2, 128)
    for error, call in [
        (ValueError, lambda: ops.beam_select(x, s, f, s, f, p, t, beams=4)),
        (ValueError, lambda: ops.beam_select(x, s, f, s, f, p, t, beams=0)),
        (ValueError, lambda: ops.beam_select(x, s[:5], f, s, f, p, t, beams=2)),
        (TypeError, lambda: ops.beam_select(x, s.double(), f, s, f, p, t, beams=2)),
        (TypeError, lambda: ops.beam_select(x, s, f.bool(), s, f, p, t, beams=2)),
        (TypeError, lambda: ops.beam_select(x.float(), s, f, s, f, p, t, beams=2)),
        (ValueError, lambda: ops.beam_select(x.cpu(), s, f, s, f, p, t, beams=2)),
        (ValueError, lambda: ops.beam_select(x, s, f, s, f, p.cpu(), t, beams=2)),
        (TypeError, lambda: ops.beam_select(x, s, f, s, f, None, t, beams=2)),
        (_lib.MoaError, lambda: ops.beam_select(x, s, f, s, f, p, t, beams=2, eos=100)),
        (_lib.MoaError, lambda: ops.beam_select(x, s, f, s, f, p, t, beams=2, eos=-2)),
        (_lib.MoaError, lambda: ops.beam_select(torch.empty((65, 10), dtype=torch.bfloat16, device=DEV), *[torch.zeros(65, dtype=d, device=DEV) for d in
                                                (torch.float32, torch.int32, torch.float32, torch.int32, torch.int32, torch.int32)], beams=65)),
        (_lib.MoaError, lambda: ops.paged_cache_reorder(st.cache, i32([0, 0, 2]), 2)),
        (_lib.MoaError, lambda: ops.paged_cache_reorder(st.cache, i32([0, 0, 2, 2]), 2)),
        (_lib.MoaError, lambda: ops.paged_cache_reorder(st.cache, i32([0, 0, 2]), 0)),
        (TypeError, lambda: ops.paged_cache_reorder(st.cache, i32([0, 0, 2]).long(), 3)),
        (TypeError, lambda: ops.paged_cache_reorder(None, i32([0, 0, 2]), 3)),
        (TypeError, lambda: ops.paged_cache_reorder(st.cache, None, 3)),
    ]:
        with pytest.raises(error):
            call()
    assert ops.device_errors() == 0


@pytest.mark.parametrize("scores", [[-0.0, 0.0, -0.0], [0.0, -0.0, 0.0]])
def test_select_of_zeros_of_both_signs(scores):
    need_gpu()
    run_select(logits_of(3, 20), scores, [1, 1, 1], 3, 4)
