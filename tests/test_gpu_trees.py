"""Drafted trees over the paged cache on the GPU: attention of the nodes against a float64 evaluation, the greedy verification
and the commit against plain models, and speculative steps of them together."""
import itertools
import math

import pytest

import candidates_model as cm
import paged_model as pm
from gpu_util import need_gpu, torch
from moa_amd import _lib, ops
from test_gpu_paged import LAYOUTS, Setup, i32, queries, raw, starts_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(got, want, a, d, dim):
    """|got - want| within: half a bf16 step of the result (2^-8 relative); weights held to 2^-16 of themselves, which moves the
    result by at most 2^-16 a; scores rounded as f32 sums of `dim` products (dim + 4 roundings of 2^-24 relative to sum |q k|), which
    moves every weight and the sum by that much: twice; exponentials, sums and the division in f32: 2^-18 of a covers them (exp2 of
    a rounded argument below 2^7, sums of up to 2^15 weights)."""
    got = got.double()
    assert torch.isfinite(got).all()
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * a * (2.0 ** -16 + 2.0 ** -18 + 2 * (dim + 4) * 2.0 ** -24 * d[..., None]) + 1e-30
    over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, f"beyond the tolerance by {over}; worst |d| {(got - want).abs().max().item()}"


def attend(st, rows, masks, heads, window=0, scale=1.0, seed=5, first=0, tail=0, max_rows=None, layer=0, words=None, junk=0):
    """One call on a Setup; masks: the integers of the rows of all sequences. Checks every row of them, and that the others keep what
    they held. junk: rows of stride beyond the heads."""
    starts = starts_of(rows, first)
    R = starts[-1] + tail
    words = words or cm.words_of(max(rows))
    q = queries(R, heads, st.dim, seed, 2.0 / scale)
    out = torch.full((R, heads + junk, st.dim), 123.0, dtype=torch.bfloat16, device=DEV)[:, :heads]
    full = [0] * first + list(masks) + [0] * tail
    ops.paged_tree_attention(q, st.cache, i32(starts), cm.mask_tensor(full, words, DEV), out, layer=layer, window=window, scale=scale,
                             max_rows=max_rows or max(rows))
    assert ops.device_errors() == 0
    k, v = st.values(layer)
    sc = (None, None) if st.k_scale is None else (st.k_scale[layer], st.v_scale[layer])
    want, a, d = cm.attention(q, k, v, st.state.table, st.state.lens, starts, full, st.slots, window, scale, *sc)
    inside = slice(first, starts[-1])
    check(out[inside], want[inside], a[inside], d[inside], st.dim)
    assert (out[:first] == 123.0).all() and (out[starts[-1]:] == 123.0).all()
    return out


def trees(sizes, seed=1, chain=False):
    r = cm.rng(seed)
    return list(itertools.chain.from_iterable(cm.tree(r, n, chain) for n in sizes))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("group,heads,dim", LAYOUTS)
def test_trees_of_ragged_sequences(group, heads, dim, fmt):
    need_gpu()
    sizes = [1, 5, 0, 8, 16, 3, 33, 64, 2]
    before = [0, 1, 40, 15, 63, 700, 129, 1000, 2049]
    st = Setup([b + n for b, n in zip(before, sizes)], 16, heads, dim, fmt)
    attend(st, sizes, trees(sizes), heads * group, scale=1.0 / math.sqrt(dim))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [64, 100, 129, 1024])
def test_a_window_counts_from_a_nodes_depth(window, fmt):
    need_gpu()
    sizes, before = [1, 7, 64, 30, 12], [0, window - 3, 2000, window + 70, 50]
    st = Setup([b + n for b, n in zip(before, sizes)], 48, 2, 128, fmt)
    attend(st, sizes, trees(sizes, 3), 8, window=window, scale=0.1)
    attend(st, sizes, trees(sizes, 3, chain=True), 8, window=window, scale=0.1)
    st = Setup([b + n for b, n in zip(before[:2], [1, 7])], 64, 8, 256, fmt)  # the joined records of few rows
    attend(st, [1, 7], trees([1, 7], 3), 8, window=window)


@pytest.mark.parametrize("n,words", [(65, 2), (128, 2), (129, 4), (200, 4), (256, 4), (3, 4), (64, 1)])
@pytest.mark.parametrize("group,heads,dim", [(2, 2, 256), (16, 1, 512), (1, 3, 64), (4, 2, 128)])
def test_masks_of_several_words(n, words, group, heads, dim):
    need_gpu()
    before = [0, 37, 1000]
    st = Setup([b + n for b in before], 24, heads, dim)
    attend(st, [n] * 3, trees([n] * 3, 4), heads * group, scale=1.0 / math.sqrt(dim), words=words)


@pytest.mark.parametrize("n,dim", [(4, 128), (16, 64), (40, 128), (90, 256), (200, 128), (33, 512)])
def test_any_set_of_nodes(n, dim):
    """Sets that are no ancestors, with later nodes and without the row itself; bits from n on; rows without bits."""
    need_gpu()
    r = cm.rng(n)
    sizes, before = [n, 1, n], [70, 5, 0]
    words = cm.words_of(n)
    masks = [r.getrandbits(64 * words) & r.getrandbits(64 * words) if i % 5 else 0 for i in range(sum(sizes))]
    masks[n] = 1
    masks[n + 1] |= 1 << n - 1  # something to see where nothing lies before the tree
    st = Setup([b + m for b, m in zip(before, sizes)], 16, 2, dim)
    # depth counts the nodes below n, wherever they are
    attend(st, sizes, [m & ((1 << n) - 1) if n <= 64 * words else m for m in masks], 8, scale=1.0 / math.sqrt(dim))
    out = attend(st, sizes, masks, 8, scale=1.0 / math.sqrt(dim))
    assert (out[0] == 0).all()


@pytest.mark.parametrize("group,heads,dim,fmt", [(16, 1, 512, "bf16"), (2, 8, 256, "e4m3"), (4, 2, 128, "bf16"), (1, 2, 64, "e4m3")])
@pytest.mark.parametrize("n", [4, 24, 64])
def test_long_sequences_split(group, heads, dim, fmt, n):
    need_gpu()
    st = Setup([9000 + n, 30 + n], 100, heads, dim, fmt)
    attend(st, [n, n], trees([n, n], 6), heads * group, scale=1.0 / math.sqrt(dim))


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
@pytest.mark.parametrize("slots", [1, 7, 64, 512])
def test_page_sizes_and_layouts(slots, layout):
    need_gpu()
    sizes, before = [9, 30, 1], [100, 55, 700]
    st = Setup([b + n for b, n in zip(before, sizes)], slots, 2, 128, layout=layout, layers=2)
    attend(st, sizes, trees(sizes), 6, scale=0.1, layer=1, first=3, tail=2, junk=2)


def test_a_chain_is_consecutive_tokens():
    need_gpu()
    for n in (1, 6, 50):
        st = Setup([n + 300, n], 16, 2, 128)
        out = attend(st, [n, n], trees([n, n], chain=True), 8, scale=0.1)
        plain = torch.empty_like(out)
        ops.paged_attention(queries(2 * n, 8, 128, 5, 20.0), st.cache, i32([0, n, 2 * n]), plain, scale=0.1, max_rows=n)
        assert torch.allclose(out.float(), plain.float(), rtol=2.0 ** -7, atol=1e-5)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,heads,group,dim", [(6, 2, 2, 128), (16, 1, 1, 512), (40, 2, 2, 128), (30, 1, 16, 512), (100, 1, 2, 256), (5, 2, 1, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_a_node_does_not_see_never_reach_it(n, heads, group, dim, fmt, bad):
    """Slots behind the sequences and one node hold NaN or infinities; the nodes that do not see it are finite and right."""
    need_gpu()
    if fmt == "e4m3" and bad == float("inf"):
        pytest.skip("E4M3 has no infinity")
    st = Setup([80 + n, n], 16, heads, dim, fmt, poison=True)
    masks = trees([n, n], 8)
    victim = n // 2
    page, slot = st.state.table[0][(80 + victim) // 16], (80 + victim) % 16
    for t in (st.k, st.v):
        if fmt == "bf16":
            t[0, page, slot] = bad
        else:
            t.view(torch.uint8)[0, page, slot] = 0x7F
    q = queries(2 * n, heads * group, dim, 5, 2.0 * math.sqrt(dim))
    out = torch.empty_like(q)
    scale = 1.0 / math.sqrt(dim)
    ops.paged_tree_attention(q, st.cache, i32([0, n, 2 * n]), cm.mask_tensor(masks, cm.words_of(n), DEV), out, scale=scale, max_rows=n)
    assert ops.device_errors() == 0
    k, v = st.values()
    k, v = (torch.where(t.isfinite(), t, 0.0) for t in (k, v))
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    want, a, d = cm.attention(q, k, v, st.state.table, st.state.lens, [0, n, 2 * n], masks, 16, 0, scale, *sc)
    rows = [i for i in range(2 * n) if i >= n or not masks[i] >> victim & 1]
    check(out[rows], want[rows], a[rows], d[rows], dim)
    if bad != bad:
        assert all(out[i].isnan().all() for i in range(n) if masks[i] >> victim & 1)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,heads,group,dim", [(6, 2, 2, 128), (20, 1, 1, 256), (12, 2, 4, 64), (50, 2, 1, 256), (25, 1, 4, 128), (40, 1, 16, 512), (200, 1, 1, 64)])
@pytest.mark.parametrize("rise", [0.05, 1.0, 40.0])
def test_scores_that_rise_along_the_sequence(rise, n, heads, group, dim, fmt):
    """The largest score grows by 700 rise over the positions, so that a reference taken early is far below it."""
    need_gpu()
    st = Setup([700 + n, 3 + n], 16, heads, dim, fmt)
    step = torch.arange(700 + n, device=DEV).float() * rise / dim
    page = torch.tensor(st.state.table[0], device=DEV)[torch.arange(700 + n, device=DEV) // 16]
    rows = step[:, None, None].expand(-1, heads, dim)
    if fmt == "bf16":
        st.k[0, page, torch.arange(700 + n, device=DEV) % 16] = rows.to(torch.bfloat16)
    else:
        codes = (rows / st.k_scale[0][:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        st.k.view(torch.uint8)[0, page, torch.arange(700 + n, device=DEV) % 16] = codes.view(torch.uint8)
    masks = trees([n, n], 3)
    q = torch.ones((2 * n, heads * group, dim), dtype=torch.bfloat16, device=DEV)
    q[::2] = -1.0
    out = torch.empty_like(q)
    ops.paged_tree_attention(q, st.cache, i32([0, n, 2 * n]), cm.mask_tensor(masks, cm.words_of(n), DEV), out, max_rows=n)
    assert ops.device_errors() == 0
    k, v = st.values()
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    want, a, d = cm.attention(q, k, v, st.state.table, st.state.lens, [0, n, 2 * n], masks, 16, 0, 1.0, *sc)
    check(out, want, a, d, dim)


@pytest.mark.parametrize("n", [2, 60])
@pytest.mark.parametrize("bad", ["page", "length", "rows", "descend"])
def test_bad_sequences_are_left_out(bad, n):
    need_gpu()
    st = Setup([40 + n] * 3, 16, 2, 128)
    starts = [0, n, 2 * n, 3 * n]
    max_rows = n
    if bad == "page":
        st.table[1, (40 + n - 1) // 16] = st.state.refs.__len__()
    elif bad == "length":
        st.lens[1] = -1
    elif bad == "rows":
        max_rows, starts = n, [0, n - 1, 2 * n, 3 * n]
    else:
        starts = [0, n, n - 1, n - 1]
    q = queries(3 * n, 4, 128, 5, 20.0)
    out = torch.full_like(q, 7.0)
    ops.paged_tree_attention(q, st.cache, i32(starts), cm.mask_tensor(trees([n] * 3), 1, DEV), out, scale=0.1, max_rows=max_rows)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    if bad in ("page", "length"):
        assert (out[n:2 * n] == 7.0).any() and (out[:n] != 7.0).any(-1).all() and (out[2 * n:] != 7.0).any(-1).all()
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("seed", range(8))
def test_random_shapes(seed):
    need_gpu()
    r = cm.rng(100 + seed)
    group, heads, dim = r.choice(LAYOUTS)
    S = r.choice([1, 2, 5, 20])
    sizes = [r.choice([0, 1, 2, 3, 8, r.randrange(1, 70)]) for _ in range(S)]
    sizes[0] = max(1, sizes[0])
    before = [r.choice([0, 1, r.randrange(0, 200), r.randrange(0, 3000)]) for _ in range(S)]
    window = r.choice([0, 0, 128, 1000])
    st = Setup([b + n for b, n in zip(before, sizes)], r.choice([1, 16, 33, 128]), heads, dim, r.choice(["bf16", "e4m3"]), seed=seed)
    masks = [m if r.random() > 0.1 else 0 for m in trees(sizes, seed)]
    attend(st, sizes, masks, heads * group, window=window, scale=1.0 / math.sqrt(dim), seed=seed)


# ---------------------------------------------------------------------------------------------- verify

def run_verify(logits, tokens, starts, masks, words=None):
    rows, S = logits.shape[0], len(starts) - 1
    best, leaves, nexts = (torch.full((n,), -5, dtype=torch.int32, device=DEV) for n in (rows, S, S))
    ops.tree_verify(logits, i32(tokens), i32(starts), cm.mask_tensor(masks, words or cm.words_of(max([1] + [b - a for a, b in zip(starts, starts[1:])])), DEV),
                    best, leaves, nexts)
    return best.tolist(), leaves.tolist(), nexts.tolist()


def drafted(logits, sizes, seed):
    """Tokens of trees that follow the logits in most nodes, and the trees' masks."""
    r = cm.rng(seed)
    masks = trees(sizes, seed)
    x = torch.where(logits.isnan(), -math.inf, logits.float())
    best = x.argmax(1).tolist()
    tokens, first = [], 0
    for n in sizes:
        for i in range(n):
            m = masks[first + i] & ~(1 << i)
            parent = m.bit_length() - 1
            tokens.append(best[first + parent] if parent >= 0 and r.random() < 0.7 else r.randrange(logits.shape[1]))
        first += n
    return tokens, masks


@pytest.mark.parametrize("vocab", [1, 7, 8, 9, 64, 1000, 4096, 32003, 262144])
def test_verify_takes_the_largest_logits_path(vocab):
    need_gpu()
    sizes = [3, 1, 20, 0, 5] if vocab > 100000 else [3, 1, 64, 0, 17, 130]
    g = torch.Generator(device=DEV).manual_seed(vocab)
    logits = (torch.randn((sum(sizes), vocab), generator=g, device=DEV) * 4).to(torch.bfloat16)
    tokens, masks = drafted(logits, sizes, 2)
    starts = starts_of(sizes)
    got = run_verify(logits, tokens, starts, masks)
    assert got == tuple(cm.verify(logits.float(), tokens, starts, masks))
    assert ops.device_errors() == 0
    if vocab > 9:
        assert max(got[1]) > 0


@pytest.mark.parametrize("stride", [1000, 1003, 1016])
def test_verify_of_rows_that_lie_apart(stride):
    need_gpu()
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = (torch.randn((30, stride), generator=g, device=DEV) * 4).to(torch.bfloat16)
    logits[:, 999:] = 500.0  # not the rows'
    logits = logits[:, :999]
    tokens, masks = drafted(logits, [10, 20], 3)
    assert run_verify(logits, tokens, [0, 10, 30], masks) == tuple(cm.verify(logits.float(), tokens, [0, 10, 30], masks))


@pytest.mark.parametrize("vocab", [50, 5000, 70000])
def test_verify_of_ties_and_numbers_that_are_none(vocab):
    need_gpu()
    logits = torch.full((9, vocab), -1.0, dtype=torch.bfloat16, device=DEV)
    logits[0, [vocab - 1, 13, 30]] = 2.0
    logits[1] = -math.inf
    logits[2] = float("nan")
    logits[3] = -math.inf
    logits[3, 11:] = float("nan")
    logits[4] = float("nan")
    logits[4, vocab - 2] = -math.inf
    logits[5] = -0.0
    logits[5, 21] = 0.0
    logits[6, 40], logits[6, 17] = -0.0, 0.0
    logits[6, 9] = -1e-39
    logits[7, 5], logits[7, 8] = float("nan"), math.inf
    logits[8, :] = torch.finfo(torch.bfloat16).min
    bits = logits.view(torch.int16)
    bits[2, ::2] = -1  # NaNs of negative sign
    masks = trees([9])
    got = run_verify(logits, [0] * 9, [0, 9], masks)
    assert got[0] == [13, 0, 0, 0, vocab - 2, 0, 17, 8, 0]
    assert got == tuple(cm.verify(logits.float(), [0] * 9, [0, 9], masks))


def test_verify_of_rows_without_a_tree():
    """Rows of no sequence keep what they held; empty sequences and first rows without bits have no leaf; bad ones raise the bit."""
    need_gpu()
    logits = torch.randn((12, 300), device=DEV).to(torch.bfloat16)
    masks = [0, 0] + [1, 3] + [0, 2] + [1, 3, 5] + [0, 0, 0]
    got = run_verify(logits, [1] * 12, [2, 4, 6, 6, 9], masks, words=1)
    want = cm.verify(logits.float(), [1] * 12, [2, 4, 6, 6, 9], masks)
    assert got[0] == [-5, -5] + want[0][2:9] + [-5] * 3 and got[1:] == (want[1], want[2])
    assert got[1][1] == -1 and got[1][2] == -1 and ops.device_errors() == 0
    for starts in ([0, 13], [-1, 3], [5, 3], [2 ** 31 - 1, -2 ** 31]):
        best, leaves, nexts = run_verify(logits, [1] * 12, starts, [1] * 12, words=1)
        assert (leaves, nexts) == ([-1], [-1]) and best == [-5] * 12
        assert ops.device_errors() == _lib.DEVERR_PAGED
    x = torch.randn((70, 40), device=DEV).to(torch.bfloat16)
    assert run_verify(x, [1] * 70, [0, 65], trees([65]) + [0] * 5, words=1)[1] == [-1]
    assert ops.device_errors() == _lib.DEVERR_PAGED
    empty = torch.empty((0, 40), dtype=torch.bfloat16, device=DEV)
    assert run_verify(empty, [], [0, 0, 0], [], words=1) == ([], [-1, -1], [-1, -1]) and ops.device_errors() == 0


def test_verify_of_a_tree_of_256_nodes_and_of_deep_chains():
    need_gpu()
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn((512, 2000), generator=g, device=DEV).to(torch.bfloat16)
    masks = trees([256], 5) + trees([256], chain=True)
    best = logits.float().argmax(1).tolist()
    tokens = drafted(logits[:256], [256], 5)[0] + [0] + best[256:511]
    assert [m for m in masks[:256]] == drafted(logits[:256], [256], 5)[1]
    got = run_verify(logits, tokens, [0, 256, 512], masks)
    assert got == tuple(cm.verify(logits.float(), tokens, [0, 256, 512], masks)) and got[1][1] == 255


# ---------------------------------------------------------------------------------------------- commit

def moved(st, moves, k, v):
    """k and v (clones of the pages before) after the moves of a commit, which do not overlap once all are read."""
    if moves:
        (sp, ss), (dp, ds) = (torch.tensor(list(x), device=DEV).T for x in zip(*moves))
        for t in (k, v):
            t[:, dp, ds] = t[:, sp, ss]
    return k, v


def run_commit(st, sizes, masks, leaves, starts=None, words=None):
    starts = starts or starts_of(sizes)
    k, v = raw(st.k).clone(), raw(st.v).clone()
    moves, left = cm.commit(st.state, starts, masks, leaves)
    k, v = moved(st, moves, k, v)
    ops.paged_tree_commit(st.cache, i32(starts), cm.mask_tensor(masks, words or cm.words_of(max(sizes)), DEV), i32(leaves))
    st.check_state()
    assert torch.equal(raw(st.k), k) and torch.equal(raw(st.v), v)
    assert ops.device_errors() == (_lib.DEVERR_PAGED if left else 0)
    return moves


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("slots", [1, 5, 16, 128])
def test_commit_keeps_a_path(layout, fmt, slots):
    need_gpu()
    sizes, before = [12, 0, 1, 64, 7, 30, 9], [0, 20, 33, 100, 15, 16, 40]
    st = Setup([b + n for b, n in zip(before, sizes)], slots, 3, 64, fmt, layers=3, layout=layout)
    masks = trees(sizes, 4)
    assert run_commit(st, sizes, masks, [11, 5, 0, 60, -1, 29, 3])


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (1, 64), (17, 128)])
def test_commit_of_head_layouts(heads, dim):
    need_gpu()
    st = Setup([100 + 20, 30 + 20], 16, heads, dim, layers=2)
    assert run_commit(st, [20, 20], trees([20, 20], 9), [19, 15])


def test_commit_of_256_nodes_and_overlapping_moves():
    need_gpu()
    st = Setup([300 + 256, 256, 10], 24, 2, 128, layers=2)
    every_other = sum(1 << i for i in range(0, 256, 2))
    masks = trees([256], 4)[:255] + [every_other] + [((1 << 256) - 1) ^ 1] * 256
    moves = run_commit(st, [256, 256, 0], masks, [255, 7, 0])
    assert len(moves) == 127 + 255


def test_commit_of_a_chain_is_a_shorter_sequence():
    need_gpu()
    st = Setup([50 + 9, 64], 16, 2, 64)
    assert run_commit(st, [9, 8], trees([9, 8], chain=True), [3, -1]) == []
    assert st.state.lens == [54, 56]


@pytest.mark.parametrize("bad", ["leaf", "leaf_low", "shared", "page", "length", "short", "rows", "descend"])
def test_commit_leaves_out_bad_sequences(bad):
    need_gpu()
    n = 10
    st = Setup([40 + n, 25 + n, 30 + n], 16, 2, 64, layers=2)
    masks, leaves, starts = trees([n] * 3, 3), [9, 9, 8], [0, n, 2 * n, 3 * n]
    words = 1
    if bad == "leaf":
        leaves[1] = n
    elif bad == "leaf_low":
        leaves[1] = -2
    elif bad == "shared":
        st.refs[st.state.table[1][(25 + n - 1) // 16]] = 2
        st.state.refs[st.state.table[1][(25 + n - 1) // 16]] = 2
    elif bad == "page":
        st.table[1, 2] = st.state.table[1][2] = 1 << 20
    elif bad in ("length", "short"):
        st.lens[1] = st.state.lens[1] = 2 ** 31 - 1 if bad == "length" else n - 1
    k, v = raw(st.k).clone(), raw(st.v).clone()
    if bad in ("rows", "descend"):
        starts = [0, n, 2 * n, 3 * n + 1] if bad == "rows" else [0, n, n - 3, n - 3]
        state = pm.State(st.state.table, st.state.lens, st.state.refs, 16)
        only = [0, n] + [n] * 2 if bad == "descend" else [0, n, 2 * n, 2 * n]
        moves, _ = cm.commit(state, only, masks, leaves)
        st.state = state
        k, v = moved(st, moves, k, v)
    else:
        moves, left = (cm.commit(st.state, starts, masks, leaves) if bad != "length" else
                       cm.commit(st.state, [0, n, n, 2 * n], masks[:n] + masks[2 * n:], leaves))
        k, v = moved(st, moves, k, v)
    ops.paged_tree_commit(st.cache, i32(starts), cm.mask_tensor(masks, words, DEV), i32(leaves))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert torch.equal(raw(st.k), k) and torch.equal(raw(st.v), v)
    assert st.lens.tolist() == st.state.lens and st.refs.tolist() == st.state.refs


def test_commit_without_rows_and_of_many_sequences():
    need_gpu()
    st = Setup([5, 40], 16, 2, 64)
    before = st.k.clone()
    ops.paged_tree_commit(st.cache, i32([0, 0, 0]), cm.mask_tensor([], 1, DEV), i32([7, 7]))
    assert st.lens.tolist() == [5, 40] and torch.equal(st.k, before) and ops.device_errors() == 0
    r = cm.rng(2)
    sizes = [r.randrange(0, 6) for _ in range(1500)]
    st = Setup([n + r.randrange(0, 20) for n in sizes], 8, 1, 64)
    run_commit(st, sizes, trees(sizes, 2), [r.randrange(-1, n) if n else 0 for n in sizes])


# ------------------------------------------------------------------------------------- steps of them together

def speculative_steps(graph):
    """Steps of three sequences: a tree is reserved, appended and attended, its logits verified, the accepted path committed. The logits are a
    function of the attention's output, so that a wrong value anywhere shows; every step is checked against the plain models."""
    need_gpu()
    S, heads, dim, slots, n, vocab, layers = 3, 2, 64, 8, 12, 500, 2
    st = Setup([20, 7, 0], slots, heads, dim, layers=layers, spare=40, columns=20)
    g = torch.Generator(device=DEV).manual_seed(0)
    head = torch.randn((2 * heads * dim, vocab), generator=g, device=DEV) * 0.3
    likely = torch.zeros(vocab, device=DEV)
    likely[7:10] = 20.0
    rows, starts = S * n, [n * i for i in range(S + 1)]
    k, v = (torch.empty((layers, rows, heads, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q, out = (torch.empty((rows, 2 * heads, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    masks, tokens = torch.empty((rows, 1), dtype=torch.int64, device=DEV), torch.empty(rows, dtype=torch.int32, device=DEV)
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device=DEV)
    best, leaves, nexts = (torch.empty(m, dtype=torch.int32, device=DEV) for m in (rows, S, S))
    new, rs = i32([n] * S), i32(starts)

    def step():
        ops.paged_cache_reserve(st.cache, new)
        for layer in range(layers):
            ops.paged_cache_append(st.cache, k[layer], v[layer], rs, layer=layer)
            ops.paged_tree_attention(q, st.cache, rs, masks, out, layer=layer, scale=0.2, max_rows=n)
        logits.copy_(torch.matmul(out.view(rows, -1).float(), head) + likely)
        ops.tree_verify(logits, tokens, rs, masks, best, leaves, nexts)
        ops.paged_tree_commit(st.cache, rs, masks, leaves)

    r = cm.rng(7)

    def inputs():
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        m = trees([n] * S, r.randrange(1000))
        if r.random() < 0.5:
            m[n - 1] = 0  # padded
        masks.copy_(cm.mask_tensor(m, 1, DEV))
        tokens.copy_(i32([r.choice([7, 8, 9]) for _ in range(rows)]))
        return m

    run = step
    if graph:
        ops.init()
        inputs()
        saved = [t.clone() for t in (st.table, st.lens, st.refs, st.k, st.v)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
        for t, x in zip((st.table, st.lens, st.refs, st.k, st.v), saved):
            t.copy_(x)
        run = captured.replay
    kept = 0
    for _ in range(5):
        m = inputs()
        run()
        assert ops.device_errors() == 0
        assert st.state.reserve([n] * S)
        kk, vv = st.values(layers - 1)
        # before the commit moved anything the tree's rows lay at its positions: put them back for the check
        for s, length in enumerate(st.state.lens):
            for j in range(n):
                t = length - n + j
                kk[st.state.table[s][t // slots], t % slots] = k[layers - 1, s * n + j].float()
                vv[st.state.table[s][t // slots], t % slots] = v[layers - 1, s * n + j].float()
        want, a, d = cm.attention(q, kk, vv, st.state.table, st.state.lens, starts, m, slots, 0, 0.2)
        check(out, want, a, d, dim)
        got = best.tolist(), leaves.tolist(), nexts.tolist()
        assert got == tuple(cm.verify(logits.float(), tokens.tolist(), starts, m))
        cm.commit(st.state, starts, m, got[1])
        kept += sum(x > 0 for x in got[1])
        st.check_state()
        for s, length in enumerate(st.state.lens):  # the accepted rows lie behind each other
            path = [j for j in range(n) if m[s * n + got[1][s]] >> j & 1]
            for p, j in enumerate(path):
                t = length - len(path) + p
                for layer in range(layers):
                    assert torch.equal(st.k[layer, st.state.table[s][t // slots], t % slots], k[layer, s * n + j])
                    assert torch.equal(st.v[layer, st.state.table[s][t // slots], t % slots], v[layer, s * n + j])
    assert kept > 3


def test_speculative_steps():
    speculative_steps(graph=False)


def test_a_captured_speculative_step_replays():
    speculative_steps(graph=True)


def test_calls_follow_the_current_stream():
    need_gpu()
    st = Setup([2000 + 20, 300 + 20], 16, 2, 128)
    masks = trees([20, 20])
    want = attend(st, [20, 20], masks, 8, scale=0.1)
    q, out = queries(40, 8, 128, 5, 20.0), torch.zeros_like(want)
    slow = torch.randn((4096, 4096), device=DEV)
    side = torch.cuda.Stream()
    mt, rs = cm.mask_tensor(masks, 1, DEV), i32([0, 20, 40])
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(10):
            slow = slow @ slow * 1e-3
        late.copy_(q)
        ops.paged_tree_attention(late, st.cache, rs, mt, out, scale=0.1, max_rows=20)
    side.synchronize()
    assert torch.equal(out, want)


def test_the_front_end_refuses():
    need_gpu()
    st = Setup([30, 40], 16, 2, 128)
    q = queries(10, 4, 128, 1)
    rs, m, out = i32([0, 5, 10]), cm.mask_tensor(trees([5, 5]), 1, DEV), torch.empty_like(q)
    for error, call in [
        (TypeError, lambda: ops.paged_tree_attention(q, None, rs, m, out)),
        (TypeError, lambda: ops.paged_tree_attention(q, st.cache, rs, None, out)),
        (TypeError, lambda: ops.paged_tree_attention(q, st.cache, rs, m.int(), out)),
        (ValueError, lambda: ops.paged_tree_attention(q, st.cache, rs, m[:9], out)),
        (ValueError, lambda: ops.paged_tree_attention(q, st.cache, rs, m.view(-1), out)),
        (ValueError, lambda: ops.paged_tree_attention(q, st.cache, rs, m.cpu(), out)),
        (ValueError, lambda: ops.paged_tree_attention(q, st.cache, rs, m, out[:9])),
        (ValueError, lambda: ops.paged_tree_attention(q, st.cache, rs[:2], m, out)),
        (_lib.MoaError, lambda: ops.paged_tree_attention(q, st.cache, rs, m, out, window=4, max_rows=5)),
        (_lib.MoaError, lambda: ops.paged_tree_attention(q, st.cache, rs, m, out, max_rows=65)),
        (_lib.MoaError, lambda: ops.paged_tree_attention(q, st.cache, rs, torch.zeros((10, 5), dtype=torch.int64, device=DEV), out)),
        (ValueError, lambda: ops.paged_tree_commit(st.cache, rs, m, i32([1]))),
        (TypeError, lambda: ops.paged_tree_commit(st.cache, rs, None, i32([1, 1]))),
        (TypeError, lambda: ops.paged_tree_commit(st.cache, rs, m, None)),
        (TypeError, lambda: ops.tree_verify(None, i32([0] * 10), rs, m, i32([0] * 10), i32([0, 0]), i32([0, 0]))),
        (TypeError, lambda: ops.tree_verify(q.view(10, -1), i32([0] * 10), rs, m, i32([0] * 10), None, i32([0, 0]))),
        (TypeError, lambda: ops.tree_verify(q.view(10, -1).float(), i32([0] * 10), rs, m, i32([0] * 10), i32([0, 0]), i32([0, 0]))),
        (ValueError, lambda: ops.tree_verify(q.view(10, -1), i32([0] * 9), rs, m, i32([0] * 10), i32([0, 0]), i32([0, 0]))),
        (ValueError, lambda: ops.tree_verify(q.view(10, -1), i32([0] * 10), rs, m, i32([0] * 10), i32([0, 0, 0]), i32([0, 0]))),
        (ValueError, lambda: ops.tree_verify(q.view(10, -1).T, i32([0] * 512), rs, m, i32([0] * 10), i32([0, 0]), i32([0, 0]))),
    ]:
        with pytest.raises(error):
            call()
    assert ops.device_errors() == 0
