"""Tree, beam and search calls on the GPU at the ends of their ranges: many sequences, large pools, results in place, numbers that are
none, row starts that are out of range, streams and graphs."""
import math

import pytest

import candidates_model as cm
import paged_model as pm
from gpu_util import need_gpu, say, torch
from moa_amd import _lib, ops
from test_gpu_beams import run_select
from test_gpu_paged import Setup, i32, queries, raw, starts_of
from test_gpu_trees import attend, check, run_commit, run_verify, trees

pytestmark = pytest.mark.gpu
DEV = "cuda"

# rows, group, KV heads, dim: few rows of a KV head, tiles of up to 128, more of them, and heads of 512
KINDS = [(2, 4, 2, 128), (3, 1, 1, 512), (30, 2, 2, 64), (60, 2, 1, 256), (60, 4, 1, 128), (40, 8, 1, 512), (200, 2, 1, 128)]


def reference(st, q, starts, masks, scale=1.0, window=0, values=None):
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    return cm.attention(q, *(values or st.values()), st.state.table, st.state.lens, starts, masks, st.slots, window, scale, *sc)


def call(st, q, starts, masks, out, most, **kw):
    ops.paged_tree_attention(q, st.cache, i32(starts), cm.mask_tensor(masks, cm.words_of(most), DEV), out, max_rows=most, **kw)


@pytest.mark.parametrize("S", [64, 65, 1100])
def test_attention_of_many_sequences(S):
    need_gpu()
    say(f"trees of {S} sequences")
    r = cm.rng(S)
    sizes = [r.choice([0, 1, 1, 2, 8, 20, 60]) for _ in range(S)]
    before = [r.choice([0, 1, 30, 200]) for _ in range(S)]
    before[S // 2] = 5000
    st = Setup([b + n for b, n in zip(before, sizes)], 16, 2, 64)
    attend(st, sizes, trees(sizes), 8, scale=0.125, first=3, tail=2)
    attend(st, sizes, trees(sizes), 4, scale=0.125, window=90)
    few = [min(n, 4) for n in sizes]
    attend(st, few, trees(few), 8, scale=0.125)


@pytest.mark.parametrize("heads,group,dim", [(128, 1, 64), (33, 3, 64), (9, 1, 512), (1, 128, 64), (2, 128, 512)])
def test_attention_of_many_heads(heads, group, dim):
    need_gpu()
    say(f"trees, {heads} KV heads x {group} of {dim}")
    for sizes in ([1, 3, 2], [20, 1, 7]):
        st = Setup([300 + sizes[0], sizes[1], 1100 + sizes[2]], 32, heads, dim)
        attend(st, sizes, trees(sizes), heads * group, scale=1 / math.sqrt(dim), window=200)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_results_in_place(n, group, heads, dim, fmt):
    need_gpu()
    say(f"trees in place, {n} of {heads} x {group} x {dim} {fmt}")
    masks = trees([n, n], 4)
    for before in (40, 5000):
        st = Setup([before + n, n], 64, heads, dim, fmt)
        q = queries(2 * n, heads * group, dim, 5, 2.0 * math.sqrt(dim))
        want, a, d = reference(st, q, [0, n, 2 * n], masks, 1 / math.sqrt(dim))
        call(st, q, [0, n, 2 * n], masks, q, n, scale=1 / math.sqrt(dim))
        assert ops.device_errors() == 0
        check(q, want, a, d, dim)


@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_scales(n, group, heads, dim):
    """Negative, zero, and such that scores reach some hundreds."""
    need_gpu()
    say(f"scales of trees, {n} of {heads} x {group} x {dim}")
    st = Setup([900 + n], 32, heads, dim)
    masks = trees([n], 2)
    for scale, spread in ((-0.5, 30.0), (0.0, 30.0), (1.0, 60.0)):
        q = queries(n, heads * group, dim, 3, spread)
        out = torch.empty_like(q)
        want, a, d = reference(st, q, [0, n], masks, scale)
        call(st, q, [0, n], masks, out, n, scale=scale)
        assert ops.device_errors() == 0
        check(out, want, a, d, dim)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", [(k[0], 4 if k[1] == 1 else k[1], 2, k[3]) for k in KINDS])
@pytest.mark.parametrize("length", [100, 9000])
def test_nan_that_a_node_sees_makes_it_nan(n, group, heads, dim, fmt, length):
    """A query that is NaN gives a NaN head, and so does a visible key or value; other rows and heads are unharmed."""
    need_gpu()
    say(f"visible NaN, {n} nodes of {heads} x {group} x {dim} after {length} {fmt}")
    st = Setup([length + n], 64, heads, dim, fmt, seed=23)
    masks = trees([n], 5)
    q = queries(n, heads * group, dim, 24, 2.0 * math.sqrt(dim))
    scale = 1 / math.sqrt(dim)
    want, a, d = reference(st, q, [0, n], masks, scale)
    out, sick = torch.zeros_like(q), q.clone()
    sick[n // 2, group] = float("nan")
    call(st, sick, [0, n], masks, out, n, scale=scale)
    assert ops.device_errors() == 0
    assert torch.isnan(out[n // 2, group].float()).all()
    well = torch.ones((n, heads * group), dtype=torch.bool, device=DEV)
    well[n // 2, group] = False
    check(out[well], want[well], a[well], d[well], dim)
    for at in (17, length + n // 2):  # a position before the tree, and a node
        page, slot = st.state.table[0][at // 64], at % 64
        sees = [i for i in range(n) if at < length or masks[i] >> n // 2 & 1]
        blind = [i for i in range(n) if i not in sees]
        for t in (st.k, st.v):
            view = t if fmt == "bf16" else t.view(torch.uint8)
            old = view[0, page, slot].clone()
            view[0, page, slot, 1, 3] = float("nan") if fmt == "bf16" else 0x7F
            call(st, q, [0, n], masks, out, n, scale=scale)
            view[0, page, slot] = old
            assert ops.device_errors() == 0
            assert torch.isnan(out[sees][:, group:, 3].float()).all()
            check(out[:, :group], want[:, :group], a[:, :group], d[:, :group], dim)
            check(out[blind], want[blind], a[blind], d[blind], dim)


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("n,group,heads,dim", [(k[0], k[1], 2, k[3]) for k in KINDS])
def test_a_scale_that_is_nan_shows_in_its_heads(which, n, group, heads, dim):
    need_gpu()
    say(f"a NaN {which}, {n} nodes of {dim}")
    st = Setup([300 + n], 16, heads, dim, "e4m3", seed=104)
    q, masks = queries(n, 2 * group, dim, 105), trees([n], 6)
    want, a, d = reference(st, q, [0, n], masks)
    getattr(st, which)[0, 1] = float("nan")
    out = torch.zeros_like(q)
    call(st, q, [0, n], masks, out, n)
    assert ops.device_errors() == 0
    assert torch.isnan(out[:, group:].float()).all()
    check(out[:, :group], want[:, :group], a[:, :group], d[:, :group], dim)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", [(2, 4, 2, 128), (30, 2, 2, 64), (32, 4, 1, 128), (32, 2, 1, 256), (32, 8, 1, 512)])
def test_values_that_nearly_cancel(n, group, heads, dim, fmt):
    """Positions in pairs of opposite values whose weights differ by 2^-10, the nodes chains, so that an odd row sees whole pairs.

    Tolerance, relative to a (the attention of |v|). A score is one product of bf16 numbers, so exact, and below 1: its factor (three
    roundings), the product with it and the distance to the reference are off by at most 5 * 2^-23 together, the exponential by
    2^-22, which moves a weight by less than 2^-20 of it. Two bf16 parts hold a weight to 2^-16. The sums of at most 96 products lose at
    most 2^-23 of a each time: 2^-16. The division and the last rounding are relative to the result."""
    need_gpu()
    say(f"values that cancel, {n} nodes of {heads} x {group} x {dim} {fmt}")
    length = 64 + n // 2 * 2
    st = Setup([length], 16, heads, dim, fmt, seed=95)
    g = torch.Generator(device=DEV).manual_seed(96)
    pairs = length // 2
    even, step, q0 = (1 + torch.randint(0, 60, (pairs, heads), generator=g, device=DEV) / 64, 2.0 ** -7, 2.0 ** -3)
    if fmt == "e4m3":
        even, step, q0 = 1 + torch.randint(0, 7, (pairs, heads), generator=g, device=DEV) / 8, 2.0 ** -3, 2.0 ** -7
        st.k_scale.fill_(1.0)
    sign = torch.randint(0, 2, (pairs, heads), generator=g, device=DEV) * 2 - 1
    k = torch.stack([even, even + step], 1)
    k = torch.where(sign[:, None] > 0, k, k.flip(1)).reshape(length, heads)
    v = torch.randn((pairs, 1, heads, dim), generator=g, device=DEV).clamp(-3, 3) * (60 if fmt == "e4m3" else 1)
    v = torch.cat([v, -v], 1).reshape(length, heads, dim)
    table, t = torch.tensor(st.state.table[0], device=DEV), torch.arange(length, device=DEV)
    kv = torch.zeros((length, heads, dim), device=DEV)
    kv[:, :, dim - 1] = k
    st.k[0, table[t // 16], t % 16] = kv.to(st.k.dtype)
    st.v[0, table[t // 16], t % 16] = v.to(st.v.dtype)
    n = n // 2 * 2
    masks = trees([n], chain=True)
    q = torch.zeros((n, heads * group, dim), dtype=torch.bfloat16, device=DEV)
    q[:, :, dim - 1] = q0
    want, a, _ = reference(st, q, [0, n], masks)
    out = torch.empty_like(q)
    call(st, q, [0, n], masks, out, n)
    assert ops.device_errors() == 0
    assert (want[-1].abs() < 2.0 ** -9 * a[-1]).float().mean() > 0.9  # they do cancel
    over = ((out.double() - want).abs() - 2.0 ** -8 * want.abs() - a * (2.0 ** -16 + 2.0 ** -16 + 2.0 ** -20)).max().item()
    assert over <= 0, f"beyond the tolerance by {over}, relative to a: {((out.double() - want).abs() / a).max().item()}"


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_a_bad_page_in_one_part_of_a_split_sequence(n, group, heads, dim, fmt):
    need_gpu()
    say(f"a bad page of a split sequence, {n} nodes of {heads} x {group} x {dim} {fmt}")
    st = Setup([16000 + n, 15000 + n], 64, heads, dim, fmt, seed=46)
    q, masks = queries(2 * n, heads * group, dim, 47), trees([n, n], 7)
    want, a, d = reference(st, q, [0, n, 2 * n], masks)
    good = st.table.clone()
    for at, p in ((3, -1), (100, 1 << 30), (16000 // 64, len(st.state.refs))):  # the last is the first node's
        st.table.copy_(good)
        st.table[0, at] = p
        out = torch.full_like(q, 123.0)
        call(st, q, [0, n, 2 * n], masks, out, n)
        assert ops.device_errors() == _lib.DEVERR_PAGED
        check(out[n:], want[n:], a[n:], d[n:], dim)
        assert (out[:n] == 123.0).all()


@pytest.mark.parametrize("n", [2, 30, 70])
@pytest.mark.parametrize("bad", [[2 ** 31 - 1, -2 ** 31], [2 ** 31 - 1, -2 ** 31 + 2], [-2 ** 31, 2 ** 31 - 1], [2 ** 30, 2 ** 30 + 1], [-1, 0]])
def test_row_starts_at_the_ends_of_int32(bad, n):
    """Pairs in the middle of a call's sequences, whose difference passes 32 bits or that lie outside: nothing out of range is
    touched, and the last sequence, whose starts are right, is."""
    need_gpu()
    say(f"row starts {bad} of {n} nodes")
    st = Setup([40 + n] * 5, 16, 2, 128, layers=1)
    starts = [0, n, *bad, 2 * n, 3 * n]
    masks = trees([n] * 3, 3)
    words = cm.words_of(n)
    q = queries(3 * n, 4, 128, 5)
    out = torch.full_like(q, 7.0)
    rs, mt = i32(starts), cm.mask_tensor(masks, words, DEV)
    ops.paged_tree_attention(q, st.cache, rs, mt, out, max_rows=n)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert torch.isfinite(out).all()
    x = torch.randn((3 * n, 50), device=DEV).to(torch.bfloat16)
    best, leaves, nexts = (torch.full((m,), -5, dtype=torch.int32, device=DEV) for m in (3 * n, 5, 5))
    ops.tree_verify(x, i32([51] * 3 * n), rs, mt, best, leaves, nexts)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    got = leaves.tolist()
    assert got[0] == 0 and got[4] == 0 and got[1] in (-1, 0) and got[2] == -1 and got[3] in (-1, 0)
    assert x[2 * n, nexts[4].item()] == x[2 * n].max()
    k = raw(st.k).clone()
    ops.paged_tree_commit(st.cache, rs, mt, i32([-1, 0, 0, 0, n - 1]))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    lens = st.lens.tolist()
    assert lens[0] == 40 and lens[2] == 40 + n and lens[4] == 40 + bin(masks[3 * n - 1]).count("1")
    changed = (raw(st.k) != k).flatten(2).any(-1)[0].nonzero().flatten().tolist()
    assert set(changed) <= set(st.state.table[4]) | set(st.state.table[3]) | set(st.state.table[1])


def large(layout):
    """A cache in a pool of more than 4 GB whose sequences lie at its two ends."""
    slots, heads, dim, pages = 64, 8, 256, 20500
    st = Setup.__new__(Setup)
    st.slots, st.heads, st.dim, st.layers, st.fmt, st.k_scale, st.v_scale = slots, heads, dim, 1, "bf16", None, None
    shape = (1, pages, heads, slots, dim) if layout == "hnd" else (1, pages, slots, heads, dim)
    st.k, st.v = torch.empty(shape, dtype=torch.bfloat16, device=DEV), torch.empty((1, pages, slots, heads, dim), dtype=torch.bfloat16, device=DEV)
    if layout == "hnd":
        st.k = st.k.transpose(2, 3)
    assert st.k.numel() * 2 > 1 << 32
    table = [[pages - 1, 0, pages - 2, 17000], [pages - 3, 5, 18000, 3]]
    refs = [0] * pages
    for p in table[0] + table[1]:
        st.k[0, p], st.v[0, p] = queries(slots, heads, dim, p, 16.0), queries(slots, heads, dim, p + 1, 16.0)
        refs[p] = 1
    st.state = pm.State(table, [250, 240], refs, slots)
    st.table, st.lens, st.refs = i32(table), i32([250, 240]), i32(refs)
    st.cache = ops.PagedCache(st.k, st.v, st.table, st.lens, st.refs)
    return st


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_offsets_past_32_bits(layout):
    need_gpu()
    say(f"trees and beams in a pool of 5.4 GB, {layout}")
    st = large(layout)
    used = sorted(set(st.state.table[0] + st.state.table[1]))
    near = [[used.index(p) for p in row] for row in st.state.table]
    for n in (2, 30, 64, 100):
        q, masks = queries(2 * n, 16, 256, 5), trees([n, n], 9)
        out = torch.empty_like(q)
        call(st, q, [0, n, 2 * n], masks, out, n)
        assert ops.device_errors() == 0
        want, a, d = cm.attention(q, st.k[0, used].float(), st.v[0, used].float(), near, st.state.lens, [0, n, 2 * n], masks, 64, 0, 1.0)
        check(out, want, a, d, 256)
    place = lambda t, s, p: t[0, st.state.table[s][p // 64], p % 64]  # noqa: E731
    rows = [[place(t, s, p).clone() for p in range(st.state.lens[s])] for t in (st.k, st.v) for s in range(2)]
    masks, n = trees([70, 60], 11), 70
    leaves = [69, 59]
    ops.paged_tree_commit(st.cache, i32([0, 70, 130]), cm.mask_tensor(masks, 2, DEV), i32(leaves))
    assert ops.device_errors() == 0
    cm.commit(st.state, [0, 70, 130], masks, leaves)
    st.check_state()
    for i, t in enumerate((st.k, st.v)):
        for s, n in enumerate((70, 60)):
            kept = [j for j in range(n) if masks[(0, 70)[s] + leaves[s]] >> j & 1]
            base = len(rows[2 * i + s]) - n
            want = rows[2 * i + s][:base] + [rows[2 * i + s][base + j] for j in kept]
            assert torch.equal(torch.stack([place(t, s, p) for p in range(st.state.lens[s])]), torch.stack(want))
            rows[2 * i + s] = want
    ops.paged_cache_reorder(st.cache, i32([0, 0]), 2)
    assert ops.device_errors() == 0
    cm.reorder(st.state, [0, 0], 2)
    st.check_state()
    for i, t in enumerate((st.k, st.v)):
        for s in range(2):
            assert torch.equal(torch.stack([place(t, s, p) for p in range(st.state.lens[s])]), torch.stack(rows[2 * i]))


@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_calls_repeat_their_bits(n, group, heads, dim):
    need_gpu()
    say(f"trees twice, {n} of {heads} x {group} x {dim}")
    st = Setup([3000 + n, 70 + n, n], 48, heads, dim, seed=33)
    starts, masks = [0, n, 2 * n, 3 * n], trees([n] * 3, 3)
    q = queries(3 * n, heads * group, dim, 2)
    outs = [torch.empty_like(q) for _ in range(2)]
    for o in outs:
        call(st, q, starts, masks, o, n)
        attend(st, [1, 0, 1], [1, 1], heads * group)
    assert torch.equal(*outs)


def test_graphs_take_turns():
    """Captured calls that share the library's scratch and counters; replayed in turn, with eager calls between, each keeps its result."""
    need_gpu()
    say("graphs of trees, verification and selection in turn")
    ops.init(0)
    made = []

    def capture(outs, run, *alive):
        run()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        made.append((graph, outs, want, alive, run))

    for i, (n, group, heads, dim) in enumerate(KINDS):
        st = Setup([9000 + n, 40 + n], 64, heads, dim, seed=52 + i)
        q, starts = queries(2 * n, heads * group, dim, 54 + i), i32([0, n, 2 * n])
        masks, out = cm.mask_tensor(trees([n, n], i), cm.words_of(n), DEV), torch.empty_like(q)
        capture([out], lambda st=st, q=q, starts=starts, masks=masks, out=out, n=n:
                ops.paged_tree_attention(q, st.cache, starts, masks, out, max_rows=n), st)
    g = torch.Generator(device=DEV).manual_seed(3)
    for sizes, vocab in (([5, 3], 40000), ([12] * 30, 9000)):
        rows = sum(sizes)
        x = torch.randn((rows, vocab), generator=g, device=DEV).to(torch.bfloat16)
        tokens, starts, masks = i32([int(t) for t in x.float().argmax(1).roll(1)]), i32(starts_of(sizes)), cm.mask_tensor(trees(sizes, 1, True), 1, DEV)
        outs = [torch.empty(m, dtype=torch.int32, device=DEV) for m in (rows, len(sizes), len(sizes))]
        capture(outs, lambda a=(x, tokens, starts, masks, *outs): ops.tree_verify(*a))
    for groups, beams, vocab in ((1, 4, 40000), (9, 12, 9000)):
        rows = groups * beams
        x = torch.randn((rows, vocab), generator=g, device=DEV).to(torch.bfloat16)
        scores, finished = torch.randn(rows, generator=g, device=DEV), i32([int(r % 5 == 3) for r in range(rows)])
        outs = [torch.empty(rows, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32, torch.int32)]
        capture(outs, lambda a=(x, scores, finished, *outs, beams, 3): ops.beam_select(*a))
    for turn in range(3):
        for graph, outs, want, _, run in made if turn % 2 == 0 else reversed(made):
            for o in outs:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
            run()
    assert ops.device_errors() == 0


def test_calls_wait_for_the_current_streams_work():
    """Every input is made by work that is still running on the side stream when the calls are issued: a call on another stream would
    read the zeros that were there before."""
    need_gpu()
    say("a speculative and a beam step behind running work of a side stream")
    n, vocab = 30, 5000
    st = Setup([100 + n, 40 + n], 16, 2, 128, seed=106, spare=10, columns=20)
    g = torch.Generator(device=DEV).manual_seed(8)
    masks = trees([n, n], 4)
    x = torch.randn((2 * n, vocab), generator=g, device=DEV).to(torch.bfloat16)
    best = x.float().argmax(1).tolist()
    tokens = [0] * (2 * n)
    for i in range(2 * n):
        m = masks[i] & ~(1 << i % n)
        if m:
            tokens[i] = best[i // n * n + m.bit_length() - 1]
    made = [queries(2 * n, 8, 128, 3), cm.mask_tensor(masks, 1, DEV), i32([0, n, 2 * n]), x, i32(tokens), i32([1, 1]),
            torch.randn(2 * n, generator=g, device=DEV)]
    late = [torch.zeros_like(t) for t in made]
    q, mt, rs, lx, lt, parents, scores = late
    zero = i32([0] * 2 * n)
    out = torch.full_like(q, 123.0)
    outs = [torch.full((m,), -5, dtype=torch.int32, device=DEV) for m in (2 * n, 2, 2)]
    total, ended, source, token = (torch.full((2 * n,), -5, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32, torch.int32))
    want, a, d = reference(st, made[0], [0, n, 2 * n], masks, 0.1)
    big = torch.randn((4096, 4096), device=DEV)
    side = torch.cuda.Stream()
    for warm in (True, False):
        with torch.cuda.stream(side):
            y = big
            for _ in range(1 if warm else 20):
                y = y @ big
                y = y / y.norm()
            nothing = y[0, 0] * 0
            for t, m in zip(late, made):
                t.copy_(m + nothing.to(m.dtype) if not warm else t)
            if not warm:
                busy = not side.query()
                ops.paged_tree_attention(q, st.cache, rs, mt, out, scale=0.1, max_rows=n)
                ops.tree_verify(lx, lt, rs, mt, *outs)
                ops.beam_select(lx, scores, zero, total, ended, source, token, 4)
                ops.paged_tree_commit(st.cache, rs, mt, outs[1])
                ops.paged_cache_reorder(st.cache, parents, 2)
        torch.cuda.synchronize()
    assert busy, "the side stream had finished before the calls were issued: the test shows nothing"
    assert ops.device_errors() == 0
    check(out, want, a, d, 128)
    verified = cm.verify(x.float(), tokens, [0, n, 2 * n], masks)
    assert tuple(o.tolist() for o in outs) == verified and max(verified[1]) > 0
    chosen = cm.select(x, made[6].tolist(), [0] * 2 * n, 4, -1)
    assert source.tolist() == chosen[2] and token.tolist() == chosen[3] and ended.tolist() == chosen[1]
    cm.commit(st.state, [0, n, 2 * n], masks, verified[1])
    cm.reorder(st.state, [1, 1], 2)
    st.check_state()


def test_the_largest_vocabulary_and_the_most_rows():
    need_gpu()
    say("2^20 logits a row, 65535 rows")
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn((12, 1 << 20), generator=g, device=DEV).to(torch.bfloat16)
    x[:, -1] = 9.0
    tokens, masks = [(1 << 20) - 1] * 12, trees([12], chain=True)
    assert run_verify(x, tokens, [0, 12], masks) == cm.verify(x.float(), tokens, [0, 12], masks)
    run_select(x, [-0.5 * r for r in range(12)], [0] * 12, 4, (1 << 20) - 1)
    rows = 65535
    x = torch.randn((rows, 9), generator=g, device=DEV).to(torch.bfloat16)
    best = x.float().argmax(1)
    outs = [torch.full((m,), -5, dtype=torch.int32, device=DEV) for m in (rows, rows, rows)]
    ops.tree_verify(x, i32([0] * rows), torch.arange(rows + 1, dtype=torch.int32, device=DEV), torch.ones((rows, 1), dtype=torch.int64, device=DEV), *outs)
    assert ops.device_errors() == 0
    assert (outs[1] == 0).all() and torch.equal(outs[0], outs[2])
    assert torch.equal(torch.gather(x, 1, outs[0].long()[:, None]), x.max(1, keepdim=True)[0]) and (outs[0] <= best).all()
    scores = torch.randn(rows, generator=g, device=DEV)
    total, ended, source, token = (torch.full((rows,), -5, dtype=t, device=DEV) for t in (torch.float32, torch.int32, torch.int32, torch.int32))
    ops.beam_select(x, scores, i32([0] * rows), total, ended, source, token, 1)
    assert ops.device_errors() == 0
    assert torch.equal(source, torch.arange(rows, dtype=torch.int32, device=DEV)) and torch.equal(token, outs[0]) and (ended == 0).all()
    want = scores.double() + torch.log_softmax(x.double(), 1).amax(1)
    assert ((total.double() - want).abs() <= 2.0 ** -18 + 2.0 ** -24 * want.abs()).all()


def test_commit_of_the_most_sequences():
    need_gpu()
    say("commit of 65536 sequences")
    S = 65536
    table = torch.arange(2 * S, dtype=torch.int32, device=DEV).view(S, 2)
    k = torch.arange(2 * S, device=DEV).float().view(1, 2 * S, 1, 1, 1).expand(1, 2 * S, 1, 1, 64).to(torch.bfloat16).contiguous()
    v = -k
    lens, refs = torch.full((S,), 2, dtype=torch.int32, device=DEV), torch.ones(2 * S, dtype=torch.int32, device=DEV)
    cache = ops.PagedCache(k, v, table, lens, refs)
    was = k.clone()
    masks = torch.tensor([[1], [2]], dtype=torch.int64, device=DEV).repeat(S, 1)
    leaves = torch.arange(S, dtype=torch.int32, device=DEV) % 3 - 1  # none, the first or the second
    ops.paged_tree_commit(cache, torch.arange(0, 2 * S + 1, 2, dtype=torch.int32, device=DEV), masks, leaves)
    assert ops.device_errors() == 0
    assert torch.equal(lens, (leaves >= 0).int())
    assert torch.equal(refs.view(S, 2)[:, 0], (leaves >= 0).int()) and (refs.view(S, 2)[:, 1] == 0).all()
    first = was.view(S, 2, 64)
    want = torch.where((leaves == 1)[:, None], first[:, 1], first[:, 0])
    assert torch.equal(k.view(S, 2, 64)[:, 0], want) and torch.equal(v.view(S, 2, 64)[:, 0], -want)
    st = Setup([5, 40], 16, 2, 64)
    run_commit(st, [5, 4], trees([5, 4], 2), [2, 3])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_sequences_shorter_than_their_trees(n, group, heads, dim, fmt):
    """The nodes that would stand before the first position are not there; a row that sees no other gives zeros."""
    need_gpu()
    say(f"{n} nodes of {heads} x {group} x {dim} {fmt} over fewer positions")
    lens = [0, n // 2, n - 1]
    st = Setup(lens, 16, heads, dim, fmt, seed=3)
    starts, masks = [0, n, 2 * n, 3 * n], trees([n] * 3, 5)
    scale = 1 / math.sqrt(dim)
    q = queries(3 * n, heads * group, dim, 4, 2.0 / scale)
    out = torch.full_like(q, 7.0)
    call(st, q, starts, masks, out, n, scale=scale)
    assert ops.device_errors() == 0
    # the same as trees of the nodes that are there, each at its position
    short = [[masks[s * n + i] >> (n - lens[s]) for i in range(n)] for s in range(3)]
    for s in range(3):
        rows = [i for i in range(n) if short[s][i]]
        assert (out[[s * n + i for i in range(n) if not short[s][i]]] == 0).all()
        if not rows:
            continue
        k, v = st.values()
        sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
        for i in rows:
            pos = [p for p in range(lens[s]) if short[s][i] >> p & 1]
            page, slot = torch.tensor([st.state.table[s][p // 16] for p in pos], device=DEV), torch.tensor([p % 16 for p in pos], device=DEV)
            kr, vr = (t[page, slot].double() * (1 if x is None else x.double()[:, None]) for t, x in zip((k, v), sc))
            qh = q[s * n + i].double().view(heads, group, dim)
            kr, vr = kr.permute(1, 2, 0).contiguous(), vr.permute(1, 0, 2).contiguous()
            w = torch.softmax(torch.matmul(qh, kr) * scale, -1)
            check(out[s * n + i], torch.matmul(w, vr).reshape(heads * group, dim), torch.matmul(w, vr.abs()).reshape(heads * group, dim),
                  (torch.matmul(qh.abs(), kr.abs()) * scale).amax(-1).reshape(heads * group), dim)


def test_commit_of_more_work_than_a_sequences_workgroups():
    need_gpu()
    say("commit of 20 layers of 33 heads of 512 dims")
    st = Setup([12 + 20, 7], 4, 33, 512, layers=20)
    run_commit(st, [20, 3], trees([20, 3], 2), [17, 2])
