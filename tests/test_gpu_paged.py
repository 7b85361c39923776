"""The paged KV cache on the GPU: attention of new rows against a float64 evaluation, the append's bits, the calls that
change the cache's state against a plain model, and runs of them together."""
import itertools
import random

import pytest

import paged_model as pm
from gpu_util import need_gpu, say, torch
from moa_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def pool(layers, pages, slots, heads, dim, dtype, layout):
    """K and V views [layers, pages, slots, heads, dim] of a layout: nhd (dense), hnd (heads outside slots), pairs (K
    and V pages side by side in one allocation), slots (K and V side by side in every slot)."""
    if layout == "nhd":
        return tuple(torch.zeros((layers, pages, slots, heads, dim), dtype=dtype, device=DEV) for _ in range(2))
    if layout == "hnd":
        return tuple(torch.zeros((layers, pages, heads, slots, dim), dtype=dtype, device=DEV).transpose(2, 3) for _ in range(2))
    if layout == "pairs":
        t = torch.zeros((layers, pages, 2, slots, heads, dim), dtype=dtype, device=DEV)
        return t[:, :, 0], t[:, :, 1]
    t = torch.zeros((layers, pages, slots, 2, heads, dim), dtype=dtype, device=DEV)
    return t[:, :, :, 0], t[:, :, :, 1]


class Setup:
    """A cache with sequences of the given lengths in shuffled pages, and its plain state."""

    def __init__(self, lens, slots, heads, dim, fmt="bf16", layers=1, seed=0, spare=3, columns=None, layout="nhd", poison=False):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.slots, self.heads, self.dim, self.layers = fmt, slots, heads, dim, layers
        used = [pm.pages_of(n, slots) for n in lens]
        pages, columns = sum(used) + spare, columns or max(used + [1])
        order = torch.randperm(pages, generator=g).tolist()
        table, refs = [], [0] * pages
        for n in used:
            table.append([order.pop() for _ in range(n)] + [-7] * (columns - n))
            for p in table[-1][:n]:
                refs[p] = 1
        self.state = pm.State(table, lens, refs, slots)
        self.table, self.lens, self.refs = i32(table), i32(lens), i32(refs)
        dtype = torch.bfloat16 if fmt == "bf16" else torch.float8_e4m3fn
        self.k, self.v = pool(layers, pages, slots, heads, dim, dtype, layout)
        gd = torch.Generator(device=DEV).manual_seed(seed + 1)
        for t in (self.k, self.v):
            x = torch.randn(t.shape, generator=gd, device=DEV)
            t.copy_(x.to(torch.bfloat16) if fmt == "bf16" else (x * 60).clamp(-448, 448).to(dtype))
        self.k_scale = self.v_scale = None
        if fmt == "e4m3":
            self.k_scale, self.v_scale = ((torch.rand((layers, heads), generator=gd, device=DEV) + 0.5) / 60 for _ in range(2))
        if poison:  # every slot that no position occupies holds NaN
            hold = torch.zeros((pages, slots), dtype=torch.bool)
            for s, n in enumerate(lens):
                for t in range(n):
                    hold[table[s][t // slots], t % slots] = True
            bad = ~hold.to(DEV)
            for t in (self.k, self.v):
                b = t if fmt == "bf16" else t.view(torch.uint8)
                b[:, bad] = float("nan") if fmt == "bf16" else 0x7F
        self.cache = ops.PagedCache(self.k, self.v, self.table, self.lens, self.refs, self.k_scale, self.v_scale)

    def values(self, layer=0):
        return self.k[layer].float(), self.v[layer].float()

    def check_state(self):
        """Everything in use: lengths, reference counts, and the table up to each sequence's pages."""
        assert self.lens.tolist() == self.state.lens
        assert self.refs.tolist() == self.state.refs
        for s, row in enumerate(self.table.tolist()):
            n = pm.pages_of(self.state.lens[s], self.slots)
            assert row[:n] == self.state.table[s][:n], f"sequence {s}"


def queries(rows, heads, dim, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((rows, heads, dim), generator=g, device=DEV) * spread / dim ** 0.5).to(torch.bfloat16)


def starts_of(rows, first=0):
    return [first] + list(itertools.accumulate(rows, initial=first))[1:]


def check_rows(got, want, a, d, dim, rows=None):
    """|got - want| within: half a bf16 step of the result (2^-8 relative); weights rounded to bf16, at most 2^-8 of each,
    which moves the result by at most 2^-8 a; scores rounded as f32 sums of `dim` products (dim + 4 roundings of 2^-24
    relative to sum |q k|), which moves every weight and the sum by that much: twice; exponentials, sums and the
    division in f32: 2^-18 of a covers them (exp2 of a rounded argument below 2^7, sums of up to 2^15 weights)."""
    sel = slice(None) if rows is None else rows
    got, want, a, d = got.double()[sel], want[sel], a[sel], d[sel]
    assert torch.isfinite(got).all()
    tol = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * a * (2.0 ** -8 + 2.0 ** -18 + 2 * (dim + 4) * 2.0 ** -24 * d[..., None]) + 1e-30
    over = ((got - want).abs() - tol).max().item() if got.numel() else 0.0
    assert over <= 0, f"beyond the tolerance by {over}; worst |d| {(got - want).abs().max().item()}"


def attend(st, rows, heads, window=0, scale=1.0, seed=5, first=0, tail=0, max_rows=None, layer=0, q=None, out=None):
    """One call on a Setup; checks every row, and that rows outside the sequences keep what they held."""
    starts = starts_of(rows, first)
    R = starts[-1] + tail
    q = queries(R, heads, st.dim, seed, 2.0 / scale) if q is None else q
    out = torch.full((R, heads, st.dim), 123.0, dtype=torch.bfloat16, device=DEV) if out is None else out
    qc = q.clone()
    ops.paged_attention(q, st.cache, i32(starts), out, layer=layer, window=window, scale=scale, max_rows=max_rows)
    assert ops.device_errors() == 0
    k, v = st.values(layer)
    sc = (None, None) if st.k_scale is None else (st.k_scale[layer], st.v_scale[layer])
    want, a, d = pm.attention(qc, k, v, st.state.table, st.state.lens, starts, st.slots, window, scale, *sc)
    inside = slice(first, starts[-1])
    check_rows(out, want, a, d, st.dim, inside)
    for t in (out[:first], out[starts[-1]:]):
        assert out.data_ptr() == q.data_ptr() or (t == 123.0).all()
    return out


LAYOUTS = [(2, 8, 256), (16, 1, 512), (4, 8, 128), (1, 3, 64), (7, 2, 128), (12, 2, 64), (1, 2, 512), (5, 1, 256), (40, 1, 64)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("group,heads,dim", LAYOUTS)
def test_single_tokens_of_ragged_sequences(group, heads, dim, fmt):
    need_gpu()
    say(f"paged attention tokens G{group} x {heads} x {dim} {fmt}")
    lens = [1, 2, 31, 32, 33, 127, 128, 129, 700, 0, 2051]
    st = Setup(lens, 24, heads, dim, fmt, seed=1, poison=True)
    attend(st, [1] * len(lens), group * heads, max_rows=1)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("group,heads,dim", LAYOUTS)
def test_chunks_beside_tokens(group, heads, dim, fmt):
    need_gpu()
    say(f"paged attention mixed G{group} x {heads} x {dim} {fmt}")
    rows = [1, 130, 0, 3, 64, 1, 17]
    lens = [600, 130, 50, 3, 371, 1, 16]  # the last has a row before position 0
    st = Setup(lens, 40, heads, dim, fmt, seed=2, poison=True)
    attend(st, rows, group * heads, first=2, tail=3)


@pytest.mark.parametrize("window", [1, 16, 100, 129, 1024])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_window(window, fmt):
    need_gpu()
    say(f"paged attention window {window} {fmt}")
    rows, lens = [1, 2, 150, 0, 1, 77], [1500, 2, 900, 5, 0, 77]
    st = Setup(lens, 48, 8, 256, fmt, seed=3, poison=True)
    attend(st, rows, 16, window=window)


@pytest.mark.parametrize("slots", [1, 7, 16, 32, 64, 100, 512])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
def test_page_sizes_and_layouts(slots, layout):
    need_gpu()
    say(f"paged attention pages of {slots}, {layout}")
    for fmt, dim in (("bf16", 128), ("e4m3", 256)):
        rows, lens = [1, 90, 4], [333, 290, 64]
        st = Setup(lens, slots, 2, dim, fmt, layers=2, seed=4, layout=layout, poison=True)
        attend(st, rows, 8, layer=1)


@pytest.mark.parametrize("group,heads,dim,fmt", [(16, 1, 512, "bf16"), (2, 8, 256, "e4m3"), (4, 2, 128, "bf16")])
def test_long_sequences_split(group, heads, dim, fmt):
    need_gpu()
    say(f"paged attention long G{group} x {heads} x {dim} {fmt}")
    for rows, lens in (([1], [32768]), ([4, 1], [20000, 3]), ([70], [9000]), ([300, 1, 2], [5000, 8001, 1])):
        st = Setup(lens, 512, heads, dim, fmt, seed=6)
        attend(st, rows, group * heads, max_rows=max(rows))


def test_many_sequences():
    need_gpu()
    say("paged attention of 700 sequences, most without rows")
    r = random.Random(1)
    lens = [r.randrange(0, 90) for _ in range(700)]
    rows = [r.choice([0, 0, 0, 1, 1, 2, 30]) if n else 0 for n in lens]
    rows = [min(n, x) for n, x in zip(lens, rows)]
    st = Setup(lens, 16, 2, 64, seed=7, poison=True)
    attend(st, rows, 8)


def test_rows_apart_and_in_place():
    need_gpu()
    say("paged attention with strided q and out, and out = q")
    rows, lens = [3, 1, 60], [100, 50, 200]
    st = Setup(lens, 32, 2, 128, seed=8)
    big = queries(64, 12, 128, 9)
    q = big[:, 2:10]
    out = torch.full((64, 3, 8, 128), 9.0, dtype=torch.bfloat16, device=DEV)[:, 1]
    attend(st, rows, 8, q=q, out=out)
    q2 = queries(64, 8, 128, 9)
    attend(st, rows, 8, q=q2, out=q2)


def test_scale_and_large_scores():
    need_gpu()
    say("paged attention with scores of some hundreds, and a negative scale")
    st = Setup([400, 90], 32, 2, 128, seed=10)
    for scale in (1.0, -0.5, 0.0883):
        attend(st, [1, 50], 8, scale=scale, q=queries(51, 8, 128, 11, 60.0))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows", [[4], [100], [1]])
@pytest.mark.parametrize("window", [0, 40])
def test_values_of_positions_that_a_row_does_not_see_never_reach_it(rows, window, fmt):
    """K and V of every new token are infinite or NaN: rows before it are unharmed."""
    need_gpu()
    n = rows[0]
    say(f"paged attention, non-finite later tokens, {n} rows window {window} {fmt}")
    st = Setup([300], 16, 2, 128, fmt, seed=12)
    clean_k, clean_v = (t.clone() for t in st.values())
    last = 299
    page, slot = st.state.table[0][last // 16], last % 16
    for t, x in ((st.k, float("inf")), (st.v, float("nan"))):
        if fmt == "bf16":
            t[0, page, slot] = x
        else:
            t.view(torch.uint8)[0, page, slot] = 0x7F
    if window and n < 300 - window:  # and what the window has left behind
        old = 300 - n - window
        page, slot = st.state.table[0][old // 16], old % 16
        (st.v if fmt == "bf16" else st.v.view(torch.uint8))[0, page, slot] = float("nan") if fmt == "bf16" else 0x7F
    q = queries(n, 8, 128, 13)
    out = torch.zeros_like(q)
    ops.paged_attention(q, st.cache, i32([0, n]), out, window=window)
    assert ops.device_errors() == 0
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    want, a, d = pm.attention(q, clean_k, clean_v, st.state.table, [300], [0, n], 16, window, 1.0, *sc)
    check_rows(out, want, a, d, 128, slice(0, n - 1))
    assert torch.isnan(out[n - 1].float()).any()


def test_offsets_past_32_bits():
    need_gpu()
    say("paged attention and append in a pool of 5.4 GB")
    slots, heads, dim, pages = 64, 8, 256, 20500
    k = torch.empty((1, pages, slots, heads, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    assert k.numel() * 2 > 1 << 32
    table = [[pages - 1, 0, pages - 2, 17000]]
    st = pm.State(table, [250], [0] * pages, slots)
    for p in table[0]:
        k[0, p], v[0, p] = queries(slots, heads, dim, p, 16.0), queries(slots, heads, dim, p + 1, 16.0)
    cache = ops.PagedCache(k, v, i32(table), i32([250]), i32(st.refs))
    nk, nv = queries(40, heads, dim, 3, 16.0), queries(40, heads, dim, 4, 16.0)
    ops.paged_cache_append(cache, nk, nv, i32([0, 40]))
    for i in range(40):
        t = 210 + i
        assert torch.equal(k[0, table[0][t // slots], t % slots], nk[i]) and torch.equal(v[0, table[0][t // slots], t % slots], nv[i])
    for n in (1, 40):
        q = queries(n, 16, dim, 5)
        out = torch.empty_like(q)
        ops.paged_attention(q, cache, i32([0, n]), out)
        assert ops.device_errors() == 0
        low = i32(sorted(set(table[0]))).long()
        small = {int(p): i for i, p in enumerate(low)}
        want, a, d = pm.attention(q, k[0, low].float(), v[0, low].float(), [[small[p] for p in table[0]]], [250], [0, n], slots, 0, 1.0)
        check_rows(out, want, a, d, dim)


# ------------------------------------------------------------------------------- bad device arguments

@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("bad", ["page_high", "page_negative", "len_negative", "len_long", "rows_over", "row_end"])
def test_bad_sequences_are_left_out(bad, n):
    need_gpu()
    say(f"paged attention, {bad}, {n} rows")
    st = Setup([200, 210, 220], 16, 2, 128, seed=14, columns=14)
    table, lens, starts, max_rows = [list(r) for r in st.state.table], list(st.state.lens), [0, n, 2 * n, 3 * n], n
    if bad == "page_high":
        table[1][2] = len(st.state.refs)
    elif bad == "page_negative":
        table[1][2] = -1
    elif bad == "len_negative":
        lens[1] = -3
    elif bad == "len_long":
        lens[1] = 14 * 16 + 1
    elif bad == "rows_over":
        starts, max_rows = [0, n, 3 * n + 1, 4 * n + 1], 2 * n
    elif bad == "row_end":
        starts = [0, n, 2 * n, 9 * n]
    st.table.copy_(i32(table))
    st.lens.copy_(i32(lens))
    R = 4 * n + 1
    q = queries(R, 8, 128, 15)
    out = torch.full_like(q, 123.0)
    ops.paged_attention(q, st.cache, i32(starts), out, max_rows=max_rows)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    k, v = st.values()
    left = 2 if bad == "row_end" else 1
    ok_lens = [st.state.lens[s] for s in range(3)]
    ok_starts = [min(x, R) for x in starts]
    want, a, d = pm.attention(q, k, v, st.state.table, ok_lens, ok_starts, 16, 0, 1.0)
    for s in range(3):
        rows = slice(ok_starts[s], ok_starts[s + 1])
        if s == left:
            assert (out[rows] == 123.0).all()
        else:
            check_rows(out, want, a, d, 128, rows)
    assert (out[ok_starts[3]:] == 123.0).all()


def test_append_leaves_out_bad_rows():
    need_gpu()
    say("append: positions and pages out of range")
    st = Setup([20, 3, 40], 16, 2, 64, seed=16, columns=3)
    st.table[2, 2] = 1 << 30
    before_k, before_v = st.k.clone(), st.v.clone()
    k, v = queries(19, 2, 64, 1, 8.0), queries(19, 2, 64, 2, 8.0)
    ops.paged_cache_append(st.cache, k, v, i32([1, 3, 8, 18]))  # 5 rows of a 3-long sequence; the third's end in a bad page
    assert ops.device_errors() == _lib.DEVERR_PAGED
    for m, s, t in pm.positions([1, 3, 8, 18], [20, 3, 40]):
        if t >= 0 and not (s == 2 and t >= 32):
            p = st.state.table[s][t // 16]
            before_k[0, p, t % 16], before_v[0, p, t % 16] = k[m], v[m]
    assert torch.equal(st.k, before_k) and torch.equal(st.v, before_v)


# ------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("layout", ["nhd", "hnd", "slots"])
@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (3, 64), (5, 128)])
def test_append_bits(heads, dim, layout):
    need_gpu()
    say(f"append {heads} x {dim} {layout}")
    rows, lens = [1, 70, 0, 5], [33, 70, 12, 300]
    starts = starts_of(rows)
    for fmt in ("bf16", "e4m3"):
        st = Setup(lens, 24, heads, dim, fmt, layers=2, seed=17, layout=layout)
        want_k, want_v = st.k.clone(), st.v.clone()
        wide = queries(starts[-1], 2 * heads + 1, dim, 18, dim ** 0.5)
        k, v = wide[:, 1:1 + heads], wide[:, 1 + heads:]
        if fmt == "e4m3":  # values over the largest code, ties, signed zeros, infinities and NaN
            special = torch.tensor([1e9, -1e9, 0.0, -0.0, float("inf"), float("-inf"), float("nan"), 2.0 ** -30], device=DEV)
            wide[2].view(-1)[:8 * ((2 * heads + 1) * dim // 8)] = special.repeat((2 * heads + 1) * dim // 8).to(torch.bfloat16)
        ops.paged_cache_append(st.cache, k, v, i32(starts), layer=1)
        assert ops.device_errors() == 0
        for x, want, scale in ((k, want_k, st.k_scale), (v, want_v, st.v_scale)):
            if fmt == "e4m3":
                x = (x.float() / scale[1][:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                want = want.view(torch.uint8)
            for m, s, t in pm.positions(starts, lens):
                want[1, st.state.table[s][t // 24], t % 24] = x[m]
        for got, want in ((st.k, want_k), (st.v, want_v)):
            if fmt == "e4m3":
                got, want = got.view(torch.uint8), want.view(torch.uint8)
                nan = (want & 0x7F) == 0x7F  # a NaN's sign is free
                assert torch.equal((got & 0x7F) == 0x7F, nan) and torch.equal(got[~nan], want[~nan])
            else:
                assert torch.equal(got.view(torch.int16), want.view(torch.int16))


# ------------------------------------------------------------------------------------- state changes

def move_pages(st, k, v):
    for a, b in st.state.moves:
        k[:, b], v[:, b] = k[:, a].clone(), v[:, a].clone()


def raw(t):
    return t.view(torch.int16) if t.dtype == torch.bfloat16 else t.view(torch.uint8)


def test_reserve_takes_the_lowest_free_pages():
    need_gpu()
    say("reserve")
    st = Setup([10, 0, 33, 16], 16, 1, 64, seed=19, spare=40, columns=30)
    for new in ([1, 1, 1, 1], [0, 0, 0, 0], [0, 100, 0, 300], [6, 0, 14, 0]):
        ops.paged_cache_reserve(st.cache, i32(new))
        assert st.state.reserve(new) and ops.device_errors() == 0
        st.check_state()


@pytest.mark.parametrize("new", [[0, 0, -1, 0], [0, 0, 0, 30 * 16], [16 * 20, 16 * 20, 16 * 20, 0], [2 ** 31 - 1, 0, 0, 0]])
def test_reserve_is_all_or_nothing(new):
    need_gpu()
    say(f"reserve refused {new}")
    st = Setup([10, 0, 33, 16], 16, 1, 64, seed=19, spare=40, columns=30)
    before = st.table.clone()
    ops.paged_cache_reserve(st.cache, i32(new))
    assert ops.device_errors() == _lib.DEVERR_PAGED and not st.state.reserve(new)
    st.check_state()
    assert torch.equal(st.table, before)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_fork_shares_full_pages_and_copies_the_last(layout, fmt):
    need_gpu()
    say(f"fork {layout} {fmt}")
    st = Setup([70, 48, 5, 0, 0, 0, 0, 0, 0], 16, 2, 64, fmt, layers=3, seed=20, spare=9, layout=layout)
    k, v = raw(st.k).clone(), raw(st.v).clone()
    parents, children = [0, 0, 1, 2, 3], [8, 4, 5, 6, 7]
    ops.paged_cache_fork(st.cache, i32(parents), i32(children))
    assert ops.device_errors() == 0 and st.state.fork(parents, children)
    st.check_state()
    move_pages(st, k, v)
    assert torch.equal(raw(st.k), k) and torch.equal(raw(st.v), v)
    attend(st, [1 if n else 0 for n in st.state.lens], 4, layer=2)
    # the parents and the children grow apart
    new = [3, 0, 0, 0, 3, 16, 20, 0, 1]
    ops.paged_cache_reserve(st.cache, i32(new))
    assert st.state.reserve(new)
    st.check_state()


@pytest.mark.parametrize("parents,children", [([0], [9]), ([-1], [3]), ([0], [1]), ([0, 0], [4, 4]), ([3, 0], [4, 3]),
                                              ([0, 2, 2, 0], [3, 4, 5, 6]), ([3], [3])])
def test_fork_is_all_or_nothing(parents, children):
    need_gpu()
    say(f"fork refused {parents} {children}")
    st = Setup([70, 48, 5, 0, 0, 0, 0, 0, 0], 16, 2, 64, layers=2, seed=21, spare=3)
    k, table = st.k.clone(), st.table.clone()
    ops.paged_cache_fork(st.cache, i32(parents), i32(children))
    assert ops.device_errors() == _lib.DEVERR_PAGED and not st.state.fork(parents, children)
    st.check_state()
    assert torch.equal(st.k, k) and torch.equal(st.table, table)


def test_free_counts_shared_pages_once_per_sequence():
    need_gpu()
    say("free")
    st = Setup([70, 48, 0, 5, 0], 16, 1, 64, seed=22, spare=9)
    ops.paged_cache_fork(st.cache, i32([0, 0]), i32([2, 4]))
    assert st.state.fork([0, 0], [2, 4])
    for seqs in ([0], [2, 2, 1], [2], [4, 3, 4, 3]):
        ops.paged_cache_free(st.cache, i32(seqs))
        st.state.free(list(dict.fromkeys(seqs)))
        assert ops.device_errors() == 0
        st.check_state()
    assert not any(st.refs.tolist())
    ops.paged_cache_free(st.cache, i32([5, -1, 1]))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    st.check_state()


def test_free_keeps_a_wrong_count_at_zero():
    need_gpu()
    say("free of pages whose count is wrong")
    st = Setup([40], 16, 1, 64, seed=23)
    st.refs[st.state.table[0][1]] = 0
    ops.paged_cache_free(st.cache, i32([0]))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert not any(st.refs.tolist()) and st.lens.tolist() == [0]


@pytest.mark.parametrize("layout", ["nhd", "hnd", "pairs", "slots"])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_compact(layout, fmt):
    need_gpu()
    say(f"compact {layout} {fmt}")
    st = Setup([70, 48, 5, 0, 200, 31], 16, 2, 64, fmt, layers=2, seed=24, spare=30, layout=layout)
    ops.paged_cache_fork(st.cache, i32([4]), i32([3]))
    assert st.state.fork([4], [3])
    for gone in ([0], [4], [], [3, 2], [1, 5]):
        k, v = raw(st.k).clone(), raw(st.v).clone()
        if gone:
            ops.paged_cache_free(st.cache, i32(gone))
            st.state.free(gone)
        ops.paged_cache_compact(st.cache)
        st.state.compact()
        assert ops.device_errors() == 0
        st.check_state()
        move_pages(st, k, v)
        assert torch.equal(raw(st.k), k) and torch.equal(raw(st.v), v)


def test_compact_of_many_pages():
    need_gpu()
    say("compact 40000 pages of one slot")
    r = random.Random(2)
    st = Setup([r.randrange(0, 800) for _ in range(90)], 1, 1, 64, seed=25, spare=9000)
    gone = r.sample(range(90), 40)
    k, v = st.k.clone(), st.v.clone()
    ops.paged_cache_free(st.cache, i32(gone))
    ops.paged_cache_compact(st.cache)
    st.state.free(gone)
    st.state.compact()
    assert ops.device_errors() == 0
    st.check_state()
    k[:, [b for _, b in st.state.moves]] = k[:, [a for a, _ in st.state.moves]]
    v[:, [b for _, b in st.state.moves]] = v[:, [a for a, _ in st.state.moves]]
    assert torch.equal(st.k, k) and torch.equal(st.v, v)
    new = [50] * 90
    ops.paged_cache_reserve(st.cache, i32(new))
    done = st.state.reserve(new)
    assert ops.device_errors() == (0 if done else _lib.DEVERR_PAGED)
    st.check_state()


@pytest.mark.parametrize("seed", range(4))
def test_a_run_of_calls_in_any_order(seed):
    """A cache lives through 60 random calls, refused ones among them; the model follows, and the attention of every
    sequence's last rows reads the values that were appended."""
    need_gpu()
    say(f"paged cache, random calls, seed {seed}")
    r = random.Random(seed)
    S, slots, heads, dim = 9, 16, 2, 64
    st = Setup([0] * S, slots, heads, dim, layers=2, seed=seed, spare=60, columns=20)
    k, v = st.k.clone(), st.v.clone()
    for step in range(60):
        what = r.choice(["grow", "grow", "fork", "free", "compact"])
        err, st.state.moves = True, []
        if what == "grow":
            new = [r.choice([0, 1, 1, 7, 40]) for _ in range(S)]
            ops.paged_cache_reserve(st.cache, i32(new))
            if not st.state.reserve(new):
                new = [0] * S
                err = False
            starts = starts_of(new)
            nk, nv = queries(starts[-1], heads, dim, step, 8.0), queries(starts[-1], heads, dim, step + 99, 8.0)
            for layer in range(2):
                ops.paged_cache_append(st.cache, nk, nv, i32(starts), layer=layer)
            for m, s, t in pm.positions(starts, st.state.lens):
                p = st.state.table[s][t // slots]
                k[:, p, t % slots], v[:, p, t % slots] = nk[m], nv[m]
        elif what == "fork":
            p, c = [r.randrange(S) for _ in range(2)], [r.randrange(S) for _ in range(2)]
            ops.paged_cache_fork(st.cache, i32(p), i32(c))
            err = st.state.fork(p, c)
            move_pages(st, k, v)
        elif what == "free":
            gone = r.sample(range(S), 2)
            ops.paged_cache_free(st.cache, i32(gone))
            st.state.free(gone)
        else:
            ops.paged_cache_compact(st.cache)
            st.state.compact()
            move_pages(st, k, v)
        assert ops.device_errors() == (0 if err else _lib.DEVERR_PAGED), what
        st.check_state()
        assert torch.equal(st.k, k) and torch.equal(st.v, v), what
    attend(st, [min(n, 3) for n in st.state.lens], 4, layer=1)


# ------------------------------------------------------------------- streams, graphs, the whole step

def test_a_captured_step_replays():
    """Reserve, append and attention captured once; each replay grows the sequences by one token and gives the eager
    results, with eager work between the replays."""
    need_gpu()
    say("paged step in a graph")
    ops.init(0)
    a = Setup([100, 7, 900], 16, 2, 128, seed=30, spare=40, columns=70)
    b = Setup([100, 7, 900], 16, 2, 128, seed=30, spare=40, columns=70)
    q, k, v = queries(3, 8, 128, 1), queries(3, 2, 128, 2, 11.0), queries(3, 2, 128, 3, 11.0)
    one, starts = i32([1, 1, 1]), i32([0, 1, 2, 3])
    out_a, out_b = torch.empty_like(q), torch.empty_like(q)

    def step(st, out):
        ops.paged_cache_reserve(st.cache, one)
        ops.paged_cache_append(st.cache, k, v, starts)
        ops.paged_attention(q, st.cache, starts, out, max_rows=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(a, out_a)
    for i in range(5):
        q.copy_(queries(3, 8, 128, 40 + i))
        k.copy_(queries(3, 2, 128, 50 + i, 11.0))
        graph.replay()
        step(b, out_b)
        assert b.state.reserve([1, 1, 1])
        torch.cuda.synchronize()
        assert torch.equal(out_a, out_b) and torch.equal(a.lens, b.lens) and torch.equal(a.table, b.table)
        assert torch.equal(a.k, b.k) and torch.equal(a.refs, b.refs)
        attend(b, [30, 7, 100], 8, seed=i)  # the same scratch between the replays
    assert ops.device_errors() == 0


def test_a_captured_chunk_and_state_calls_replay():
    need_gpu()
    say("paged chunk attention, fork, free and compact in a graph")
    ops.init(0)
    st = Setup([500, 0, 300], 16, 2, 128, seed=31, spare=50, columns=40)
    start = [t.clone() for t in (st.table, st.lens, st.refs, st.k, st.v)]
    q = queries(260, 8, 128, 1)
    out = torch.empty_like(q)
    parents, children, gone, starts = i32([0]), i32([1]), i32([0]), i32([0, 0, 200, 260])

    def step():
        for t, x in zip((st.table, st.lens, st.refs, st.k, st.v), start):
            t.copy_(x)
        ops.paged_cache_fork(st.cache, parents, children)
        ops.paged_cache_free(st.cache, gone)
        ops.paged_cache_compact(st.cache)
        ops.paged_attention(q, st.cache, starts, out, max_rows=200)

    step()
    assert st.state.fork([0], [1])
    st.state.free([0])
    st.state.compact()
    st.check_state()
    want = [t.clone() for t in (out, st.table, st.lens, st.refs)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, x in zip((out, st.table, st.lens, st.refs), want):
            assert torch.equal(t, x)
        attend(st, [0, 20, 1], 8)
    assert ops.device_errors() == 0


def test_calls_follow_the_current_stream():
    need_gpu()
    say("paged calls on a side stream")
    st = Setup([100, 40], 16, 2, 128, seed=32, spare=10, columns=20)
    side = torch.cuda.Stream()
    big = torch.randn((4096, 4096), device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big
            big = big / big.norm()
        nk = (queries(2, 2, 128, 1, 11.0).float() + big[0, 0] * 0).to(torch.bfloat16)
        ops.paged_cache_reserve(st.cache, i32([1, 1]))
        ops.paged_cache_append(st.cache, nk, nk, i32([0, 1, 2]))
        assert st.state.reserve([1, 1])
        attend(st, [1, 1], 8)
    st.check_state()


def test_a_sliding_layer_over_pages_gives_what_the_ring_gives():
    """QKV of two sequences into scratch rings, their rows appended to the cache, attention and O: the ring's own
    attention of the same tokens gives the same result within both calls' rounding."""
    need_gpu()
    say("sliding layer: QKV -> append -> paged attention -> O, against the ring")
    from gpu_util import dev, dev_zeros
    from moa_amd import synth
    lens, M = [40, 9], [40, 9]
    st = Setup([0, 0], 64, 8, 256, seed=40, spare=4, columns=2)
    ops.paged_cache_reserve(st.cache, i32(M))
    st.state.reserve(M)
    layers, ring, q_all = [], [], []
    for s, m in enumerate(M):
        d = synth.cfg_qkv(seed=3, M=m, pos=0)
        kc, vc, q = dev_zeros(1024 * 2048), dev_zeros(1024 * 2048), dev_zeros(m * 4096)
        ops.sliding_project_qkv(*[dev(d[n]) for n in ("x", "q_weight", "k_weight", "v_weight", "q_weight_scale", "k_weight_scale",
                                                      "v_weight_scale", "input_rms_weight", "q_rms_weight", "k_rms_weight")],
                                i32([0]), i32([0]), dev(d["cos"]), dev(d["sin"]), kc, vc, q)
        mask = (torch.arange(1024, device=DEV)[None] <= torch.arange(m, device=DEV)[:, None]).float()
        o = dev_zeros(m * 4096)
        ops.sliding_attention(q, kc, vc, mask, o)
        ring.append(o.view(torch.bfloat16).view(m, 16, 256))
        layers.append([t.view(torch.bfloat16).view(1024, 8, 256)[:m] for t in (kc, vc)])
        q_all.append(q.view(torch.bfloat16).view(m, 16, 256))
    starts = i32(starts_of(M))
    k, v, q = torch.cat([a for a, _ in layers]), torch.cat([b for _, b in layers]), torch.cat(q_all)
    ops.paged_cache_append(st.cache, k, v, starts)
    out = torch.empty_like(q)
    ops.paged_attention(q, st.cache, starts, out, window=1024, max_rows=max(M))
    assert ops.device_errors() == 0
    kk, vv = st.values()
    want, a, d = pm.attention(q, kk, vv, st.state.table, lens, starts_of(M), 64, 1024, 1.0)
    check_rows(out, want, a, d, 256)
    check_rows(torch.cat(ring), want, a, d, 256)
    o = synth.cfg_o(seed=4, M=sum(M))
    res = [dev(o["residual"]) for _ in range(2)]
    for r, x in zip(res, (out, torch.cat(ring))):
        ops.sliding_attention_output(x.reshape(sum(M), 4096), dev(o["post_attn_rms_weight"]), dev(o["o_weight"]), dev(o["o_weight_scale"]), r)
    a, b = (r.view(torch.bfloat16).float() for r in res)
    assert torch.isfinite(a).all() and (a - b).abs().max() <= 0.05 * b.abs().max()


def test_a_full_layers_pages_are_pages_of_the_cache():
    """full_project_qkv writes into the cache's own page; paged_attention then gives full_attention's out / sum."""
    need_gpu()
    say("full layer: QKV into a page of the cache, paged attention against full_attention")
    from gpu_util import dev, dev_zeros
    from moa_amd import synth
    d = synth.cfg_full_qkv(seed=5, M=3, pos=700)
    st = Setup([703], 512, 1, 512, seed=41, layers=1)
    page = st.state.table[0][1]
    q = dev_zeros(3 * 8192)
    ops.full_project_qkv(dev(d["x"]), dev(d["q_weight"]), dev(d["k_weight"]), dev(d["q_weight_scale"]), dev(d["k_weight_scale"]),
                         dev(d["input_rms_weight"]), dev(d["q_rms_weight"]), dev(d["k_rms_weight"]), i32([d["kv_offset"]]),
                         i32([d["rope_offset"]]), dev(d["cos"]), dev(d["sin"]), st.k[0, page].view(torch.int16),
                         st.v[0, page].view(torch.int16), q)
    q = q.view(torch.bfloat16).view(3, 16, 512)
    out = torch.empty_like(q)
    ops.paged_attention(q, st.cache, i32([0, 3]), out)
    assert ops.device_errors() == 0
    k, v = st.values()
    want, a, dd = pm.attention(q, k, v, st.state.table, [703], [0, 3], 512, 0, 1.0)
    check_rows(out, want, a, dd, 512)
    pages = torch.tensor(st.state.table[0], device=DEV)
    masks = torch.stack([(torch.arange(512, device=DEV)[None] + 512 * p <= 700 + torch.arange(3, device=DEV)[:, None]).float() for p in range(2)])
    mx, sm, o = torch.empty(48, device=DEV), torch.empty(48, device=DEV), torch.empty_like(q)
    ops.full_attention(q, st.k[0, pages].contiguous(), st.v[0, pages].contiguous(), masks.contiguous(), mx, sm, o)
    check_rows(o.double() / sm.view(3, 16, 1).double(), want, a, dd, 512)
    # full_attention_output divides by the running sum: with a normalised row it is one
    w = synth.cfg_full_o(seed=6, M=3)
    res = [dev(w["residual"]) for _ in range(2)]
    for r, x, total in zip(res, (out, o), (torch.ones(48, device=DEV), sm)):
        ops.full_attention_output(x, total, dev(w["post_attn_rms_weight"]), dev(w["o_weight"]), dev(w["o_weight_scale"]), r)
    a, b = (r.view(torch.bfloat16).float() for r in res)
    assert torch.isfinite(a).all() and (a - b).abs().max() <= 0.05 * b.abs().max()


def test_calls_of_one_process_repeat_their_bits():
    need_gpu()
    say("paged attention twice, the same bits")
    st = Setup([3000, 70, 1200], 48, 1, 512, seed=33)
    for rows in ([1, 1, 1], [200, 1, 40]):
        q = queries(sum(rows), 16, 512, 2)
        outs = [torch.empty_like(q) for _ in range(2)]
        for o in outs:
            ops.paged_attention(q, st.cache, i32(starts_of(rows)), o, max_rows=max(rows))
            attend(st, [1, 0, 0], 16)
        assert torch.equal(*outs)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,heads,dim", [(2, 8, 256), (4, 2, 128), (1, 1, 512), (90, 2, 128), (40, 1, 512)])
def test_in_place_beside_values_that_a_row_does_not_see(n, heads, dim, fmt):
    """out = q, one short sequence (nothing to merge), V of the last token NaN: the rows before it are right."""
    need_gpu()
    say(f"paged attention in place, non-finite last token, {n} rows of {heads} x {dim} {fmt}")
    length = 100
    st = Setup([length], 16, heads, dim, fmt, seed=21)
    clean_k, clean_v = (t.clone() for t in st.values())
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    at = length if n == 1 else length - 1  # of a single token, what lies behind the sequence
    page, slot = st.state.table[0][at // 16], at % 16
    (st.v if fmt == "bf16" else st.v.view(torch.uint8))[0, page, slot] = float("nan") if fmt == "bf16" else 0x7F
    q = queries(n, 4 * heads, dim, 22)
    want, a, d = pm.attention(q, clean_k, clean_v, st.state.table, [length], [0, n], 16, 0, 1.0, *sc)
    ops.paged_attention(q, st.cache, i32([0, n]), q)
    assert ops.device_errors() == 0
    check_rows(q, want, a, d, dim, slice(0, n - 1 if n > 1 else 1))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,length", [(1, 9000), (4, 9000), (90, 9000), (1, 120000), (40, 100), (3, 100)])
def test_nan_that_a_row_sees_makes_it_nan(n, length, fmt):
    """A query that is NaN gives a NaN row, and so does a visible key or value, split or not; other rows are unharmed."""
    need_gpu()
    say(f"paged attention, visible NaN, {n} rows over {length} positions {fmt}")
    st = Setup([length], 64, 2, 128, fmt, seed=23)
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    q = queries(n, 8, 128, 24)
    want, a, d = pm.attention(q, *st.values(), st.state.table, [length], [0, n], 64, 0, 1.0, *sc)
    out = torch.zeros_like(q)
    sick = q.clone()
    sick[n // 2, 5] = float("nan")
    ops.paged_attention(sick, st.cache, i32([0, n]), out)
    assert ops.device_errors() == 0
    assert torch.isnan(out[n // 2, 5].float()).all()
    well = torch.ones((n, 8), dtype=torch.bool, device=DEV)
    well[n // 2, 5] = False
    check_rows(out[well], want[well], a[well], d[well], 128)
    page, slot = st.state.table[0][17 // 64], 17
    for t in (st.k, st.v):  # one position, far from where the largest scores may lie
        view = t if fmt == "bf16" else t.view(torch.uint8)
        old = view[0, page, slot].clone()
        view[0, page, slot, 1, 3] = float("nan") if fmt == "bf16" else 0x7F
        ops.paged_attention(q, st.cache, i32([0, n]), out)
        assert ops.device_errors() == 0
        assert torch.isnan(out[:, 4:, 3].float()).all(), "K" if t is st.k else "V"
        check_rows(out[:, :4], want[:, :4], a[:, :4], d[:, :4], 128)
        view[0, page, slot] = old


# --------------------------------------------------------------------------------- ends of the ranges

def test_overlapping_row_starts_are_found():
    need_gpu()
    say("paged attention, row starts that descend")
    st = Setup([900, 900, 900, 900, 900], 32, 2, 64, seed=41)
    q = queries(300, 16, 64, 42)
    out = torch.full_like(q, 123.0)
    ops.paged_attention(q, st.cache, i32([0, 300, 0, 300, 0, 300]), out)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert (out == 123.0).all()
    # 2^31 tiles by the starts' account
    rows = S = 1 << 16
    table = torch.zeros((S, 1), dtype=torch.int32, device=DEV)
    pages = torch.zeros((1, 1, 1024, 1, 64), dtype=torch.bfloat16, device=DEV)
    lens, refs = torch.full((S,), 8, dtype=torch.int32, device=DEV), i32([1])
    cache = ops.PagedCache(pages, pages.clone(), table, lens, refs)
    starts = torch.zeros(S + 1, dtype=torch.int32, device=DEV)
    starts[1::2] = rows
    q = torch.zeros((rows, 128, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.full_like(q, 123.0)
    ops.paged_attention(q, cache, starts, out)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert (out == 123.0).all()


@pytest.mark.parametrize("S,base", [(1, 0), (65, 0), (1500, 2), (2300, 0)])
def test_reserve_fork_free_of_many_sequences(S, base):
    """More sequences and forks than a workgroup has threads."""
    need_gpu()
    say(f"reserve, fork, free of {S} sequences")
    rng = random.Random(S)
    lens = [rng.choice([0, 0, 1, 3, 4, 5, 11]) for _ in range(S)]
    st = Setup(lens, 4, 1, 64, seed=43, spare=5 * S + 20, columns=6)
    new = [rng.choice([0, 1, 2, 4, 9]) for _ in range(S)]
    ops.paged_cache_reserve(st.cache, i32(new))
    assert st.state.reserve(new) and ops.device_errors() == 0
    st.check_state()
    gone = [rng.randrange(S) for _ in range(S // 2 + 1)]  # some twice
    ops.paged_cache_free(st.cache, i32(gone))
    st.state.free(gone)
    assert ops.device_errors() == 0
    st.check_state()
    children = [s for s in range(S) if st.state.lens[s] == 0]
    rng.shuffle(children)
    live = [s for s in range(S) if st.state.lens[s]]
    if live and children:
        parents = [rng.choice(live) for _ in children]
        k = st.k.clone()
        ops.paged_cache_fork(st.cache, i32(parents), i32(children))
        assert st.state.fork(parents, children) and ops.device_errors() == 0
        st.check_state()
        for a, b in st.state.moves:
            k[:, b] = k[:, a]
        assert torch.equal(st.k, k)
    ops.paged_cache_compact(st.cache)
    st.state.compact()
    assert ops.device_errors() == 0
    st.check_state()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,group,dim", [(256, 1, 64), (256, 1, 512), (200, 2, 256), (1, 128, 512), (2, 128, 64), (3, 17, 128)])
def test_many_heads(heads, group, dim, fmt):
    need_gpu()
    say(f"paged attention, {heads} KV heads x {group} of {dim} {fmt}")
    st = Setup([300, 5, 1100], 32, heads, dim, fmt, seed=44)
    attend(st, [1, 1, 1], heads * group)
    attend(st, [20, 1, 2], heads * group, window=200)


@pytest.mark.parametrize("window", [0, 1000, 6000])
@pytest.mark.parametrize("group,heads,dim,fmt", [(16, 1, 512, "bf16"), (2, 2, 256, "e4m3"), (4, 1, 128, "bf16"), (8, 1, 64, "e4m3")])
def test_long_chunks_split(group, heads, dim, fmt, window):
    need_gpu()
    say(f"paged attention, split chunks of {heads} x {group} of {dim} {fmt} window {window}")
    st = Setup([20011, 1, 9000, 300], 64, heads, dim, fmt, seed=45)
    attend(st, [33, 1, 70, 1], heads * group, window=window)
    attend(st, [1, 0, 17, 2], heads * group, window=window, max_rows=17)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", [(1, 4, 2, 128), (3, 1, 1, 512), (50, 4, 2, 128), (40, 8, 1, 512), (60, 2, 1, 64)])
def test_a_bad_page_in_one_part_of_a_split_sequence(n, group, heads, dim, fmt):
    need_gpu()
    say(f"paged attention, a bad page of a split sequence, {n} rows of {heads} x {group} of {dim} {fmt}")
    st = Setup([16000, 15000], 64, heads, dim, fmt, seed=46)
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    q = queries(2 * n, heads * group, dim, 47)
    want, a, d = pm.attention(q, *st.values(), st.state.table, st.state.lens, [0, n, 2 * n], 64, 0, 1.0, *sc)
    good = st.table.clone()
    for at, p in ((3, -1), (100, 1 << 30), (249, len(st.state.refs))):  # the last page of sequence 0 is 249
        st.table.copy_(good)
        st.table[0, at] = p
        out = torch.full_like(q, 123.0)
        ops.paged_attention(q, st.cache, i32([0, n, 2 * n]), out)
        assert ops.device_errors() == _lib.DEVERR_PAGED
        check_rows(out, want, a, d, dim, slice(n, 2 * n))
        assert (out[:n] == 123.0).all()


@pytest.mark.parametrize("S", [64, 65, 1100])
def test_tokens_and_chunks_of_many_sequences(S):
    need_gpu()
    say(f"paged attention, {S} sequences of one to forty rows")
    rng = random.Random(S)
    lens = [rng.choice([0, 1, 2, 40, 300]) for _ in range(S)]
    lens[S // 2] = 5000
    rows = [rng.choice([0, 1, 1, 1, 2, 9, 40]) if n else 0 for n in lens]
    st = Setup(lens, 16, 2, 64, seed=48)
    attend(st, rows, 8, first=3, tail=2)
    attend(st, [min(r, 4) for r in rows], 8, max_rows=4)
    attend(st, rows, 8, window=33, max_rows=40)


def test_offsets_between_31_and_32_bits():
    need_gpu()
    say("paged attention in pools of 3 GB, K and V with other strides")
    slots, heads, dim, pages = 64, 8, 128, 23000
    k = torch.empty((1, pages, slots, heads, dim), dtype=torch.bfloat16, device=DEV)
    v = torch.empty((1, pages, heads, slots, dim), dtype=torch.bfloat16, device=DEV).transpose(2, 3)
    assert 1 << 31 < k.numel() * 2 < 1 << 32
    table = [[pages - 1, 0, pages - 2, 17000]]
    for p in table[0]:
        k[0, p], v[0, p] = queries(slots, heads, dim, p, 11.0), queries(slots, heads, dim, p + 1, 11.0)
    cache = ops.PagedCache(k, v, i32(table), i32([250]), torch.zeros(pages, dtype=torch.int32, device=DEV))
    low = sorted(table[0])
    for n in (1, 40):
        q = queries(n, 16, dim, 5)
        out = torch.empty_like(q)
        ops.paged_attention(q, cache, i32([0, n]), out)
        assert ops.device_errors() == 0
        want, a, d = pm.attention(q, k[0, low].float(), v[0, low].float(), [[low.index(p) for p in table[0]]], [250], [0, n], slots, 0, 1.0)
        check_rows(out, want, a, d, dim)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_layers_of_one_cache(fmt):
    need_gpu()
    say(f"paged append and attention of three layers {fmt}")
    st = Setup([70, 3], 16, 2, 64, fmt, layers=3, seed=49)
    before = raw(st.k).clone()
    nk, nv = queries(5, 2, 64, 1, 8.0), queries(5, 2, 64, 2, 8.0)
    ops.paged_cache_append(st.cache, nk, nv, i32([0, 3, 5]), layer=1)
    after = raw(st.k)
    assert torch.equal(after[0], before[0]) and torch.equal(after[2], before[2]) and not torch.equal(after[1], before[1])
    for layer in range(3):
        attend(st, [20, 3], 8, layer=layer)
        attend(st, [1, 1], 8, layer=layer)


@pytest.mark.parametrize("slots", [1, 3, 4097, 65536])
def test_smallest_and_largest_pages(slots):
    need_gpu()
    say(f"paged cache of {slots} slots a page")
    st = Setup([1, 0], slots, 1, 64, seed=50, spare=6, columns=4)
    for new in ([1, 1], [2 * slots, 0], [0, slots]):
        ops.paged_cache_reserve(st.cache, i32(new))
        fits = st.state.reserve(new)
        assert ops.device_errors() == (0 if fits else _lib.DEVERR_PAGED)
        st.check_state()
    attend(st, [1, 1], 4)
    attend(st, [min(20, st.state.lens[0]), 1], 4, window=5)


def test_calls_without_rows():
    need_gpu()
    say("paged calls of no rows and no sequences")
    st = Setup([0], 16, 2, 128, seed=51, spare=1)
    none = torch.empty((0, 8, 128), dtype=torch.bfloat16, device=DEV)
    kv = torch.empty((0, 2, 128), dtype=torch.bfloat16, device=DEV)
    ops.paged_attention(none, st.cache, i32([0, 0]), none.clone())
    ops.paged_cache_append(st.cache, kv, kv, i32([0, 0]))
    ops.paged_cache_fork(st.cache, i32([]), i32([]))
    ops.paged_cache_free(st.cache, i32([]))
    ops.paged_cache_reserve(st.cache, i32([0]))
    ops.paged_cache_compact(st.cache)
    attend(st, [0], 8, first=1, tail=2)
    attend(st, [2], 8)  # rows of an empty sequence see nothing: zeros
    assert ops.device_errors() == 0
    st.check_state()


def test_two_graphs_take_turns():
    """Two captured calls share the library's scratch; replayed in turn, with eager calls between, each keeps its result."""
    need_gpu()
    say("two paged graphs in turn")
    ops.init(0)
    made = []
    for i, (lens, rows, heads, dim) in enumerate([([9000, 40], [1, 1], 2, 128), ([5000, 300], [60, 1], 1, 512)]):
        st = Setup(lens, 64, heads, dim, seed=52 + i)
        q = queries(sum(rows), 8, dim, 54 + i)
        out, want, starts = torch.empty_like(q), torch.empty_like(q), i32(starts_of(rows))
        ops.paged_attention(q, st.cache, starts, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(q, st.cache, starts, out)
        made.append((graph, out, want, st, q, starts))  # what a graph reads stays alive
    for _ in range(3):
        for graph, out, want, *_ in made:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        attend(made[0][3], [30, 2], 8)
    assert ops.device_errors() == 0


@pytest.mark.parametrize("seed", range(12))
def test_random_shapes(seed):
    need_gpu()
    rng = random.Random(1000 + seed)
    dim, fmt, layout = rng.choice([64, 128, 256, 512]), rng.choice(["bf16", "e4m3"]), rng.choice(["nhd", "hnd", "pairs", "slots"])
    heads, group, slots = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 3, 5, 8, 16, 30]), rng.choice([1, 5, 16, 48, 64, 256])
    S = rng.choice([1, 3, 20, 70])
    lens = [rng.choice([0, 1, rng.randrange(2, 400), rng.randrange(2, 3000)]) for _ in range(S)]
    rows = [min(n, rng.choice([0, 1, 1, 2, 7, rng.randrange(1, 200)])) for n in lens]
    window, scale = rng.choice([0, 0, 1, 31, 512]), rng.choice([1.0, 0.0625, -1.0])
    say(f"paged attention {heads} x {group} of {dim} {fmt} {layout}, {slots} slots, rows {rows} of {lens}, window {window}, scale {scale}")
    st = Setup(lens, slots, heads, dim, fmt, seed=seed, layout=layout, poison=True)
    # poisoned slots are NaN: the oracle reads only the visible ones
    attend(st, rows, heads * group, window=window, scale=scale, first=rng.choice([0, 2]), tail=rng.choice([0, 3]))


def test_the_front_end_refuses():
    """Tensors of a wrong type, shape, device or order never reach the library, and nothing is written."""
    need_gpu()
    say("paged front end refusals")
    st = Setup([20, 3], 16, 2, 64, seed=60, spare=4)
    before = [t.clone() for t in (st.k, st.v, st.table, st.lens, st.refs)]
    q, out, kv = queries(4, 8, 64, 1), queries(4, 8, 64, 2), queries(4, 2, 64, 3)
    starts, held = i32([0, 3, 4]), out.clone()
    make = lambda **kw: ops.PagedCache(**{**dict(k_pages=st.k, v_pages=st.v, page_table=st.table, seq_lens=st.lens,  # noqa: E731
                                                ref_counts=st.refs), **kw})
    codes = st.k.to(torch.float8_e4m3fn)
    scale = torch.ones((1, 2), device=DEV)
    calls = {
        "a page pool on the host": lambda: make(k_pages=st.k.cpu()),
        "a table on the host": lambda: make(page_table=st.table.cpu()),
        "pages of other shapes": lambda: make(v_pages=st.v[:, :-1]),
        "pages of other types": lambda: make(v_pages=codes),
        "f32 pages": lambda: make(k_pages=st.k.float(), v_pages=st.v.float()),
        "head dims apart": lambda: make(k_pages=st.k.transpose(3, 4), v_pages=st.v.transpose(3, 4)),
        "no pages": lambda: make(k_pages=st.k[:, :0], v_pages=st.v[:, :0]),
        "codes without scales": lambda: make(k_pages=codes, v_pages=codes),
        "codes with one scale": lambda: make(k_pages=codes, v_pages=codes, k_scale=scale),
        "scales of another layer count": lambda: make(k_pages=codes, v_pages=codes, k_scale=scale[:, :1], v_scale=scale),
        "scales with bf16": lambda: make(k_scale=scale, v_scale=scale),
        "a table of int64": lambda: make(page_table=st.table.long()),
        "a table with columns apart": lambda: make(page_table=st.table.t()),
        "lengths of another number": lambda: make(seq_lens=i32([1, 2, 3])),
        "counts of another number": lambda: make(ref_counts=st.refs[:-1]),
        "lengths that are a list": lambda: make(seq_lens=[20, 3]),
        "no cache": lambda: ops.paged_cache_compact(st),
        "new tokens of another number": lambda: ops.paged_cache_reserve(st.cache, i32([1])),
        "new tokens of int64": lambda: ops.paged_cache_reserve(st.cache, i32([1, 1]).long()),
        "new tokens on the host": lambda: ops.paged_cache_reserve(st.cache, i32([1, 1]).cpu()),
        "new tokens apart": lambda: ops.paged_cache_reserve(st.cache, i32([1, 0, 1, 0])[::2]),
        "row starts of another number": lambda: ops.paged_cache_append(st.cache, kv, kv, i32([0, 4])),
        "k of other heads": lambda: ops.paged_cache_append(st.cache, q, kv, starts),
        "v of other rows": lambda: ops.paged_cache_append(st.cache, kv, kv[:3], starts),
        "f32 rows": lambda: ops.paged_cache_append(st.cache, kv.float(), kv, starts),
        "flat rows": lambda: ops.paged_cache_append(st.cache, kv.view(4, 128), kv, starts),
        "heads apart": lambda: ops.paged_cache_append(st.cache, queries(4, 4, 64, 3)[:, ::2], kv, starts),
        "dims apart": lambda: ops.paged_cache_append(st.cache, queries(4, 2, 128, 3)[:, :, ::2], kv, starts),
        "rows on top of each other": lambda: ops.paged_cache_append(st.cache, kv[:1].expand(4, 2, 64), kv, starts),
        "a layer behind the last": lambda: ops.paged_cache_append(st.cache, kv, kv, starts, layer=1),
        "a negative layer": lambda: ops.paged_attention(q, st.cache, starts, out, layer=-1),
        "q of other dims": lambda: ops.paged_attention(queries(4, 8, 128, 1), st.cache, starts, out),
        "heads that are no multiple": lambda: ops.paged_attention(q[:, :7].contiguous(), st.cache, starts, out[:, :7].contiguous()),
        "out of other rows": lambda: ops.paged_attention(q, st.cache, starts, out[:3]),
        "out of other heads": lambda: ops.paged_attention(q, st.cache, starts, queries(4, 4, 64, 1)),
        "q on the host": lambda: ops.paged_attention(q.cpu(), st.cache, starts, out),
        "max_rows of zero": lambda: ops.paged_attention(q, st.cache, starts, out, max_rows=0),
        "max_rows over the rows": lambda: ops.paged_attention(q, st.cache, starts, out, max_rows=5),
        "a negative window": lambda: ops.paged_attention(q, st.cache, starts, out, window=-1),
        "an infinite scale": lambda: ops.paged_attention(q, st.cache, starts, out, scale=float("inf")),
        "q that is not aligned": lambda: ops.paged_attention(queries(5, 8, 64, 1).view(-1)[1:1 + q.numel()].view(q.shape), st.cache, starts, out),
        "children of another number": lambda: ops.paged_cache_fork(st.cache, i32([0]), i32([0, 1])),
        "sequences of int64": lambda: ops.paged_cache_free(st.cache, i32([0]).long()),
    }
    for name, call in calls.items():
        with pytest.raises((TypeError, ValueError, _lib.MoaError)):
            call()
            pytest.fail(f"{name} was taken")
    assert ops.device_errors() == 0 and torch.equal(out, held)
    for t, old in zip((st.k, st.v, st.table, st.lens, st.refs), before):
        assert torch.equal(t, old)


def test_joined_records_leave_nothing_for_the_next_call():
    """Single tokens in a window, whose parts are joined by their last workgroup: calls of other shapes, with bad pages and
    with NaN between, and each result stays bit for bit what it was."""
    need_gpu()
    say("paged attention, joined records call after call")
    made = []
    for i, (lens, heads, group, dim, fmt, window) in enumerate([([700], 8, 2, 256, "bf16", 1024), ([1500, 9, 1100, 640], 8, 2, 256, "e4m3", 1024),
                                                                ([300] * 70, 2, 4, 128, "bf16", 0), ([1900], 1, 2, 512, "bf16", 1500)]):
        st = Setup(lens, 16, heads, dim, fmt, seed=70 + i)
        q = queries(len(lens), heads * group, dim, 80 + i)
        out = attend(st, [1] * len(lens), heads * group, window=window, q=q, max_rows=1)
        made.append((st, q, out, i32(range(len(lens) + 1)), window))
    for turn in range(6):
        for st, q, want, starts, window in made:
            got = torch.empty_like(q)
            good = st.table.clone()
            if turn in (1, 4):  # a bad page of the first sequence, inside its window
                st.table[0, (st.state.lens[0] - 1) // 16 - 3 * turn] = -1
            sick = q.clone()
            if turn == 2:
                sick[0, 0] = float("nan")
            ops.paged_attention(sick, st.cache, starts, got, window=window, max_rows=1)
            first = 1 if turn in (1, 2, 4) else 0
            assert ops.device_errors() == (_lib.DEVERR_PAGED if turn in (1, 4) else 0)
            assert torch.equal(got[first:], want[first:])
            if turn == 2:
                assert torch.isnan(got[0, 0].float()).all() and torch.equal(got[0, 1:], want[0, 1:])
            st.table.copy_(good)


@pytest.mark.parametrize("heads,group,dim,fmt", [(8, 2, 256, "bf16"), (8, 1, 128, "e4m3"), (1, 2, 512, "bf16"), (3, 4, 64, "e4m3"), (1, 16, 512, "bf16")])
def test_a_value_before_the_window_never_reaches_a_joined_row(heads, group, dim, fmt):
    """A NaN just before the window shares a tile with its first positions; the sequence is split, its first part is
    computed again, and out is q."""
    need_gpu()
    say(f"paged attention, NaN before the window of a split token, {heads} x {group} of {dim} {fmt}")
    st = Setup([1900, 1500], 16, heads, dim, fmt, seed=90)
    clean = tuple(t.clone() for t in st.values())
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    for s, at in ((0, 897), (1, 499)):  # the windows begin at 900 and 500
        page, slot = st.state.table[s][at // 16], at % 16
        for t in (st.k, st.v):
            (t if fmt == "bf16" else t.view(torch.uint8))[0, page, slot] = float("nan") if fmt == "bf16" else 0x7F
    q = queries(2, heads * group, dim, 91)
    want, a, d = pm.attention(q, *clean, st.state.table, st.state.lens, [0, 1, 2], 16, 1000, 1.0, *sc)
    for _ in range(3):
        out = q.clone()
        ops.paged_attention(out, st.cache, i32([0, 1, 2]), out, window=1000, max_rows=1)
        assert ops.device_errors() == 0
        check_rows(out, want, a, d, dim)


# ------------------------------------------------------------------------- what the weights keep

@pytest.mark.parametrize("n,heads,group,dim,fmt", [
    # single tokens: 32 positions a tile, and 16 (256 dims of bf16, 512 of either type)
    (1, 8, 2, 128, "bf16"), (1, 3, 5, 64, "e4m3"), (4, 2, 4, 256, "e4m3"), (1, 8, 2, 256, "bf16"), (1, 1, 16, 512, "bf16"), (2, 1, 8, 512, "e4m3"),
    # chunks: a wave per 32 rows, and pairs of waves (512 dims)
    (60, 2, 4, 128, "bf16"), (33, 1, 8, 64, "e4m3"), (50, 4, 2, 256, "bf16"), (20, 2, 2, 256, "e4m3"), (40, 1, 16, 512, "bf16"), (64, 1, 3, 512, "e4m3")])
def test_values_that_nearly_cancel(n, heads, group, dim, fmt):
    """Positions come in pairs of opposite values whose weights differ by 2^-10: what is left of a pair is far below the
    rounding of a weight to one bf16 number (2^-8 of it), so every row would have wrong signs with such weights.

    Tolerance, relative to a (the attention of |v|). A score is one product of bf16 numbers, so exact, and below 1: its
    factor (three roundings), the product with it and the distance to the reference are off by at most 5 * 2^-23 together, the
    exponential by 2^-22, which moves a weight by less than 2^-20 of it. Two bf16 parts hold a weight to (2^-8)^2 = 2^-16. The sums of at
    most 64 products lose at most 2^-23 of a each time: 2^-17. The division and the last rounding are relative to the result."""
    need_gpu()
    say(f"paged attention, values that cancel, {n} rows of {heads} x {group} of {dim} {fmt}")
    length = 64
    st = Setup([length], 16, heads, dim, fmt, seed=95)
    g = torch.Generator(device=DEV).manual_seed(96)
    even, step, q0 = (1 + torch.randint(0, 60, (length // 2, heads), generator=g, device=DEV) / 64, 2.0 ** -7, 2.0 ** -3)
    if fmt == "e4m3":
        even, step, q0 = 1 + torch.randint(0, 7, (length // 2, heads), generator=g, device=DEV) / 8, 2.0 ** -3, 2.0 ** -7
        st.k_scale.fill_(1.0)
    sign = torch.randint(0, 2, (length // 2, heads), generator=g, device=DEV) * 2 - 1  # which of a pair weighs more
    k = torch.stack([even, even + step], 1)
    k = torch.where(sign[:, None] > 0, k, k.flip(1)).reshape(length, heads)
    v = torch.randn((length // 2, 1, heads, dim), generator=g, device=DEV).clamp(-3, 3) * (60 if fmt == "e4m3" else 1)
    v = torch.cat([v, -v], 1).reshape(length, heads, dim)
    table = torch.tensor(st.state.table[0], device=DEV)
    t = torch.arange(length, device=DEV)
    kv = torch.zeros((length, heads, dim), device=DEV)
    kv[:, :, dim - 1] = k
    st.k[0, table[t // 16], t % 16] = kv.to(st.k.dtype)
    st.v[0, table[t // 16], t % 16] = v.to(st.v.dtype)
    q = torch.zeros((n, heads * group, dim), dtype=torch.bfloat16, device=DEV)
    q[:, :, dim - 1] = q0
    sc = (None, None) if st.k_scale is None else (st.k_scale[0], st.v_scale[0])
    want, a, _ = pm.attention(q, *st.values(), st.state.table, [length], [0, n], 16, 0, 1.0, *sc)
    out = torch.empty_like(q)
    ops.paged_attention(q, st.cache, i32([0, n]), out)
    assert ops.device_errors() == 0
    assert (want[-1].abs() < 2.0 ** -9 * a[-1]).float().mean() > 0.9  # they do cancel
    over = ((out.double() - want).abs() - 2.0 ** -8 * want.abs() - a * (2.0 ** -16 + 2.0 ** -17 + 2.0 ** -20)).max().item()
    assert over <= 0, f"beyond the tolerance by {over}, relative to a: {((out.double() - want).abs() / a).max().item()}"


# ---------------------------------------------------------------------------- bad row starts and states

@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("bad", [[2 ** 31 - 1, -2 ** 31], [2 ** 31 - 1, -2 ** 31 + 2], [-2 ** 31, 2 ** 31 - 1], [2 ** 30, 2 ** 30 + 1], [-1, 0], [2 ** 31 - 1, 2 ** 31 - 1]])
def test_row_starts_at_the_ends_of_int32(bad, n):
    """Starts whose difference passes 32 bits, or that lie outside the call's rows, in the middle of a call's sequences: those
    sequences are left out, the others' rows are right, and nothing else is written."""
    need_gpu()
    say(f"paged attention, row starts {bad}, {n} rows")
    st = Setup([200, 210, 220, 230, 240], 16, 2, 128, seed=97)
    q = queries(3 * n, 8, 128, 98)
    out = torch.full_like(q, 123.0)
    ops.paged_attention(q, st.cache, i32([0, n, *bad, 2 * n, 3 * n]), out, max_rows=n)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    k, v = st.values()
    for s, rows in ((0, slice(0, n)), (4, slice(2 * n, 3 * n))):
        want, a, d = pm.attention(q[rows], k, v, [st.state.table[s]], [st.state.lens[s]], [0, n], 16, 0, 1.0)
        check_rows(out[rows], want, a, d, 128)
    assert (out[n:2 * n] == 123.0).all()


@pytest.mark.parametrize("starts,written", [([0, 5, 3, 8], {0: (0, 3), 2: (5, 8)}), ([0, 2, -2 ** 31, 8], {2: (2, 8)}), ([0, 2, 2 ** 31 - 1, 8], {0: (0, 2)})])
def test_append_with_row_starts_that_are_out_of_order(starts, written):
    """Rows whose sequence's starts descend or end past the call's rows raise the bit and are not written; those of the others are."""
    need_gpu()
    say(f"append, row starts {starts}")
    st = Setup([40, 50, 60], 16, 2, 64, seed=99)
    want = st.k.clone()
    k = queries(8, 2, 64, 1, 8.0)
    ops.paged_cache_append(st.cache, k, k, i32(starts))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    for s, (m0, m1) in written.items():
        for m in range(m0, m1):
            t = st.state.lens[s] - (starts[s + 1] - m)
            want[0, st.state.table[s][t // 16], t % 16] = k[m]
    assert torch.equal(raw(st.k), raw(want))


@pytest.mark.parametrize("length", [-1, -2 ** 31, 6 * 16 + 1, 2 ** 31 - 1])
def test_free_leaves_a_sequence_with_a_bad_length(length):
    """Its length, its pages' counts and its table stay, so that the caller can put the length right; the others are freed."""
    need_gpu()
    say(f"free, a length of {length}")
    st = Setup([70, 48, 5], 16, 1, 64, seed=100, columns=6)
    table = st.table.clone()
    st.lens[1] = length
    ops.paged_cache_free(st.cache, i32([0, 1, 2, 1]))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert st.lens.tolist() == [0, length, 0]
    st.lens[1] = 48
    st.state.free([0, 2])
    st.check_state()
    assert torch.equal(st.table, table)
    ops.paged_cache_free(st.cache, i32([1, 1]))
    st.state.free([1])
    assert ops.device_errors() == 0
    st.check_state()


@pytest.mark.parametrize("what", ["first page", "last full page", "partly filled page", "negative page", "length", "negative length", "parent of the last fork"])
def test_fork_of_a_broken_parent_changes_nothing(what):
    need_gpu()
    say(f"fork refused: {what}")
    S = 1200  # more forks than a workgroup has threads
    st = Setup([70, 48, 5, 64] + [0] * S, 16, 2, 64, layers=2, seed=101, spare=2 * S, columns=6)
    parents, children = [0, 1, 3] + [0] * (S - 4) + [2], list(range(4, 4 + S))
    at, value = {"first page": ((0, 0), len(st.state.refs)), "last full page": ((3, 3), 1 << 30), "partly filled page": ((0, 4), 1 << 29),
                 "negative page": ((1, 2), -1), "parent of the last fork": ((2, 0), -5)}.get(what, (None, None))
    good_table, good_lens = st.table.clone(), st.lens.clone()
    if at:
        st.table[at] = value
    else:
        st.lens[1] = 6 * 16 + 1 if what == "length" else -1
    before = [t.clone() for t in (st.table, st.lens, st.refs, st.k, st.v)]
    ops.paged_cache_fork(st.cache, i32(parents), i32(children))
    assert ops.device_errors() == _lib.DEVERR_PAGED
    for t, x in zip((st.table, st.lens, st.refs, st.k, st.v), before):
        assert torch.equal(t, x)
    st.table.copy_(good_table)  # put right, the same call goes through
    st.lens.copy_(good_lens)
    ops.paged_cache_fork(st.cache, i32(parents), i32(children))
    assert ops.device_errors() == 0 and st.state.fork(parents, children)
    st.check_state()


@pytest.mark.parametrize("at,length", [(1, -1), (1, 6 * 16 + 1), (0, 2 ** 31 - 1), (1499, -2 ** 31)])
def test_compact_with_a_bad_length_changes_nothing(at, length):
    need_gpu()
    say(f"compact, sequence {at} of length {length}")
    st = Setup([70, 48, 5, 96] + [0, 3] * 748, 16, 1, 64, layers=2, seed=102, spare=40, columns=6)
    ops.paged_cache_free(st.cache, i32([2, 0]))
    st.state.free([2, 0])
    st.lens[at] = length
    before = [t.clone() for t in (st.table, st.lens, st.refs, st.k, st.v)]
    ops.paged_cache_compact(st.cache)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    for t, x in zip((st.table, st.lens, st.refs, st.k, st.v), before):
        assert torch.equal(t, x)
    st.lens[at] = st.state.lens[at]
    ops.paged_cache_compact(st.cache)
    st.state.compact()
    assert ops.device_errors() == 0
    st.check_state()


def test_compact_leaves_an_entry_outside_the_pool():
    need_gpu()
    say("compact, a table entry outside the pool")
    st = Setup([70, 48, 5, 96], 16, 1, 64, seed=103, spare=9, columns=6)
    ops.paged_cache_free(st.cache, i32([2, 0]))
    st.state.free([2, 0])
    for at, value in ((1, 1), len(st.state.refs)), ((3, 2), -9):
        st.table[at] = value
    ops.paged_cache_compact(st.cache)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    st.state.compact()
    st.state.table[1][1], st.state.table[3][2] = len(st.state.refs), -9
    st.check_state()


@pytest.mark.parametrize("n,group,dim", [(1, 4, 128), (1, 2, 256), (40, 4, 128), (40, 2, 256), (30, 4, 512)])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_scale_that_is_nan_shows_in_its_heads(which, n, group, dim):
    """E4M3 pages: the query heads of that KV head are NaN, in single tokens and in chunks; the others are unharmed."""
    need_gpu()
    say(f"paged attention, a NaN {which}, {n} rows of {dim}")
    st = Setup([300], 16, 2, dim, "e4m3", seed=104)
    sc = st.k_scale[0].clone(), st.v_scale[0].clone()
    getattr(st, which)[0, 1] = float("nan")
    q = queries(n, 2 * group, dim, 105)
    out = torch.zeros_like(q)
    ops.paged_attention(q, st.cache, i32([0, n]), out)
    assert ops.device_errors() == 0
    want, a, d = pm.attention(q, *st.values(), st.state.table, [300], [0, n], 16, 0, 1.0, *sc)
    assert torch.isnan(out[:, group:].float()).all()
    check_rows(out[:, :group], want[:, :group], a[:, :group], d[:, :group], dim)


def test_calls_wait_for_the_current_streams_work():
    """New keys, values and queries are made by work that is still running on the side stream when the calls are issued: nothing between it
    and the calls waits, so a call on another stream would read the zeros that were there before."""
    need_gpu()
    say("paged calls behind running work of a side stream")
    st = Setup([100, 40], 16, 2, 128, seed=106, spare=10, columns=20)
    lens, rows = [101, 70], [1, 30]
    side = torch.cuda.Stream()
    new, starts = i32(rows), i32(starts_of(rows))
    nk, nv, q = (torch.zeros((31, h, 128), dtype=torch.bfloat16, device=DEV) for h in (2, 2, 8))
    made = queries(31, 2, 128, 1, 11.0), queries(31, 2, 128, 2, 11.0), queries(31, 8, 128, 3)
    out = torch.full_like(q, 123.0)
    big = torch.randn((4096, 4096), device=DEV)
    before = [t.float().clone() for t in (st.k[0], st.v[0])]
    for warm in (True, False):  # the first turn loads what the second one needs, so that it runs without a pause
        with torch.cuda.stream(side):
            x = big
            for _ in range(1 if warm else 20):
                x = x @ big
                x = x / x.norm()
            zero = (x[0, 0] * 0).to(torch.bfloat16)
            for t, m in zip((nk, nv, q), made):
                t.copy_(m + zero if not warm else t)
            if not warm:
                busy = not side.query()
                ops.paged_cache_reserve(st.cache, new)
                ops.paged_cache_append(st.cache, nk, nv, starts)
                ops.paged_attention(q, st.cache, starts, out, max_rows=30)
        torch.cuda.synchronize()
    assert busy, "the side stream had finished before the calls were issued: the test shows nothing"
    assert ops.device_errors() == 0 and st.state.reserve(rows)
    st.check_state()
    for t, old, m in zip((st.k[0], st.v[0]), before, made):
        for i, s, pos in pm.positions(starts_of(rows), lens):
            old[st.state.table[s][pos // 16], pos % 16] = m[i].float()
        assert torch.equal(t.float(), old)
    want, a, d = pm.attention(made[2], *before, st.state.table, lens, starts_of(rows), 16, 0, 1.0)
    check_rows(out, want, a, d, 128)


def test_one_scratch_ring_serves_the_projections_of_a_whole_step():
    """Sequences at positions of their own: a QKV call each, into one ring, at the slots of their rows in the step; the rows then lie in the
    order that one append and one attention take."""
    need_gpu()
    say("QKV of three sequences into one scratch ring, one append, one attention")
    from gpu_util import dev, dev_zeros
    from moa_amd import synth
    before, M = [700, 31, 0], [1, 3, 20]
    lens, starts = [b + m for b, m in zip(before, M)], starts_of(M)
    st = Setup(before, 64, 8, 256, seed=107, spare=20, columns=12)
    ops.paged_cache_reserve(st.cache, i32(M))
    assert st.state.reserve(M)
    kr, vr, q = dev_zeros(1024 * 2048), dev_zeros(1024 * 2048), dev_zeros(sum(M) * 4096)
    apart = []
    names = ("x", "q_weight", "k_weight", "v_weight", "q_weight_scale", "k_weight_scale", "v_weight_scale", "input_rms_weight",
             "q_rms_weight", "k_rms_weight")
    for s, m in enumerate(M):
        d = synth.cfg_qkv(seed=3 + s, M=m, pos=before[s])
        w = [dev(d[n]) for n in names]
        cos, sin, rope = dev(d["cos"]), dev(d["sin"]), i32([512 * before[s]])
        ops.sliding_project_qkv(*w, i32([4096 * starts[s]]), rope, cos, sin, kr, vr, q[starts[s] * 4096:starts[s + 1] * 4096])
        own = dev_zeros(1024 * 2048), dev_zeros(1024 * 2048), dev_zeros(m * 4096)
        ops.sliding_project_qkv(*w, i32([4096 * before[s]]), rope, cos, sin, *own)
        apart.append([own[0].view(1024, 2048)[before[s]:lens[s]], own[1].view(1024, 2048)[before[s]:lens[s]], own[2]])
    k, v = (t.view(torch.bfloat16).view(1024, 8, 256)[:sum(M)] for t in (kr, vr))
    q = q.view(torch.bfloat16).view(sum(M), 16, 256)
    for got, i in ((k, 0), (v, 1), (q, 2)):
        assert torch.equal(raw(got).flatten(), torch.cat([a[i].flatten().view(torch.int16) for a in apart]))
    out = torch.empty_like(q)
    ops.paged_cache_append(st.cache, k, v, i32(starts))
    ops.paged_attention(q, st.cache, i32(starts), out, window=1024, max_rows=max(M))
    assert ops.device_errors() == 0
    want, a, d = pm.attention(q, *st.values(), st.state.table, lens, starts, 64, 1024, 1.0)
    check_rows(out, want, a, d, 256)
    for m, s, t in pm.positions(starts, lens):
        assert torch.equal(raw(st.k)[0, st.state.table[s][t // 64], t % 64], raw(k)[m])
