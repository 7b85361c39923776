"""What a call over drafted trees leaves out where one sequence is bad, and that it keeps the others right, on the GPU."""
import math

import pytest

import candidates_model as cm
from gpu_util import need_gpu, say, torch
from moa_amd import _lib, ops
from test_gpu_candidates_ends import KINDS, call, reference
from test_gpu_paged import Setup, queries
from test_gpu_trees import check, trees

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", KINDS)
@pytest.mark.parametrize("bad", ["page", "length", "long", "rows", "descend"])
def test_a_bad_sequence_alone_is_left_out(bad, n, group, heads, dim, fmt):
    """The middle one of three: with a bad length, or more rows than max_rows, all of it is left as it was; with a bad page every row
    that sees it, the others right or as they were. The first and the last are right, but where starts descend, where no row that is
    not the first's is touched and the first's are right or as they were."""
    need_gpu()
    say(f"a bad {bad} among {n} nodes of {heads} x {group} x {dim} {fmt}")
    st = Setup([40 + n] * 3, 16, heads, dim, fmt, seed=3)
    masks, starts = trees([n] * 3, 5), [0, n, 2 * n, 3 * n]
    scale = 1 / math.sqrt(dim)
    q = queries(3 * n, heads * group, dim, 4, 2.0 / scale)
    hit = (40 + n - 1) // 16                   # the page of the last node
    if bad == "rows":                          # one row more than max_rows, one of the first's
        starts[1] = n - 1
    elif bad == "descend":
        starts[2:] = [n - 1, n - 1]
    sound = [s for s in (0, 2) if starts[s + 1] > starts[s]]
    want, a, d = reference(st, q, [0, n, n, n] if bad == "descend" else starts, masks, scale)
    if bad == "page":
        st.table[1, hit] = len(st.state.refs)
    elif bad in ("length", "long"):
        st.lens[1] = -1 if bad == "length" else st.table.shape[1] * 16 + 1
    out = torch.full_like(q, 7.0)
    call(st, q, starts, masks, out, n, scale=scale)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    right = lambda rows: check(out[rows], want[rows], a[rows], d[rows], dim)  # noqa: E731
    kept = lambda row: bool((out[row] == 7.0).all())  # noqa: E731
    if bad == "descend":
        assert all(kept(r) for r in range(n, 3 * n))
        right([r for r in range(n) if not kept(r)])
        return
    for s in sound:
        right(list(range(starts[s], starts[s + 1])))
    middle = range(starts[1], starts[2])
    if bad != "page":
        assert all(kept(r) for r in middle)
        return
    first = max(0, 16 * hit - 40)              # the first node in the bad page
    for r in middle:
        if masks[r] >> first or 16 * hit < 40:
            assert kept(r), r
    right([r for r in middle if not kept(r)])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,group,heads,dim", KINDS)
def test_padded_rows_may_hold_anything(n, group, heads, dim, fmt):
    """Rows without bits give zeros whatever their queries are, and change no other row, before few positions and many."""
    need_gpu()
    say(f"padded rows among {n} nodes of {heads} x {group} x {dim} {fmt}")
    for before in (3, 3000):
        st = Setup([before + n, 20 + n], 32, heads, dim, fmt, seed=6)
        masks = trees([n, n], 5)
        pads = [i for i in range(2 * n) if i % n and (i % 3 == 2 or i % n >= n - 2)]
        for i in pads:
            first = i // n * n
            masks[i] = 0
            for j in range(first, first + n):
                masks[j] &= ~(1 << i - first)
        scale = 1 / math.sqrt(dim)
        q = queries(2 * n, heads * group, dim, 4, 2.0 / scale)
        want, a, d = reference(st, q, [0, n, 2 * n], masks, scale)
        for i in pads:
            q[i] = (float("nan"), float("inf"), -3e38)[i % 3]
        out = torch.full_like(q, 7.0)
        call(st, q, [0, n, 2 * n], masks, out, n, scale=scale)
        assert ops.device_errors() == 0
        assert (out[pads] == 0).all()
        rows = [i for i in range(2 * n) if i not in pads]
        check(out[rows], want[rows], a[rows], d[rows], dim)
