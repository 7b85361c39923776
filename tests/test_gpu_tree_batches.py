"""Batches of drafted trees on the GPU whose calls leave max_rows to its default."""
import math

import pytest

import candidates_model as cm
from gpu_util import need_gpu, say, torch
from moa_amd import _lib, ops
from test_gpu_paged import Setup, i32, queries, starts_of
from test_gpu_trees import check, trees

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("sizes,words,window", [([30] * 5, 1, 0), ([64, 1, 64], 1, 64), ([7] * 40, 2, 128), ([130, 200, 3], 4, 0), ([1] * 300, 4, 1024)])
@pytest.mark.parametrize("group,heads,dim", [(2, 2, 64), (4, 1, 128), (1, 1, 512)])
def test_the_default_takes_a_batch_of_more_rows_than_a_tree_has(group, heads, dim, sizes, words, window):
    need_gpu()
    say(f"trees of {len(sizes)} sequences, {sum(sizes)} rows, {words} words, window {window}, {heads} x {group} x {dim}")
    st = Setup([50 + n for n in sizes], 16, heads, dim)
    masks, starts = trees(sizes, 7), starts_of(sizes)
    q = queries(sum(sizes), heads * group, dim, 5, 2.0 * math.sqrt(dim))
    out = torch.full_like(q, 123.0)
    ops.paged_tree_attention(q, st.cache, i32(starts), cm.mask_tensor(masks, words, DEV), out, window=window, scale=1 / math.sqrt(dim))
    assert ops.device_errors() == 0
    want, a, d = cm.attention(q, *st.values(), st.state.table, st.state.lens, starts, masks, 16, window, 1 / math.sqrt(dim))
    check(out, want, a, d, dim)


def test_the_default_leaves_out_a_sequence_of_more_rows_than_mask_bits():
    need_gpu()
    say("70 rows of a sequence, one word")
    st = Setup([90, 60], 16, 2, 64)
    masks = trees([70, 20], 7)
    q = queries(90, 4, 64, 5, 16.0)
    out = torch.full_like(q, 7.0)
    m = cm.mask_tensor([x & (1 << 64) - 1 for x in masks], 1, DEV)
    ops.paged_tree_attention(q, st.cache, i32([0, 70, 90]), m, out, scale=0.125)
    assert ops.device_errors() == _lib.DEVERR_PAGED
    assert (out[:70] == 7.0).all()
    want, a, d = cm.attention(q, *st.values(), st.state.table, st.state.lens, [70, 70, 90], masks, 16, 0, 0.125)
    check(out[70:], want[70:], a[70:], d[70:], 64)


def test_a_window_below_the_default_is_refused():
    """A smaller max_rows says that no tree is larger than the window."""
    need_gpu()
    st = Setup([40, 40, 40], 16, 2, 64)
    masks = cm.mask_tensor(trees([30] * 3, 7), 1, DEV)
    q = queries(90, 4, 64, 5, 16.0)
    out = torch.empty_like(q)
    with pytest.raises(_lib.MoaError, match="window"):
        ops.paged_tree_attention(q, st.cache, i32([0, 30, 60, 90]), masks, out, window=63)
    ops.paged_tree_attention(q, st.cache, i32([0, 30, 60, 90]), masks, out, window=64)
    ops.paged_tree_attention(q, st.cache, i32([0, 30, 60, 90]), masks, out, window=30, max_rows=30)
    assert ops.device_errors() == 0
