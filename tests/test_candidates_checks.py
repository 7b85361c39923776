"""Host checks of the tree, beam and search calls (no GPU): a bad argument is refused before anything is launched; the counters
that their kernels join at; and the plain models that the GPU tests follow."""
import ctypes as C
import math
import random
import shutil
import subprocess
from pathlib import Path

import pytest

import candidates_model as cm
import paged_model as pm
from moa_amd import _lib
from test_paged_checks import OK, cache, refused

ROOT = Path(__file__).resolve().parent.parent


def tree_attention(**change):
    a = dict(q=OK, qs=1024, c=cache(), starts=OK, masks=OK, words=1, out=OK, os=1024, rows=3, heads=8, layer=0, window=0, scale=1.0,
             most=3, stream=None)
    a.update(change)
    return _lib.load().moa_paged_tree_attention(*a.values())


def commit(**change):
    a = dict(c=cache(), starts=OK, masks=OK, words=1, leaves=OK, rows=3, stream=None)
    a.update(change)
    return _lib.load().moa_paged_tree_commit(*a.values())


def reorder(**change):
    a = dict(c=cache(), parents=OK, count=4, beams=2, stream=None)
    a.update(change)
    return _lib.load().moa_paged_cache_reorder(*a.values())


def verify(**change):
    a = dict(logits=OK, stride=100, tokens=OK, starts=OK, masks=OK, words=1, best=OK, leaves=OK, next=OK, rows=3, vocab=100,
             sequences=2, stream=None)
    a.update(change)
    return _lib.load().moa_tree_verify(*a.values())


def select(**change):
    a = dict(logits=OK, stride=100, scores=OK, finished=OK, out_scores=OK, out_finished=OK, parents=OK, tokens=OK, groups=2, beams=4,
             vocab=100, eos=5, stream=None)
    a.update(change)
    return _lib.load().moa_beam_select(*a.values())


@pytest.mark.parametrize("call", [tree_attention, commit, reorder])
@pytest.mark.parametrize("change,code,word", [
    (dict(k_pages=0), -1, "k_pages"), (dict(page_table=OK + 2), -2, "page_table"), (dict(head_dim=96), -1, "head_dim"),
    (dict(pages=(1 << 20) + 1), -1, "pages"), (dict(sequences=65537), -1, "sequences"), (dict(element=1), -1, "k_scale"),
    (dict(k1=4100), -1, "page stride"), (dict(table_stride=7), -1, "table_stride"),
])
def test_bad_caches_are_refused(call, change, code, word):
    refused(call(c=cache(**change)), code, word)
    refused(call(c=None), -1, "cache is NULL")


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), -1, "q is NULL"), (dict(q=OK + 8), -2, "q "), (dict(out=OK + 8), -2, "out"), (dict(starts=None), -1, "row_starts"),
    (dict(masks=None), -1, "masks"), (dict(masks=OK + 4), -2, "masks"), (dict(words=0), -1, "mask_words"),
    (dict(words=5), -1, "mask_words"), (dict(rows=-1), -1, "rows"), (dict(rows=(1 << 20) + 1), -1, "rows"),
    (dict(heads=7), -1, "q_heads"), (dict(heads=258), -1, "q_heads"), (dict(layer=2), -1, "layer"), (dict(window=-1), -1, "window"),
    (dict(window=2), -1, "window"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=-1e30), -1, "scale"),
    (dict(most=0), -1, "max_rows"), (dict(most=4), -1, "max_rows"), (dict(rows=65, most=65), -1, "max_rows"),
    (dict(rows=300, most=257, words=4), -1, "max_rows"), (dict(qs=1020), -1, "row strides"), (dict(os=1016), -1, "row strides"),
])
def test_bad_tree_attention_is_refused(change, code, word):
    refused(tree_attention(**change), code, word)


@pytest.mark.parametrize("change,code,word", [
    (dict(starts=None), -1, "row_starts"), (dict(masks=None), -1, "masks"), (dict(masks=OK + 4), -2, "masks"),
    (dict(leaves=None), -1, "leaves"), (dict(leaves=OK + 2), -2, "leaves"), (dict(words=0), -1, "mask_words"),
    (dict(words=5), -1, "mask_words"), (dict(rows=-1), -1, "rows"), (dict(rows=(1 << 20) + 1), -1, "rows"),
])
def test_bad_commits_are_refused(change, code, word):
    refused(commit(**change), code, word)


@pytest.mark.parametrize("change,code,word", [
    (dict(parents=None), -1, "parents"), (dict(parents=OK + 2), -2, "parents"), (dict(count=-2), -1, "count"),
    (dict(count=6), -1, "count"), (dict(count=3), -1, "multiple of beams"), (dict(beams=0), -1, "beams"), (dict(beams=65), -1, "beams"),
])
def test_bad_reorders_are_refused(change, code, word):
    refused(reorder(**change), code, word)


@pytest.mark.parametrize("change,code,word", [
    (dict(logits=None), -1, "logits"), (dict(logits=OK + 1), -2, "logits"), (dict(stride=99), -1, "logit_row_stride"),
    (dict(tokens=None), -1, "tokens"), (dict(starts=None), -1, "row_starts"), (dict(masks=OK + 4), -2, "masks"),
    (dict(words=0), -1, "mask_words"), (dict(words=5), -1, "mask_words"), (dict(best=None), -1, "best"), (dict(leaves=None), -1, "leaves"),
    (dict(next=OK + 2), -2, "next_tokens"), (dict(rows=-1), -1, "rows"), (dict(rows=65536), -1, "rows"), (dict(vocab=0), -1, "vocab"),
    (dict(vocab=(1 << 20) + 1, stride=1 << 21), -1, "vocab"), (dict(sequences=0), -1, "sequences"), (dict(sequences=65537), -1, "sequences"),
])
def test_bad_verifications_are_refused(change, code, word):
    refused(verify(**change), code, word)


@pytest.mark.parametrize("change,code,word", [
    (dict(logits=None), -1, "logits"), (dict(logits=OK + 1), -2, "logits"), (dict(stride=99), -1, "logit_row_stride"),
    (dict(scores=None), -1, "scores"), (dict(finished=OK + 2), -2, "finished"), (dict(out_scores=None), -1, "out_scores"),
    (dict(out_finished=None), -1, "out_finished"), (dict(parents=None), -1, "parents"), (dict(tokens=None), -1, "tokens"),
    (dict(groups=-1), -1, "groups"), (dict(groups=16384), -1, "groups"), (dict(beams=0), -1, "beams"), (dict(beams=65), -1, "beams"),
    (dict(vocab=0, eos=-1), -1, "vocab"), (dict(vocab=(1 << 20) + 1, stride=1 << 21), -1, "vocab"), (dict(eos=-2), -1, "eos"),
    (dict(eos=100), -1, "eos"),
])
def test_bad_selections_are_refused(change, code, word):
    refused(select(**change), code, word)


def test_a_single_row_needs_no_strides():
    """One row's distance to the next is not looked at: the next refused argument is named instead."""
    refused(tree_attention(rows=1, most=1, qs=0, os=0, masks=None), -1, "masks")
    refused(verify(rows=1, stride=0, tokens=None), -1, "tokens")
    refused(select(groups=1, beams=1, stride=0, scores=None), -1, "scores")


def test_empty_calls_launch_nothing():
    assert tree_attention(q=None, starts=None, masks=None, out=None, rows=0, most=1) == 0
    assert commit(starts=None, masks=None, leaves=None, rows=0) == 0
    assert reorder(parents=None, count=0) == 0
    assert select(logits=None, scores=None, finished=None, out_scores=None, out_finished=None, parents=None, tokens=None, groups=0) == 0


def test_front_end_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from moa_amd import ops
    x, i = torch.zeros((4, 100), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.tree_verify(x, i, i, torch.zeros((4, 1), dtype=torch.int64), i, i, i)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.beam_select(x, torch.zeros(4), i, torch.zeros(4), i, i, i, 2)
    for call in (lambda: ops.paged_tree_attention(x, i, i, x[:, None], x), lambda: ops.paged_tree_commit(x, i, i, i),
                 lambda: ops.paged_cache_reorder(x, i, 2)):
        with pytest.raises(TypeError, match="PagedCache"):
            call()


@pytest.fixture(scope="module")
def turns(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    lib = tmp_path_factory.mktemp("turns") / "join_turns.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    f"-I{ROOT / 'moa-workspace_amd' / 'csrc'}", "-o", str(lib), str(ROOT / "tests" / "cpp" / "join_turns.cpp")], check=True)
    lib = C.CDLL(str(lib))
    lib.join_share.restype, lib.join_share.argtypes = C.c_uint, [C.c_int, C.c_int, C.c_uint]
    lib.join_last.restype, lib.join_last.argtypes = C.c_int, [C.c_uint, C.c_uint, C.c_uint]
    return lib


@pytest.mark.parametrize("turn,most", [(128, 64), (512, 512)])
def test_counters_of_longer_turns_join_once(turns, turn, most):
    """Arrivals in any order, from any multiple of the turn: the last of a launch joins, and alone."""
    rng = random.Random(turn)
    for parts in [1, 2, 3, most - 1, most]:
        for held in (0, turn, 2 ** 32 - turn):
            order = [i == 0 for i in range(parts)]
            rng.shuffle(order)
            counter, joins = held, []
            for i, first in enumerate(order):
                share = turns.join_share(first, parts, turn)
                if turns.join_last(counter, share, turn):
                    joins.append(i)
                counter = (counter + share) % 2 ** 32
            assert joins == [parts - 1] and counter % turn == 0


def test_model_of_trees():
    # node 0 with children 1 and 2, 2 with child 3
    masks = [0b1, 0b11, 0b101, 0b1101]
    st = pm.State([[0, 1], [2, -1]], [20, 3], [1, 1, 1, 0], 16)
    moves, left = cm.commit(st, [0, 4, 4], masks, [3, 0])
    assert not left and st.lens == [19, 3] and st.refs == [1, 1, 1, 0]
    assert moves == [((1, 2), (1, 1)), ((1, 3), (1, 2))]
    assert cm.commit(st, [0, 1, 4], [1] * 4, [-1, 1])[1] == [] and st.lens == [18, 1]
    assert cm.commit(st, [0, 0, 1], [1], [0, 1])[1] == [1] and st.lens == [18, 1]
    torch = pytest.importorskip("torch")
    x = torch.zeros((4, 8))
    x[0, 5] = x[2, 7] = x[3, 1] = 1.0
    x[1] = math.nan
    assert cm.verify(x, [9, 4, 5, 7], [0, 4, 4], masks) == ([5, 0, 7, 1], [3, -1], [1, -1])
    assert [m.bit_count() if hasattr(m, "bit_count") else bin(m).count("1") for m in cm.tree(cm.rng(1), 5, chain=True)] == [1, 2, 3, 4, 5]


def test_model_of_beams():
    st = pm.State([[0, 1], [2, 3]], [20, 20], [1, 1, 1, 1], 16)
    assert cm.reorder(st, [0, 0], 2) == [(1, 3, 4)]
    assert st.table == [[0, 1], [0, 3]] and st.refs == [2, 1, 0, 1]
    assert cm.reorder(st, [0, 2], 2) is None and st.refs == [2, 1, 0, 1]
    torch = pytest.importorskip("torch")
    x = torch.tensor([[0.0, 1.0, 0.0], [2.0, 0.0, 0.0]])
    scores, finished, parents, tokens = cm.select(x, [-1.0, -2.0], [0, 1], 2, 2)
    assert parents == [0, 1] and tokens == [1, 2] and finished == [0, 1] and scores[1] == -2.0
    assert abs(scores[0] - (-1.0 + 1.0 - math.log(math.e + 2))) < 1e-6
