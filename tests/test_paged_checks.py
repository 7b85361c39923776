"""The paged cache's host checks (no GPU): a bad argument is refused before anything is launched; and the plain state
model that the GPU tests follow."""
import ctypes as C
import struct

import pytest

import paged_model as pm
from moa_amd import _lib

FIELDS = ["k_pages", "v_pages", "k_scale", "v_scale", "page_table", "seq_lens", "ref_counts", "k0", "k1", "k2", "k3", "v0", "v1",
          "v2", "v3", "table_stride", "layers", "pages", "slots", "kv_heads", "head_dim", "element", "sequences", "columns"]
BUF = (C.c_uint8 * 4096)()
OK = (C.addressof(BUF) + 15) // 16 * 16


def cache(**change):
    c = dict(k_pages=OK, v_pages=OK, k_scale=0, v_scale=0, page_table=OK, seq_lens=OK, ref_counts=OK, k0=1 << 20, k1=4096, k2=256,
             k3=128, v0=1 << 20, v1=4096, v2=256, v3=128, table_stride=8, layers=2, pages=10, slots=16, kv_heads=2, head_dim=128,
             element=0, sequences=4, columns=8)
    c.update(change)
    return struct.pack("=7Q9q8i", *[c[f] for f in FIELDS])


def calls(c):
    lib = _lib.load()
    return {
        "reserve": lambda: lib.moa_paged_cache_reserve(c, OK, None),
        "append": lambda: lib.moa_paged_cache_append(c, OK, 256, OK, 256, OK, 3, 0, None),
        "fork": lambda: lib.moa_paged_cache_fork(c, OK, OK, 1, None),
        "free": lambda: lib.moa_paged_cache_free(c, OK, 1, None),
        "compact": lambda: lib.moa_paged_cache_compact(c, None),
        "attention": lambda: lib.moa_paged_attention(OK, 1024, c, OK, OK, 1024, 3, 8, 0, 0, 1.0, 3, None),
    }


def refused(rc, code, word):
    msg = _lib.load().moa_last_error_string().decode()
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("call", ["reserve", "append", "fork", "free", "compact", "attention"])
@pytest.mark.parametrize("change,code,word", [
    (dict(k_pages=0), -1, "k_pages"), (dict(v_pages=OK + 8), -2, "v_pages"), (dict(page_table=0), -1, "page_table"),
    (dict(seq_lens=OK + 2), -2, "seq_lens"), (dict(ref_counts=0), -1, "ref_counts"), (dict(layers=0), -1, "layers"),
    (dict(pages=0), -1, "pages"), (dict(pages=(1 << 20) + 1), -1, "pages"), (dict(slots=0), -1, "slots"),
    (dict(slots=65537), -1, "slots"), (dict(kv_heads=0), -1, "kv_heads"), (dict(head_dim=96), -1, "head_dim"),
    (dict(element=2), -1, "element"), (dict(sequences=0), -1, "sequences"), (dict(sequences=65537), -1, "sequences"),
    (dict(columns=0), -1, "columns"), (dict(columns=1 << 20, table_stride=1 << 20, slots=4096), -1, "2^30"),
    (dict(table_stride=7), -1, "table_stride"), (dict(k_scale=OK), -1, "scales"), (dict(element=1), -1, "k_scale"),
    (dict(element=1, k_scale=OK, v_scale=OK + 1), -2, "v_scale"), (dict(k1=4100), -1, "page stride"),
    (dict(v2=64), -1, "slot stride"), (dict(k3=-128), -1, "head stride"), (dict(k0=0), -1, "layer stride"),
    (dict(element=1, k_scale=OK, v_scale=OK, v3=136), -1, "head stride"),
])
def test_bad_caches_are_refused(call, change, code, word):
    refused(calls(cache(**change))[call](), code, word)


def test_a_null_cache_is_refused():
    for call in calls(None).values():
        refused(call(), -1, "cache is NULL")


def test_bad_arguments_are_refused():
    lib, c = _lib.load(), cache()
    refused(lib.moa_paged_cache_reserve(c, None, None), -1, "new_tokens")
    refused(lib.moa_paged_cache_append(c, OK, 256, OK, 256, OK, -1, 0, None), -1, "rows")
    refused(lib.moa_paged_cache_append(c, OK, 256, OK, 256, OK, 3, 2, None), -1, "layer")
    refused(lib.moa_paged_cache_append(c, OK, 256, OK, 260, OK, 3, 0, None), -1, "row strides")
    refused(lib.moa_paged_cache_append(c, OK, 248, OK, 256, OK, 3, 0, None), -1, "row strides")
    refused(lib.moa_paged_cache_append(c, OK, 256, OK + 8, 256, OK, 3, 0, None), -2, "v ")
    refused(lib.moa_paged_cache_append(c, OK, 256, OK, 256, None, 3, 0, None), -1, "row_starts")
    refused(lib.moa_paged_cache_fork(c, None, OK, 1, None), -1, "parents")
    refused(lib.moa_paged_cache_fork(c, OK, OK + 2, 1, None), -2, "children")
    refused(lib.moa_paged_cache_fork(c, OK, OK, -1, None), -1, "count")
    refused(lib.moa_paged_cache_free(c, None, 1, None), -1, "sequences")
    att = lambda **k: lib.moa_paged_attention(*[{**dict(q=OK, qs=1024, c=c, rs=OK, o=OK, os=1024, rows=3, heads=8, layer=0,  # noqa: E731
                                                        window=0, scale=1.0, most=3, s=None), **k}[x] for x in
                                                ("q", "qs", "c", "rs", "o", "os", "rows", "heads", "layer", "window", "scale", "most", "s")])
    for change, code, word in ((dict(q=None), -1, "q is NULL"), (dict(o=OK + 8), -2, "out"), (dict(rs=None), -1, "row_starts"),
                               (dict(rows=-1), -1, "rows"), (dict(heads=7), -1, "q_heads"), (dict(heads=0), -1, "q_heads"),
                               (dict(heads=258), -1, "q_heads"), (dict(layer=-1), -1, "layer"), (dict(window=-1), -1, "window"),
                               (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
                               (dict(most=0), -1, "max_rows"), (dict(most=4), -1, "max_rows"), (dict(qs=1020), -1, "row strides"),
                               (dict(os=1016), -1, "row strides")):
        refused(att(**change), code, word)


def test_empty_calls_launch_nothing():
    lib, c = _lib.load(), cache()
    assert lib.moa_paged_cache_append(c, None, 0, None, 0, None, 0, 0, None) == 0
    assert lib.moa_paged_cache_fork(c, None, None, 0, None) == 0
    assert lib.moa_paged_cache_free(c, None, 0, None) == 0
    assert lib.moa_paged_attention(None, 0, c, None, None, 0, 0, 8, 0, 0, 1.0, 1, None) == 0


def test_front_end_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from moa_amd import ops
    k = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.PagedCache(k, k, i[None], i[:1], i)
    with pytest.raises(TypeError, match="PagedCache"):
        ops.paged_cache_compact(k)


def test_model_of_the_state():
    s = pm.State([[0, 1, -1], [3, -1, -1], [-1] * 3], [20, 16, 0], [1, 1, 0, 1, 0, 0], 16)
    assert s.reserve([0, 1, 0]) and s.table[1][:2] == [3, 2] and s.lens == [20, 17, 0]
    assert s.fork([0], [2]) and s.table[2][:2] == [0, 4] and s.refs == [2, 1, 1, 1, 1, 0] and s.moves == [(1, 4)]
    s.free([0])
    assert s.refs == [1, 0, 1, 1, 1, 0]
    s.compact()
    assert s.refs == [1, 1, 1, 1, 0, 0] and s.table[2][:2] == [0, 1] and s.moves == [(4, 1)]
    assert not s.reserve([0, 0, 1000]) and not s.fork([1], [2])
