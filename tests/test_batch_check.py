"""Lengths and page tables that a batch plan refuses, and calls without a plan: host checks, no device."""
import ctypes as C

import pytest

import gguf_runner_b200 as g

OK, INVALID, RANGE = 0, 1, 4


@pytest.mark.parametrize("want,q_len,kv_len,table,more", [
    (OK, [], [], None, {}),
    (OK, [0, 1, 17], [0, 1, 33], [[0, 0, 0], [7, 0, 0], [1, 2, 3]], {}),
    (OK, [0, 1], [32, 33], [[4, 5, 0], [4, 5, 6]], {}),              # a common prefix
    (OK, [1], [16], [[0]], {}),
    (INVALID, [-1], [1], [[0]], {}),
    (INVALID, [2], [1], [[0]], {}),
    (RANGE, [1], [17], [[0]], {}),                                   # 17 positions, one page
    (RANGE, [1], [1], [[8]], {}),
    (RANGE, [1], [1], [[-1]], {}),
    (RANGE, [0], [33], [[0, 1, 8]], {}),                             # a bad page that is only read
    (INVALID, [1], [1], None, dict(table_missing=True)),
    (INVALID, [1, 1], [20, 20], [[0, 1], [2, 1]], {}),               # one page, two sequences
    (INVALID, [17], [33], [[0, 1, 1]], {}),                          # one page, two stretches of a sequence
    (INVALID, [33], [33], [[1, 2, 1]], {}),
    (OK, [1], [33], [[1, 1, 2]], {}),                                # pages that are only read may repeat
    (RANGE, [5, 6], [5, 6], [[0], [1]], dict(max_tokens=10)),
    (RANGE, [1, 1], [32, 32], [[0, 1], [2, 3]], dict(max_pages=3)),
    (RANGE, [0, 0], [2 ** 31 - 1, 2], [[0]], {}),
])
def test_page_tables(want, q_len, kv_len, table, more):
    more = dict(more)
    if more.pop("table_missing", False):
        import numpy as np
        q, kv = np.array(q_len, np.int32), np.array(kv_len, np.int32)
        assert g.lib().ggr_batch_check(16, 8, 1, q.ctypes.data, kv.ctypes.data, None, 4, 100, 100) == want
        return
    assert g.batch_check(q_len, kv_len, table, page_size=16, n_pages=8, **more) == want


@pytest.mark.parametrize("want,q_len,kv_len", [(OK, [3, 0, 9], None), (INVALID, [3], [4]), (INVALID, [-2], None)])
def test_packed_prompts(want, q_len, kv_len):
    assert g.batch_check(q_len, kv_len) == want


def test_null_handles():
    L = g.lib()
    out = C.c_void_p()
    assert L.ggr_pages_create(None, 1, 16, 1, None, None, None, None, C.byref(out)) == INVALID
    assert L.ggr_batch_create(None, None, 1, 1, 1, 0, C.byref(out)) == INVALID
    assert L.ggr_batch_set(None, 0, None, None, None, 0) == INVALID
    assert L.ggr_paged_append(None, None, 0, 0, None, 0, None, 0, None, 0, None) == INVALID
    assert L.ggr_paged_read(None, None, 0, 0, None, 0, None, 0) == INVALID
    assert L.ggr_paged_attention(None, None, 0, None, 0, None, 0) == INVALID
    assert L.ggr_packed_attention(None, None, 0, None, 0, None, 0, None, 0, None, 0) == INVALID
    assert L.ggr_pages_device_ptrs(None, None, None, None, None, None) == INVALID
    L.ggr_pages_destroy(None)
    L.ggr_batch_destroy(None)


def test_unknown_names_are_refused_before_the_library_is_called():
    with pytest.raises(ValueError):
        g.Batch(None, None, "f16", 1, 1)
    with pytest.raises(ValueError):
        g.Pages(None, 1, 16, "q4")
