"""The size limits of the paged KV4 entry points, refused before any CUDA call (no GPU needed)."""
import ctypes as C

import pytest

from fnfl_v100_b200 import _lib, build

A16 = 0x7F0000001000   # aligned, never dereferenced: rejection happens before any launch


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


SHAPE = dict(q=A16, k_cache=A16, v_cache=A16, k_scale=A16, v_scale=A16, table=A16, n_cells=A16, row_start=A16, out=A16, workspace=A16,
             workspace_bytes=1 << 30, cache_slots=4096, rows=8, n_req=8, max_pages=100, page_size=16, max_rows=1, n_q_heads=16,
             n_kv_heads=2, head_dim=256, scale=0.0625)


@pytest.mark.parametrize("change", [
    dict(rows=1 << 27, n_q_heads=16),                                     # rows x heads 2^31
    dict(cache_slots=(1 << 31) - 16, n_kv_heads=4, n_q_heads=16),         # slots x heads past 2^32
    dict(cache_slots=1 << 31), dict(cache_slots=1 << 22, page_size=1 << 21), dict(n_q_heads=1026, n_kv_heads=2), dict(cache_slots=8)])
def test_attend_limits(lib, change):
    a = _lib.AttendPagedArgs(**{**SHAPE, **change})
    assert lib.fnb_attend_paged_kv4(C.byref(a), None) == _lib.REJECTED
    assert lib.fnb_attend_paged_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("rows,n_kv", [(1 << 31, 1), (1 << 30, 4), (8, 257)])
def test_read_limits(lib, rows, n_kv):
    a = _lib.KvReadArgs(A16, A16, A16, A16, None, rows, 64, 0, n_kv, 256)
    assert lib.fnb_kv4_read_f32(C.byref(a), None) == _lib.REJECTED


def test_workspace_is_needed_only_where_items_are_cut(lib):
    """Up to 256 cells a request nothing is folded: a token size, whatever the shape; beyond it the size goes by the columns."""
    size = lambda **d: lib.fnb_attend_paged_workspace_bytes(C.byref(_lib.AttendPagedArgs(**{**SHAPE, **d})))  # noqa: E731
    small = {size(max_pages=16), size(max_pages=1), size(max_pages=2, page_size=128), size(max_pages=16, max_rows=9)}
    assert len(small) == 1 and 0 < small.pop() <= 256
    assert size(max_pages=17) == size(max_pages=1 << 20) < size(max_pages=17, max_rows=2)


def test_table_stride(lib):
    """0 stands for max_pages; less than max_pages is refused."""
    for stride, ok in ((0, True), (100, True), (5000, True), (99, False), (-1, False), (-100, False)):
        a = _lib.AttendPagedArgs(**{**SHAPE, "table_stride": stride})
        assert (lib.fnb_attend_paged_workspace_bytes(C.byref(a)) > 0) == ok
        if not ok:
            assert lib.fnb_attend_paged_kv4(C.byref(a), None) == _lib.REJECTED
