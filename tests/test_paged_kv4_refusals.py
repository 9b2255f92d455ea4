"""The paged KV4 entry points refuse what is outside their contract before touching CUDA (no GPU needed)."""
import ctypes as C

import pytest
import torch

from fnfl_v100_b200 import _lib, build, ops

A16 = 0x7F0000001000   # a 16-byte aligned, never dereferenced address: rejection happens before any launch
ODD = A16 + 4


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


TABLES = dict(n_old=A16, n_new=A16, free_pages=A16, free_head=A16, table=A16, n_cells=A16, row_start=A16, slots=A16, pos=A16,
              free_head_out=A16, err=None, rows=64, n_free=100, n_req=8, max_pages=16, n_pages=200, page_size=16)


@pytest.mark.parametrize("field,bad", [
    ("n_old", None), ("n_new", A16 + 2), ("table", None), ("n_cells", None), ("row_start", None), ("slots", A16 + 1), ("pos", None),
    ("free_pages", None), ("free_head", A16 + 2), ("err", A16 + 2), ("rows", 0), ("rows", 2**31), ("n_free", -1), ("n_req", 0),
    ("n_req", 2049), ("max_pages", 0), ("n_pages", 0), ("page_size", 0), ("page_size", 24), ("page_size", -16), ("n_pages", 2**27)])
def test_page_tables_refusals(lib, field, bad):
    a = _lib.PageTablesArgs(**{**TABLES, field: bad})
    assert lib.fnb_page_tables(C.byref(a), None) == _lib.REJECTED
    assert lib.fnb_page_tables(None, None) == _lib.REJECTED


@pytest.mark.parametrize("field,bad", [("head_dim", 96), ("cell0", 60), ("rows", 0), ("out", None), ("cache", ODD), ("n_kv_heads", 0),
                                       ("scale", None), ("scale", A16 + 8), ("cache_slots", 0), ("cell0", -1)])
def test_read_refusals(lib, field, bad):
    a = _lib.KvReadArgs(A16, A16, None, A16, None, 8, 64, 0, 2, 256)
    setattr(a, field, bad)
    assert lib.fnb_kv4_read_f32(C.byref(a), None) == _lib.REJECTED
    assert lib.fnb_kv4_read_f32(None, None) == _lib.REJECTED


@pytest.mark.parametrize("field,bad", [("head_dim", 96), ("n_rot", 66), ("n_rot", 512), ("rows", 0), ("cache_slots", 0), ("q", ODD),
                                       ("k_cache", None), ("theta_scale", 0.0), ("pos", None), ("eps", -1.0)])
def test_append_refusals(lib, field, bad):
    a = _lib.RopeKvArgs(A16, A16, A16, A16, None, None, None, A16, A16, A16, None, None, 4, 64, 16, 2, 256, 64, 0.5, 1e-6)
    setattr(a, field, bad)
    assert lib.fnb_rope_neox_kv4_append(C.byref(_lib.RopeKv8Args(a, A16, A16)), None) == _lib.REJECTED


def test_append_refuses_missing_or_misaligned_scales(lib):
    a = _lib.RopeKvArgs(A16, A16, A16, A16, None, None, None, A16, A16, A16, None, None, 4, 64, 16, 2, 256, 64, 0.5, 1e-6)
    for ks, vs in ((None, A16), (A16, None), (A16 + 8, A16)):
        assert lib.fnb_rope_neox_kv4_append(C.byref(_lib.RopeKv8Args(a, ks, vs)), None) == _lib.REJECTED
    assert lib.fnb_rope_neox_kv4_append(None, None) == _lib.REJECTED


PAGED = dict(q=A16, gate=A16, k_cache=A16, v_cache=A16, k_scale=A16, v_scale=A16, table=A16, n_cells=A16, row_start=A16, out=A16,
             workspace=A16, workspace_bytes=1 << 30, err=None, cache_slots=4096, rows=8, n_req=8, max_pages=100, page_size=16,
             max_rows=1, n_q_heads=16, n_kv_heads=2, head_dim=256, scale=0.0625)


@pytest.mark.parametrize("field,bad", [
    ("q", ODD), ("q", None), ("gate", ODD), ("out", None), ("k_cache", None), ("v_cache", ODD), ("k_scale", None), ("v_scale", A16 + 8),
    ("table", None), ("n_cells", A16 + 2), ("row_start", A16 + 1), ("err", A16 + 2), ("workspace", None), ("workspace", ODD),
    ("workspace_bytes", 1000), ("head_dim", 96), ("head_dim", 512), ("n_q_heads", 15), ("n_kv_heads", 0), ("rows", 0), ("n_req", 0),
    ("n_req", 2049), ("max_pages", 0), ("page_size", 8), ("page_size", 48), ("cache_slots", 4100), ("cache_slots", 0), ("max_rows", -1),
    ("scale", 0.0), ("scale", float("inf")), ("scale", float("nan"))])
def test_attend_refusals(lib, field, bad):
    a = _lib.AttendPagedArgs(**{**PAGED, field: bad})
    assert lib.fnb_attend_paged_kv4(C.byref(a), None) == _lib.REJECTED


def test_attend_needs_a_row_for_each_request_without_row_start(lib):
    a = _lib.AttendPagedArgs(**{**PAGED, "row_start": None, "rows": 7})
    assert lib.fnb_attend_paged_kv4(C.byref(a), None) == _lib.REJECTED
    assert lib.fnb_attend_paged_workspace_bytes(C.byref(a)) == 0
    assert lib.fnb_attend_paged_kv4(None, None) == _lib.REJECTED


def test_workspace_is_a_function_of_the_shape_alone(lib):
    need = [lib.fnb_attend_paged_workspace_bytes(C.byref(_lib.AttendPagedArgs(**{**PAGED, **d})))
            for d in (dict(), dict(n_req=1, rows=1, max_pages=20000, cache_slots=1 << 20), dict(max_rows=5), dict(max_pages=8))]
    assert need[0] == need[1] and need[2] > need[0] > need[3] > 0


def test_python_checks_refuse_host_tensors_and_wrong_planes():
    """The Python operators refuse before any CUDA call: host tensors, wrong types and shapes raise ValueError."""
    i32 = torch.zeros(4, dtype=torch.int32)
    codes, scale = ops.new_kv_cache(64, 2, 128, "cpu", fmt="kv4")
    assert tuple(codes.shape) == (2, 64, 64) and tuple(scale.shape) == (2, 64, 4)
    with pytest.raises(ValueError):
        ops.page_tables(torch.zeros((4, 8), dtype=torch.int32), i32, i32, i32, page_size=16, n_pages=8, rows=4)
    with pytest.raises(ValueError):
        ops.kv4_read_f32(codes, scale)
    with pytest.raises(ValueError):
        ops.attend_paged_kv4(torch.zeros((4, 8, 128)), codes, codes, scale, scale, i32.view(1, 4), i32[:1], page_size=16)
    with pytest.raises(ValueError):
        ops.rope_neox_kv4_append(torch.zeros((4, 8, 128)), torch.zeros((4, 2, 128)), torch.zeros((4, 2, 128)), i32, n_rot=64,
                                 theta_scale=0.5, k_cache=codes, v_cache=codes, k_scale=scale, v_scale=scale)
