"""Paged attention over part of a wide table and over pages that requests share, on the GPU."""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth
from test_gpu_paged_kv4 import attend_plain, make_pages, to_dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,n_q,n_kv", [(256, 16, 2), (128, 8, 4), (64, 2, 2)])
def test_first_columns_of_a_wide_table(dev, hd, n_q, n_kv):
    """The view table[:, :w] gives the bits of its contiguous copy, whichever way its width has the work split."""
    g = synth.rng(400 + hd)
    lens, page = [250, 0, 33, 256, 1, 100], 16
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    big = np.full((6, 1000), 0x7FFFFFF0, np.int32)                     # ids outside the cache behind what a view shows
    big[:, :16] = table[:, :16]
    q = synth.normal(g, (6, n_q, hd))
    ref, tol = attend_plain(q, kv, vv, table, lens, [1] * 6, page, hd ** -0.5, None)
    wide, n = to_dev(big, dev), to_dev(np.array(lens, np.int32), dev)
    for w in (16, 17, 200, 999):
        err = ops.new_err(dev)
        got = ops.attend_paged_kv4(to_dev(q, dev), *planes, wide[:, :w], n, page_size=page, err=err)
        same = ops.attend_paged_kv4(to_dev(q, dev), *planes, wide[:, :w].contiguous(), n, page_size=page, err=err)
        assert int(err.item()) == 0 and torch.equal(got, same), w
        assert (np.abs(got.cpu().numpy() - ref) <= tol).all(), w
    one = ops.attend_paged_kv4(to_dev(q[:1], dev), *planes, wide[:1, :16], n[:1], page_size=page)   # one row: any stride
    assert (np.abs(one.cpu().numpy() - ref[:1]) <= tol[:1]).all()
    for bad in (wide[:, ::2], wide.t()):
        with pytest.raises(ValueError):
            ops.attend_paged_kv4(to_dev(q, dev), *planes, bad, n, page_size=page)
    with pytest.raises(ValueError):
        ops.attend_paged_kv4(to_dev(q, dev), *planes, wide[:1, :16].expand(6, 16), n, page_size=page)


def test_requests_share_pages(dev):
    """A common prefix listed by every request, and one request's table given twice."""
    g = synth.rng(410)
    hd, n_q, n_kv, page = 128, 8, 2, 16
    planes, table, kv, vv = make_pages(g, dev, [300, 500, 400], n_kv, hd, page)
    rows = np.full((5, 34), -1, np.int32)
    rows[:, :6] = table[0, :6]                                         # 96 cells of prefix
    rows[0, 6:19], rows[1, 6:32], rows[2, 6:25], rows[3, 6:32], rows[4] = table[0, 6:19], table[1, 6:32], table[2, 6:25], table[1, 6:32], rows[1]
    rows[4, 6:32] = rows[1, 6:32]
    lens = [300, 500, 400, 500, 499]
    q = synth.normal(g, (5, n_q, hd))
    q[3] = q[1]
    ref, tol = attend_plain(q, kv, vv, rows, lens, [1] * 5, page, hd ** -0.5, None)
    for width in (34, 400):
        wide = np.full((5, width), -1, np.int32)
        wide[:, :34] = rows
        err = ops.new_err(dev)
        got = ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(wide, dev), to_dev(np.array(lens, np.int32), dev), page_size=page, err=err)
        assert int(err.item()) == 0 and (np.abs(got.cpu().numpy() - ref) <= tol).all(), width


def test_more_tiles_than_the_line_counts(dev):
    """Lengths that are valid one by one but make 2^31 tiles or more together: flagged, nothing read or written."""
    n_req, page = 400, 1 << 20
    kc, ks = ops.new_kv_cache(page, 1, 64, dev, fmt="kv4")
    table = torch.zeros((n_req, 2047), dtype=torch.int32, device=dev)
    lens = torch.full((n_req,), 2047 * page, dtype=torch.int32, device=dev)
    q = torch.ones((n_req, 8, 64), device=dev)
    out, err = torch.full_like(q, 9.0), ops.new_err(dev)
    ops.attend_paged_kv4(q, kc, kc, ks, ks, table, lens, page_size=page, out=out, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == ops.ERR_PAGES and bool((out == 9.0).all())


@pytest.mark.parametrize("rows,shift", [(30, 1), (5000, 0), (20000, 1), (20003, 2), (66001, 3)])
def test_slot_map_in_arrays_of_any_alignment(dev, rows, shift):
    """Slots and positions into views that begin anywhere: the same numbers, and nothing beside them."""
    g = synth.rng(420 + rows)
    n_req, page = 37, 16
    old = g.integers(0, 90, n_req).astype(np.int32)
    new = np.diff(np.concatenate(([0], np.sort(g.integers(0, rows - 4, n_req - 1)), [rows - 5]))).astype(np.int32)
    held = -(-old // page)
    n_pages = int((-(-(old + new) // page)).sum()) + 5
    ids = g.permutation(n_pages).astype(np.int32)
    table = np.full((n_req, int((-(-(old + new) // page)).max()) + 1), -1, np.int32)
    at = 0
    for r in range(n_req):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    want_slot, want_pos = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    i, free = 0, at
    for r in range(n_req):
        need = -(-(old[r] + new[r]) // page) - held[r]
        pages = np.concatenate((table[r, :held[r]], ids[free:free + need])).astype(np.int64)
        free += need
        c = old[r] + np.arange(new[r])
        want_slot[i:i + new[r]], want_pos[i:i + new[r]] = pages[c // page] * page + c % page, c
        i += int(new[r])
    slots, pos = (torch.full((rows + 8,), 77, dtype=torch.int32, device=dev) for _ in range(2))
    err = ops.new_err(dev)
    ops.page_tables(to_dev(table, dev), to_dev(old, dev), to_dev(new, dev), to_dev(ids[at:], dev), page_size=page, n_pages=n_pages,
                    rows=rows, slots=slots[shift:shift + rows], pos=pos[shift:shift + rows], err=err)
    assert int(err.item()) == 0
    for got, want in ((slots, want_slot), (pos, want_pos)):
        got = got.cpu().numpy()
        assert np.array_equal(got[shift:shift + rows], want)
        assert (got[:shift] == 77).all() and (got[shift + rows:] == 77).all()
