"""Paged attention's two ways of splitting work, on the GPU: requests whose table lists few cells, whose tiles a cluster of
CTAs shares, and the same requests under a wide table, whose tiles go on one line that is cut into pieces."""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth
from test_gpu_paged_kv4 import attend_plain, make_pages, to_dev

pytestmark = pytest.mark.gpu


def widths(dev, seed, lens, rows, n_q, n_kv, hd, page, cells, max_rows, gate=True):
    """The step under tables of each number of cells, against 64 bits; rows of no request stay as they were."""
    g = synth.rng(seed)
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    total = sum(rows)
    q, gt = synth.normal(g, (total + 3, n_q, hd)), synth.normal(g, (total + 3, n_q, hd), 1.5)
    start = to_dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32), dev)
    ref, tol = attend_plain(q[:total], kv, vv, table, lens, rows, page, hd ** -0.5, gt[:total] if gate else None)
    for n in cells:
        wide = np.full((len(lens), n // page), -1, np.int32)
        used = min(table.shape[1], n // page)
        wide[:, :used] = table[:, :used]
        out, err = torch.full(q.shape, 9.0, device=dev), ops.new_err(dev)
        for _ in range(2):
            ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(wide, dev), to_dev(np.array(lens, np.int32), dev), page_size=page,
                                 row_start=start, max_rows=max_rows, gate=to_dev(gt, dev) if gate else None, out=out, err=err)
            got = out.cpu().numpy()
            assert int(err.item()) == 0, n
            assert (np.abs(got[:total] - ref) <= tol).all(), (n, np.argwhere(np.abs(got[:total] - ref) > tol)[:4].tolist())
            assert (got[total:] == 9.0).all(), n


@pytest.mark.parametrize("hd,n_q,n_kv,rows", [(256, 16, 2, 1), (256, 8, 2, 1), (256, 16, 2, 2), (256, 12, 1, 5), (128, 32, 8, 1), (128, 16, 2, 3), (64, 8, 2, 1), (64, 4, 4, 4)])
def test_each_number_of_tiles(dev, hd, n_q, n_kv, rows):
    """Lengths on either side of every tile's end; tables for two, three, four, eight, sixteen and many tiles."""
    lens = [0, 1, 127, 128, 129, 256, 257, 500]
    widths(dev, 300 + hd, lens, [rows] * 8, n_q, n_kv, hd, 16, (512, 528, 1024, 2048, 4096, 20000), rows)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_shares_of_every_size(dev, hd):
    """Numbers of requests that give an item eight, four and two CTAs, and none; some requests are empty or have no rows."""
    for n_req in (1, 5, 18, 37, 74, 149):
        g = synth.rng(n_req)
        lens = g.integers(0, 500, n_req).tolist()
        rows = [int(x) for x in g.integers(0, 2, n_req)]
        rows[0], lens[0] = 1, 512
        widths(dev, 310, lens, rows, 4, 2, hd, 32, (512, 2048), 1, gate=False)


def test_more_items_than_clusters(dev):
    """max_rows says one row where requests have up to forty: clusters take several items one after the other."""
    for hd, n_q, n_kv in ((256, 16, 2), (128, 8, 2), (64, 8, 1), (256, 4, 1)):
        widths(dev, 320, [700, 40, 3, 512], [40, 1, 5, 33], n_q, n_kv, hd, 16, (1024, 2048), 1)


def test_rows_that_do_not_see_a_cell_that_holds_no_number(dev):
    """A drafted row's cell is NaN, in a share that other rows read too: they are as if it were not there."""
    g = synth.rng(330)
    n, m, n_q, n_kv, hd, page = 500, 4, 8, 2, 256, 16
    planes, table, kv, vv = make_pages(g, dev, [n], n_kv, hd, page)
    q = synth.normal(g, (m, n_q, hd))
    start, lens = to_dev(np.array([0, m], np.int32), dev), to_dev(np.array([n], np.int32), dev)
    call = lambda: ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(table, dev), lens, page_size=page, row_start=start, max_rows=m).cpu().numpy()  # noqa: E731
    clean = call()
    slot = int(table[0, (n - 2) // page]) * page + (n - 2) % page                 # row 2 of 4 appended it
    for plane in planes[2:]:
        kept = plane[:, slot].clone()
        plane[:, slot] = 0x7E00
        got = call()
        plane[:, slot] = kept
        assert np.array_equal(got[:2], clean[:2]) and np.isnan(got[2:]).all()


def test_one_captured_graph_over_changing_lengths(dev):
    """The split goes by the table, so one captured call serves all lengths it can list, empty requests and full ones."""
    g = synth.rng(340)
    n_req, page, hd, n_q, n_kv = 6, 16, 128, 8, 2
    full = [1024] * n_req
    planes, table, kv, vv = make_pages(g, dev, full, n_kv, hd, page, garbage=False)
    table = np.ascontiguousarray(table[:, :64])
    q, lens = torch.zeros((n_req, n_q, hd), device=dev), torch.zeros(n_req, dtype=torch.int32, device=dev)
    t, out, err = to_dev(table, dev), torch.zeros((n_req, n_q, hd), device=dev), ops.new_err(dev)
    ops.prepare_device()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attend_paged_kv4(q, *planes, t, lens, page_size=page, out=out, err=err)
    for n in ([1, 2, 3, 4, 5, 6], [1024, 0, 1023, 512, 257, 256], [0] * 6, [700, 800, 900, 1000, 1, 1024]):
        x = synth.normal(g, (n_req, n_q, hd))
        q.copy_(to_dev(x, dev))
        lens.copy_(to_dev(np.array(n, np.int32), dev))
        graph.replay()
        torch.cuda.synchronize()
        ref, tol = attend_plain(x, kv, vv, table, n, [1] * n_req, page, hd ** -0.5, None)
        assert int(err.item()) == 0 and (np.abs(out.cpu().numpy() - ref) <= tol).all(), n
