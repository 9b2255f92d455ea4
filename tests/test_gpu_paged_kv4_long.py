"""Paged attention over many cells and many rows, held to bounds that a cell lost or counted twice would break.

The bound of an output is its arithmetic's, term by term, times sum p |v|:
  2 delta        the scores: delta as in test_gpu_paged_kv4.attend_plain (0 for queries of zero)
  32 2^-23       the tensor core's sums of one tile: at most two steps for each of at most 16 runs of cells, each off by at
                 most 2^-23 of what the tile has summed
  (t + 64) 2^-24 the joins in rounded F32: t tiles one after the other in a CTA, then the groups of cells, the pieces (a thread
                 at most ten of 296, then 32 threads) and the weights' own sums
  2^-20          exp2, the second parts' residuals (2^-22 each), the division
and beside them 2^-39 times the sum of |v| alone: a weight's second part is FP16, whose smallest step is 2^-24, so a weight is off
by up to 2^-25 however small it is, where the row's largest is 2^14.  That shows where the cells that lead a row hold a value
of zero, and what is left of sum p |v| comes from weights below 2^-17 of the largest.
For even weights over 50 000 cells that is 9e-6 of sum p |v|, and one cell is 2e-5 of it.
"""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth
from test_gpu_paged_kv4 import make_pages, slots_of, to_dev

pytestmark = pytest.mark.gpu


def reference(q, kv, vv, table, lens, rows, page):
    """64-bit attention, [row][head][dim], and what `bound` needs: sum p |v|, sum |v|, the scores' delta."""
    n_kv, hd = kv.shape[0], q.shape[2]
    group = q.shape[1] // n_kv
    out, mass, seen, delta = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2] + (1,))
    at = 0
    for r, (n, m) in enumerate(zip(lens, rows)):
        s = slots_of(table, r, n, page)
        upto = np.maximum(n - m + np.arange(m) + 1, 0)
        if m and n:
            hides = torch.from_numpy(np.arange(n)[None, :] >= upto[:, None])[:, None]           # [row][1][cell]
            for h in range(n_kv):
                k, v = (torch.from_numpy(x[h, s]) for x in (kv, vv))
                heads = slice(h * group, (h + 1) * group)
                x = torch.from_numpy(q[at:at + m, heads].astype(np.float64))
                z = (x @ k.T) * hd ** -0.5
                off = (x.abs() @ k.abs().T).masked_fill(hides, 0.0).amax(-1, keepdim=True)
                p = torch.softmax(z.masked_fill(hides, -np.inf), -1)
                p = torch.where(torch.isnan(p), 0.0, p)                                         # a row that sees nothing
                out[at:at + m, heads], mass[at:at + m, heads] = p @ v, p @ v.abs()
                seen[at:at + m, heads] = (torch.cumsum(v.abs(), 0)[np.maximum(upto, 1) - 1])[:, None]
                delta[at:at + m, heads] = 2.0**-23 * (hd / 8 + hd / 32 + 4) * hd ** -0.5 * off
        at += m
    return out, (mass, seen, delta)


def bound(terms, lens, rows, group, n_kv):
    mass, seen, delta = terms
    t = np.concatenate([np.full(m, n // 128 + 1) for n, m in zip(lens, rows)])
    units = n_kv * sum(-(-m * group // 4) * (n // 128 + 2) for n, m in zip(lens, rows))
    t = np.minimum(t, units / 296 + 2)[:, None, None]
    return (2 * delta + 32 * 2.0**-23 + (t + 64) * 2.0**-24 + 2.0**-20) * mass + 2.0**-39 * seen


def attend(dev, q, planes, table, lens, rows, page, cells=None, max_rows=None):
    wide = table
    if cells is not None:
        wide = np.full((len(lens), cells // page), -1, np.int32)
        used = min(table.shape[1], cells // page)
        wide[:, :used] = table[:, :used]
    err = ops.new_err(dev)
    start = to_dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32), dev)
    got = ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(wide, dev), to_dev(np.array(lens, np.int32), dev), page_size=page,
                               row_start=start, max_rows=max(rows) if max_rows is None else max_rows, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    return got.cpu().numpy().astype(np.float64)


LONG = [
    # head_dim, query heads, KV heads, page, lengths, rows a request, cells a table row lists
    (256, 16, 2, 64, [50001], 1, None),               # one item a head in hundreds of pieces
    (256, 8, 2, 16, [50001, 7], 1, None),             # four columns in a block
    (256, 16, 2, 64, [30000, 129], 2, None),          # sixteen columns a unit
    (256, 12, 1, 32, [9000, 16384, 1, 700], 5, None),
    (256, 16, 2, 16, [4096, 40, 1000, 2503, 128, 127] * 4, 1, None),
    (128, 32, 8, 128, [20000, 5000], 1, None),
    (128, 16, 2, 32, [40000], 1, None),
    (128, 32, 8, 128, [3000, 33, 2049, 256, 257, 1] * 7, 1, None),   # many items, few pieces each
    (64, 8, 1, 16, [50001], 1, None),
    (64, 32, 8, 16, [8192, 255, 3000], 1, None),
    (256, 16, 2, 16, [1000, 1024, 1], 1, 1024),       # clusters
    (128, 8, 2, 16, [2047, 2048, 129], 1, 2048),
    (64, 8, 2, 16, [2047, 500, 129], 1, 2048),
    (256, 16, 2, 16, [256, 255, 129, 1] * 20, 1, 256),  # whole
]


@pytest.mark.parametrize("hd,n_q,n_kv,page,lens,m,cells", LONG)
def test_even_weights_count_every_cell_once(dev, hd, n_q, n_kv, page, lens, m, cells):
    """Queries of zero: the mean of the cells a row sees."""
    g = synth.rng(hd + len(lens))
    rows = [m] * len(lens)
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    q = np.zeros((sum(rows), n_q, hd), np.float32)
    ref, terms = reference(q, kv, vv, table, lens, rows, page)
    tol = bound(terms, lens, rows, n_q // n_kv, n_kv)
    off = np.abs(attend(dev, q, planes, table, lens, rows, page, cells) - ref)
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("hd,n_q,n_kv,page,lens,m,cells", LONG)
def test_marked_cells_beside_every_border(dev, hd, n_q, n_kv, page, lens, m, cells):
    """Only the cells on either side of a tile's border, where work is cut, hold values: each is a part of its own size of the sum."""
    g = synth.rng(7 * hd + len(lens))
    rows = [m] * len(lens)
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page, garbage=False)
    keep = np.zeros(vv.shape[1], bool)
    for r, n in enumerate(lens):
        c = np.arange(n)
        keep[slots_of(table, r, n, page)[(c % 128 == 0) | (c % 128 == 127) | (c == n - 1)]] = True
    gone = to_dev(np.flatnonzero(~keep), dev)
    planes[3].index_fill_(1, gone, 0)                                           # their scales are 0
    vv = np.where(keep[None, :, None], vv, 0.0)
    q = np.zeros((sum(rows), n_q, hd), np.float32)
    ref, terms = reference(q, kv, vv, table, lens, rows, page)
    tol = bound(terms, lens, rows, n_q // n_kv, n_kv)
    off = np.abs(attend(dev, q, planes, table, lens, rows, page, cells) - ref)
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("q_scale", [1.0, 6.0])
@pytest.mark.parametrize("hd,n_q,n_kv,page,lens,m,cells", LONG)
def test_error_of_the_whole_output(dev, hd, n_q, n_kv, page, lens, m, cells, q_scale):
    """The bound element by element, and the 2-norm within 2e-6 of the output's (the header says about 5e-7; scores four times
    as large as usual count four times)."""
    g = synth.rng(3 * hd + len(lens))
    rows = [m] * len(lens)
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    q = synth.normal(g, (sum(rows), n_q, hd), q_scale)
    ref, terms = reference(q, kv, vv, table, lens, rows, page)
    tol = bound(terms, lens, rows, n_q // n_kv, n_kv)
    off = np.abs(attend(dev, q, planes, table, lens, rows, page, cells) - ref)
    assert (off <= tol).all(), float((off / np.maximum(tol, 1e-300)).max())
    assert np.linalg.norm(off) <= 2e-6 * max(1.0, q_scale / 1.5) * np.linalg.norm(ref)


PROMPTS = [
    # head_dim, query heads, KV heads, page, lengths, rows, the hint
    (256, 8, 1, 16, [900, 5, 301], [700, 1, 301], 700),
    (256, 16, 2, 64, [1500], [1500], 1500),
    (256, 4, 2, 32, [3000, 64], [257, 64], 257),
    (128, 8, 2, 16, [900, 5, 301], [700, 1, 301], 700),
    (128, 16, 2, 128, [2300], [1030], 1030),
    (128, 8, 2, 16, [600, 40], [600, 0], 1),            # a hint of one row
    (64, 8, 2, 16, [900, 5, 301], [700, 1, 301], 700),
    (64, 2, 1, 256, [1200], [1200], 1200),
    (256, 8, 1, 16, [100, 400], [300, 399], 399),       # more rows than cells: the first see nothing
]


@pytest.mark.parametrize("hd,n_q,n_kv,page,lens,rows,hint", PROMPTS)
def test_prompts(dev, hd, n_q, n_kv, page, lens, rows, hint):
    """Requests of a prompt's size, from their first cell or behind cells they held before."""
    g = synth.rng(hd + lens[0])
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    q = synth.normal(g, (sum(rows), n_q, hd))
    ref, terms = reference(q, kv, vv, table, lens, rows, page)
    tol = bound(terms, lens, rows, n_q // n_kv, n_kv)
    for cells in (None, 1 << 16):                       # the longest request's table, and a wide one
        off = np.abs(attend(dev, q, planes, table, lens, rows, page, cells, hint) - ref)
        assert (off <= tol).all(), (cells, float((off / np.maximum(tol, 1e-300)).max()))
