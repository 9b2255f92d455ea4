"""Paged attention where scores are large: queries far outside the usual range, up to the header's limit, in every form
the step takes (cells cut over the machine and folded, whole requests, clusters).

A row whose best cell leads by more than the scores can be off, and by 60 beside that, has that cell's values for an
answer: the others' weights together are below n e^-60.  What is left is the weight's residual (2^-22), the division and
the sums of a tile: 2^-20 of the value covers them.  Where several cells come that close together F32 scores do not say
which leads, so such rows are only held to the hull of their cells' values."""
import numpy as np
import pytest

import torch

from fnfl_v100_b200 import ops, synth
from test_gpu_paged_kv4 import make_pages, slots_of, to_dev

pytestmark = pytest.mark.gpu

FORMS = [
    # lengths, cells a table row lists
    ([3000, 1, 700, 5000], 6000),                 # cut and folded
    ([256, 17, 130, 1] * 40, 256),                # whole
    ([500, 129, 40, 1000], 1024),                 # clusters
]
SHAPES = [
    # head_dim, query heads, KV heads, rows a request
    (256, 16, 2, 1), (256, 8, 2, 1), (256, 16, 2, 2), (128, 8, 2, 1), (128, 8, 1, 2), (64, 4, 1, 1),
]


def leads(q, kv, vv, table, lens, m, page, n_kv):
    """For each row and head: the best cell's value, whether it leads by enough, and its cells' smallest and largest value."""
    rows, n_q, hd = q.shape
    group = n_q // n_kv
    best, low, high = (np.zeros(q.shape) for _ in range(3))
    clear = np.zeros((rows, n_q), bool)
    for r, n in enumerate(lens):
        s = slots_of(table, r, n, page)
        for i in range(m):
            upto, t = n - m + i + 1, r * m + i
            if upto < 1:
                clear[t] = True
                continue
            for h in range(n_kv):
                k, v = kv[h, s[:upto]], vv[h, s[:upto]]
                x = q[t, h * group:(h + 1) * group].astype(np.float64)
                z = (x @ k.T) * hd ** -0.5
                delta = 2.0**-23 * (hd / 8 + hd / 32 + 4) * hd ** -0.5 * (np.abs(x) @ np.abs(k).T).max(-1)
                top = np.sort(z, -1)
                lead = top[:, -1] - top[:, -2] if upto > 1 else np.full(group, np.inf)
                heads = slice(h * group, (h + 1) * group)
                clear[t, heads] = lead > 2 * delta + 60
                best[t, heads] = v[z.argmax(-1)]
                low[t, heads], high[t, heads] = v.min(0), v.max(0)
    return best, clear, low, high


def large_case(lens, cells, hd, n_q, n_kv, m, q_scale, dev):
    g = synth.rng(len(lens) + hd + n_q)
    page = 16
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    wide = np.full((len(lens), cells // page), -1, np.int32)
    used = min(table.shape[1], cells // page)
    wide[:, :used] = table[:, :used]
    q = synth.normal(g, (len(lens) * m, n_q, hd)) * np.float32(q_scale)
    return planes, wide, q, leads(q, kv, vv, table, lens, m, page, n_kv), page


@pytest.mark.parametrize("hd,n_q,n_kv,m", SHAPES)
@pytest.mark.parametrize("lens,cells", FORMS)
@pytest.mark.parametrize("q_scale", [3e5, 3e7, 1e8, 1e12, 2.0**60])
def test_one_cell_leads(dev, q_scale, lens, cells, hd, n_q, n_kv, m):
    planes, table, q, (best, clear, low, high), page = large_case(lens, cells, hd, n_q, n_kv, m, q_scale, dev)
    assert clear.mean() > 0.95
    start = to_dev((np.arange(len(lens) + 1) * m).astype(np.int32), dev)
    err = ops.new_err(dev)
    got = ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(table, dev), to_dev(np.array(lens, np.int32), dev), page_size=page,
                               row_start=start, max_rows=m, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    got = got.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:4].tolist()
    off = np.abs(got - best)[clear]
    assert (off <= 2.0**-20 * np.abs(best[clear])).all()
    room = 2.0**-18 * np.maximum(np.abs(low), np.abs(high))
    assert ((got >= low - room) & (got <= high + room)).all()


@pytest.mark.parametrize("hd,n_q,n_kv,m", SHAPES)
@pytest.mark.parametrize("lens,cells", FORMS)
def test_a_query_that_is_no_number_stays_alone(dev, lens, cells, hd, n_q, n_kv, m):
    """One head's query holds an infinity or a NaN: that head's row is NaN, every other row and head keeps its bits."""
    planes, table, q, _, page = large_case(lens, cells, hd, n_q, n_kv, m, 1.0, dev)
    start = to_dev((np.arange(len(lens) + 1) * m).astype(np.int32), dev)
    rest = (*planes, to_dev(table, dev), to_dev(np.array(lens, np.int32), dev))
    call = lambda x: ops.attend_paged_kv4(to_dev(x, dev), *rest, page_size=page, row_start=start, max_rows=m).cpu().numpy()  # noqa: E731
    clean = call(q)
    for row, head, what in ((0, 0, np.nan), (0, n_q - 1, np.inf), (len(lens) * m - 1 - 2 * m, 1, -np.inf), (m, 2, np.nan)):
        x = q.copy()
        x[row, head, 17] = what
        got, same = call(x), np.ones(q.shape[:2], bool)
        same[row, head] = False
        assert np.array_equal(got[same], clean[same])
        assert np.isnan(got[row, head]).all() or lens[row // m] - m + row % m + 1 < 1
