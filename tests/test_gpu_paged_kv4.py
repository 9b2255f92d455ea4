"""The paged 4-bit cache on the GPU: block tables, append, read-back and attention against plain statements of each.

Whole numbers (tables, slots, codes, scales) are held to equality: the quantiser's rule is F32 arithmetic, restated here
in numpy.  Attention is held to a 64-bit evaluation over the decoded cells with the error bound of its arithmetic,
element by element: F32 accumulation over tensor-core steps of sixteen terms, every step off by at most 2^-23 of what it
has summed so far (a truncated F32 sum), on both products; see attend_tolerance.
"""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth

pytestmark = pytest.mark.gpu


def to_dev(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


# ---- the format, restated -----------------------------------------------------------------------------------------------

def kv4_rule(x):
    """Codes 0 .. 15 [..., hd] (uint8) and FP16 scales [..., hd / 32] of F32 values."""
    g = np.ascontiguousarray(x, np.float32).reshape(x.shape[:-1] + (-1, 32))
    finite = np.isfinite(g).all(-1)
    g = np.where(finite[..., None], g, np.float32(0))
    top, low = g.max(-1), g.min(-1)
    m = np.where(top >= -low, top, low).astype(np.float32)
    d = torch.from_numpy(m / np.float32(-8)).to(torch.bfloat16).to(torch.float32).numpy()
    d = np.clip(d, -2720, 2720).astype(np.float16)
    wide = d.astype(np.float32)
    inv = np.divide(np.float32(1), wide, out=np.zeros_like(wide), where=wide != 0)
    with np.errstate(over="ignore", invalid="ignore"):
        code = np.clip(np.rint((g * inv[..., None]).astype(np.float32)), -8, 7).astype(np.int64) + 8
    d = np.where(finite, np.where(wide == 0, np.float16(0), d), np.float16(np.nan))
    return code.astype(np.uint8).reshape(x.shape), d


def pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def decode(codes, scale):
    """[..., hd / 2] bytes and FP16 scales to F64 values."""
    v = np.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), np.float64)
    v[..., 0::2] = (codes & 15).astype(np.float64) - 8
    v[..., 1::2] = (codes >> 4).astype(np.float64) - 8
    return v * np.repeat(scale.astype(np.float64), 32, -1)


# ---- append ---------------------------------------------------------------------------------------------------------------

APPEND = [
    # rows, q heads, kv heads, head_dim, n_rot, norms
    (1, 16, 2, 256, 64, True),
    (7, 12, 1, 256, 64, True),
    (300, 16, 2, 256, 128, False),
    (33, 8, 4, 128, 128, True),
    (129, 32, 8, 128, 64, True),
    (50, 4, 4, 64, 64, True),
    (5, 2, 1, 64, 0, False),
    (19, 6, 2, 256, 32, True),     # rotary halves inside a 32-value block: the row-per-warp kernel
    (3, 6, 2, 128, 24, True),
    (40, 3, 3, 64, 36, False),
    (6, 0, 2, 128, 64, True),      # K and V alone
]


@pytest.mark.parametrize("rows,n_q,n_kv,hd,n_rot,norms", APPEND)
def test_append_writes_the_rules_codes(dev, rows, n_q, n_kv, hd, n_rot, norms):
    g = synth.rng(rows * 31 + hd)
    slots_n = rows + 40
    q, k, v = (synth.normal(g, (rows, n, hd), 1.0) for n in (n_q, n_kv, n_kv))
    w = [to_dev(1 + 0.1 * synth.normal(g, (hd,)), dev) if norms else None for _ in range(2)]
    pos = (np.arange(rows) + 250000).astype(np.int32)
    slots = g.permutation(slots_n)[:rows].astype(np.int32)
    slots[::5] = -1                                                    # padding
    kc, ks = ops.new_kv_cache(slots_n, n_kv, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(slots_n, n_kv, hd, dev, fmt="kv4")
    for t in (kc, vc):
        t.fill_(0xA5)
    for t in (ks, vs):
        t.fill_(-77)
    ts = ops.theta_scale(1e7, n_rot) if n_rot else 1.0
    d = [to_dev(x, dev) for x in (q, k, v)]
    err = ops.new_err(dev)
    q_out, kf = torch.full_like(d[0], -3.0), torch.full_like(d[1], -3.0)
    ops.rope_neox_kv4_append(*d, to_dev(pos, dev), n_rot=n_rot, theta_scale=ts, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs,
                             slots=to_dev(slots, dev), q_norm_w=w[0], k_norm_w=w[1], q_out=q_out, k_f32=kf, err=err)
    # the same step into 8-bit cells, whose F32 rows are pinned elsewhere
    c8 = [ops.new_kv_cache(slots_n, n_kv, hd, dev) for _ in range(2)]
    q8, k8 = torch.full_like(d[0], -3.0), torch.full_like(d[1], -3.0)
    ops.rope_neox_q8_0_append(*d, to_dev(pos, dev), n_rot=n_rot, theta_scale=ts, k_cache=c8[0], v_cache=c8[1],
                              slots=to_dev(slots, dev), q_norm_w=w[0], k_norm_w=w[1], q_out=q8, k_f32=k8)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(q_out, q8) and torch.equal(kf, k8)              # padding rows untouched in both
    live = slots >= 0
    for codes, scale, rows_f32 in ((kc, ks, kf.cpu().numpy()), (vc, vs, v)):
        want_c = np.full(codes.shape, 0xA5, np.uint8)
        want_s = np.full(scale.shape, -77, np.int16)
        c, s = kv4_rule(rows_f32)
        want_c[:, slots[live]] = pack(c)[live].transpose(1, 0, 2)
        want_s[:, slots[live]] = s.view(np.int16)[live].transpose(1, 0, 2)
        assert np.array_equal(codes.cpu().numpy(), want_c)
        assert np.array_equal(scale.cpu().numpy(), want_s)


@pytest.mark.parametrize("hd,n_rot", [(256, 0), (128, 0), (64, 0), (128, 24)])
def test_append_special_groups(dev, hd, n_rot):
    """Zeros, ties of either order, values that overflow or underflow the scale, infinities and NaN; n_rot 24 takes the
    row-per-warp kernel.  V passes through the quantiser alone."""
    g = synth.rng(5)
    rows = 24
    v = synth.normal(g, (rows, 1, hd))
    f = v.reshape(rows, -1, 32)
    f[0] = 0.0
    f[1, :, 3], f[1, :, 9] = 4.0, -4.0
    f[2, :, 3], f[2, :, 9] = -4.0, 4.0
    f[3] *= 1e30
    f[4] *= 1e-7                                                     # subnormal FP16 scales
    f[5] *= 1e-9                                                     # scales that round to zero
    f[6, :, 31] = 3.4e38
    f[7, 0, 0] = np.inf
    f[8, :, 17] = -np.inf
    f[9, 0, 5] = np.nan
    f[10, -1, 30], f[10, -1, 2] = np.nan, np.inf
    f[11] = -0.0
    f[12] = 1e-45
    f[13] = np.arange(-16, 16) * 0.5                                 # quotients on the border between two codes
    f[14] = 21760.0
    f[15] = 30000.0
    kc, ks = ops.new_kv_cache(rows, 1, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(rows, 1, hd, dev, fmt="kv4")
    k = np.zeros_like(v)
    q = np.zeros((rows, 1, hd), np.float32)
    err = ops.new_err(dev)
    ops.rope_neox_kv4_append(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), to_dev(np.arange(rows, dtype=np.int32), dev), n_rot=n_rot,
                             theta_scale=0.5, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, err=err)
    got = ops.kv4_read_f32(vc, vs).cpu().numpy()
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    c, s = kv4_rule(v)
    assert np.array_equal(vc.cpu().numpy()[0], pack(c)[:, 0])
    assert np.array_equal(vs.cpu().numpy()[0], s.view(np.int16)[:, 0])
    want = decode(vc.cpu().numpy(), vs.cpu().numpy().view(np.float16))[0]
    assert np.array_equal(got[:, 0].astype(np.float64), want, equal_nan=True)
    bad = np.isnan(got[:, 0].reshape(rows, -1, 32))
    assert bad.any(-1).sum() == bad.all(-1).sum() == 3 + hd // 32   # rows 7, 9 and 10 hold one bad group each, row 8 all of its


def test_append_bad_slots_and_planes(dev):
    """A slot outside the cache is flagged and writes nothing; position planes of image rows go through as in the 8-bit form."""
    g = synth.rng(8)
    rows, n_q, n_kv, hd = 9, 4, 2, 256
    d = [to_dev(synth.normal(g, (rows, n, hd)), dev) for n in (n_q, n_kv, n_kv)]
    slots = np.array([0, 1, 64, 2, -2, 3, -1, 4, 5], np.int32)
    kc, ks = ops.new_kv_cache(64, n_kv, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(64, n_kv, hd, dev, fmt="kv4")
    planes = to_dev(g.integers(0, 5000, (rows, 4)).astype(np.int32), dev)
    err = ops.new_err(dev)
    kw = dict(n_rot=64, theta_scale=ops.theta_scale(1e7, 64), slots=to_dev(slots, dev), planes=planes)
    pos = to_dev(np.arange(rows, dtype=np.int32), dev)
    q_out, kf = torch.zeros_like(d[0]), torch.zeros_like(d[1])
    ops.rope_neox_kv4_append(*d, pos, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, q_out=q_out, k_f32=kf, err=err, **kw)
    c8 = [ops.new_kv_cache(64, n_kv, hd, dev) for _ in range(2)]
    q8, k8 = torch.zeros_like(d[0]), torch.zeros_like(d[1])
    ops.rope_neox_q8_0_append(*d, pos, k_cache=c8[0], v_cache=c8[1], q_out=q8, k_f32=k8, **kw)
    torch.cuda.synchronize()
    assert int(err.item()) == ops.ERR_SLOT
    assert torch.equal(q_out, q8) and torch.equal(kf, k8)
    assert not bool(vs[:, 6:].any())
    assert bool((vs[:, :6] != 0).all())


# ---- read -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_kv,rows", [(256, 2, 1), (256, 1, 333), (128, 8, 77), (64, 3, 500), (64, 1, 1)])
def test_read_widens_exactly(dev, hd, n_kv, rows):
    g = synth.rng(rows + hd)
    slots = rows + 21
    codes = g.integers(0, 256, (n_kv, slots, hd // 2)).astype(np.uint8)
    scale = (synth.normal(g, (n_kv, slots, hd // 32)) * 3).astype(np.float16)
    cells = g.permutation(slots)[:rows].astype(np.int32)
    cells[rows // 2] = -1 if rows > 1 else cells[0]
    dc, ds = to_dev(codes, dev), to_dev(scale.view(np.int16), dev)
    err = ops.new_err(dev)
    out = torch.full((rows, n_kv, hd), 5.0, device=dev)
    ops.kv4_read_f32(dc, ds, cells=to_dev(cells, dev), out=out, err=err)
    span = ops.kv4_read_f32(dc, ds, cell0=21)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    v = decode(codes, scale).transpose(1, 0, 2)
    want = np.where((cells >= 0)[:, None, None], v[cells], 5.0)
    assert np.array_equal(out.cpu().numpy().astype(np.float64), want)
    assert np.array_equal(span.cpu().numpy().astype(np.float64), v[21:])
    bad = cells.copy()
    bad[0] = slots
    ops.kv4_read_f32(dc, ds, cells=to_dev(bad, dev), out=out.fill_(5.0), err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == ops.ERR_SLOT
    assert np.array_equal(out.cpu().numpy()[0], np.full((n_kv, hd), 5.0))


# ---- block tables ---------------------------------------------------------------------------------------------------------

def tables_plain(table, old, new, free, head, page, n_pages, rows):
    """The definition, request by request."""
    table = table.copy()
    slots, pos = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    start, n_cells, taken, row, fault, wanted = [0], [], 0, 0, False, 0
    for r, (o, n) in enumerate(zip(old.tolist(), new.tolist())):
        ok = o >= 0 and n >= 0 and o + n <= table.shape[1] * page
        first, row = row, row + max(n, 0)
        ok = ok and row <= rows
        grow = -(-(o + n) // page) - -(-o // page) if ok else 0
        wanted += grow
        if grow and wanted > (len(free) - head if 0 <= head <= len(free) else 0):
            ok = False
        if ok:
            held = -(-o // page)
            table[r, held:held + grow] = free[head + taken:head + taken + grow]
            taken += grow
            for i in range(n):
                p = table[r, (o + i) // page]
                pos[first + i] = o + i
                if 0 <= p < n_pages:
                    slots[first + i] = p * page + (o + i) % page
                else:
                    fault = True
        fault = fault or not ok
        n_cells.append(o + n if ok else o)
        start.append(min(row, rows))
    return table, slots, pos, np.array(start), np.array(n_cells), head + taken, fault


def run_tables(dev, old, new, page, rows, *, spare=3, n_free=None, head=2, inplace=False, max_pages=None, spoil=None):
    g = synth.rng(old.size * 7 + page)
    n_req = old.size
    held = -(-np.maximum(old, 0) // page)
    need = -(-np.maximum(old + new, 0) // page)
    max_pages = int(max(need.max(), held.max(), 1) + spare) if max_pages is None else max_pages
    total = int(np.minimum(need, 10**5).sum()) + 20    # of a length that no table row can list, no more
    ids = g.permutation(total).astype(np.int32)
    table = np.full((n_req, max_pages), -9, np.int32)
    at = 0
    for r in range(n_req):
        k = min(int(held[r]), max_pages)
        table[r, :k] = ids[at:at + k]
        at += k
    free = ids[at:] if n_free is None else ids[at:at + n_free]
    if spoil is not None:
        spoil(table, free)
    d = [to_dev(x.astype(np.int32), dev) for x in (table, old, new, free)]
    head_t = to_dev(np.array([head], np.int32), dev)
    err = ops.new_err(dev)
    kw = dict(n_cells=d[1], free_head_out=head_t) if inplace else {}
    t = ops.page_tables(*d, page_size=page, n_pages=total, rows=rows, free_head=head_t, err=err, **kw)
    torch.cuda.synchronize()
    want = tables_plain(table, old, new, free, head, page, total, rows)
    for name, got, w in zip(("table", "slots", "pos", "row_start", "n_cells", "free_head"),
                            (d[0], t.slots, t.pos, t.row_start, t.n_cells, t.free_head), want):
        assert np.array_equal(got.cpu().numpy().astype(np.int64).reshape(-1), np.asarray(w, np.int64).reshape(-1)), name
    assert int(err.item()) == (ops.ERR_PAGES if want[-1] else 0)
    return want


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("n_req,top_old,top_new,page,pad", [
    (1, 0, 1, 16, 0), (1, 5000, 1, 64, 3), (3, 40, 100, 16, 5), (64, 3000, 1, 16, 0), (200, 900, 9, 1, 1), (1024, 50, 3, 32, 17),
    (1025, 50, 2, 16, 0), (2048, 70, 4, 256, 9), (7, 100, 9000, 16, 40), (2048, 10, 40, 16, 1), (1, 0, 70000, 16, 0)])
def test_page_tables_match_the_definition(dev, n_req, top_old, top_new, page, pad, inplace):
    g = synth.rng(n_req + top_new)
    old = g.integers(0, top_old + 1, n_req)
    new = g.integers(0, top_new + 1, n_req)
    old[n_req // 2] = 0
    new[-1] = top_new
    run_tables(dev, old, new, page, int(new.sum()) + pad, inplace=inplace)


def test_page_tables_without_rows_or_room(dev):
    old, new = np.array([16, 0, 5, 32]), np.array([0, 0, 0, 0])
    run_tables(dev, old, new, 16, 1)                                         # nothing to do: one row of padding
    g = synth.rng(3)
    old, new = g.integers(0, 60, 50), g.integers(0, 60, 50)
    rows = int(new.sum())
    full = run_tables(dev, old, new, 16, rows, n_free=40)                     # the free list gives out on the way
    assert full[-1] and full[5] <= 40
    run_tables(dev, old, new, 16, rows, n_free=0, head=0)
    run_tables(dev, old, new, 16, rows, n_free=10, head=11)                   # an index behind the list
    run_tables(dev, old, new, 16, rows, n_free=10, head=-1)
    run_tables(dev, old, new, 16, rows - 200)                                 # rows that end behind the launch's
    old[7], new[20], new[21] = -4, -1, 2**31 - 1
    run_tables(dev, old, new, 16, rows + 60, max_pages=12)
    run_tables(dev, np.array([10, 20]), np.array([30, 500]), 16, 600, max_pages=3)   # longer than a table row


def test_page_tables_flag_page_ids_outside_the_cache(dev):
    def spoil(table, free):
        table[1, 2] = 10**6                                                   # a page request 1 already holds and still fills
        free[3] = -5
    old, new = np.array([4, 40, 100]), np.array([20, 3, 40])
    run_tables(dev, old, new, 16, 70, spoil=spoil)


# ---- attention ------------------------------------------------------------------------------------------------------------

def make_pages(g, dev, lens, n_kv, hd, page, spare=4, garbage=True):
    """Random cells in shuffled pages: device planes, table, and the host's decoded values."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    slots = n_pages * page
    codes = [np.clip(np.rint(synth.normal(g, (n_kv, slots, hd)) * 2.9), -8, 7).astype(np.int64) + 8 for _ in range(2)]
    scale = [(np.exp(0.3 * synth.normal(g, (n_kv, slots, hd // 32))) * np.sign(synth.normal(g, (n_kv, slots, hd // 32))) * 0.3)
             for _ in range(2)]
    scale = [torch.from_numpy(s.astype(np.float32)).to(torch.bfloat16).to(torch.float16).numpy() for s in scale]
    codes = [pack(c.astype(np.uint8)) for c in codes]
    ids = g.permutation(n_pages)
    table = np.full((len(lens), max(max(need), 1) + 1), -1, np.int32)
    at, used = 0, np.zeros(slots, bool)
    for r, n in enumerate(lens):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        used[slots_of(table, r, n, page)] = True
    if garbage:
        for s in scale:
            s[:, ~used] = np.float16(np.nan)
        codes[0][:, ~used] = 0xFF
    planes = [to_dev(codes[0], dev), to_dev(codes[1], dev), to_dev(scale[0].view(np.int16), dev), to_dev(scale[1].view(np.int16), dev)]
    return planes, table, decode(codes[0], scale[0]), decode(codes[1], scale[1])


def slots_of(table, r, n, page):
    return (table[r, :-(-n // page)].astype(np.int64)[:, None] * page + np.arange(page)).reshape(-1)[:n]


def attend_plain(q, kv, vv, table, lens, rows, page, scale, gate):
    """64-bit attention, and beside it the tolerance of each element: (2 delta + (8 + n / 16) 2^-23 + 2^-20) sum p |v|.
    delta bounds a score's error: its sum of |scale q k| times one truncated F32 step (2^-23) for each of the hd / 8 steps
    of the split product and the hd / 32 groups, the query's residual (2^-22) and two roundings of the F32 result.  A
    weight is then off by at most 2 delta of itself (numerator and denominator).  The output's own sum takes two steps
    for every sixteen cells, each off by at most 2^-23 of a partial sum that is half the whole on average.  2^-20 covers the
    probabilities' exp2 and residual (2^-22 each) and the division, the sigmoid and the products at the end."""
    n_kv, hd = kv.shape[0], q.shape[2]
    group = q.shape[1] // n_kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for r, (n, m) in enumerate(zip(lens, rows)):
        s = slots_of(table, r, n, page)
        for i in range(m):
            upto = n - m + i + 1
            if upto > 0:
                for h in range(q.shape[1]):
                    k, v = kv[h // group, s[:upto]], vv[h // group, s[:upto]]
                    x = q[at + i, h].astype(np.float64)
                    z = scale * (k @ x)
                    w = np.exp(z - z.max())
                    w /= w.sum()
                    delta = 2.0**-23 * (hd / 8 + hd / 32 + 4) * scale * (np.abs(k) @ np.abs(x)).max()
                    out[at + i, h] = w @ v
                    tol[at + i, h] = (2 * delta + (8 + upto / 16) * 2.0**-23 + 2.0**-20) * (w @ np.abs(v))
        at += m
    if gate is not None:
        sig = 1 / (1 + np.exp(-gate.astype(np.float64)))
        out, tol = out * sig, tol * sig
    return out, tol


def run_attend(dev, seed, lens, rows, n_q, n_kv, hd, page, *, gate=False, max_rows=None, extra_rows=2, q_scale=1.0, use_row_start=True):
    g = synth.rng(seed)
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    total = sum(rows)
    q = synth.normal(g, (total + extra_rows, n_q, hd), q_scale)
    gt = synth.normal(g, q.shape, 1.5) if gate else None
    start = np.concatenate(([0], np.cumsum(rows))).astype(np.int32)
    out = torch.full(q.shape, 9.0, device=dev)
    err = ops.new_err(dev)
    ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(table, dev), to_dev(np.array(lens, np.int32), dev), page_size=page,
                         row_start=to_dev(start, dev) if use_row_start else None, max_rows=max(rows) if max_rows is None else max_rows,
                         gate=None if gt is None else to_dev(gt, dev), out=out, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    got = out.cpu().numpy().astype(np.float64)
    ref, tol = attend_plain(q[:total], kv, vv, table, lens, rows, page, hd ** -0.5, None if gt is None else gt[:total])
    off = np.abs(got[:total] - ref)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), (float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(off > tol)[:4].tolist())
    assert (got[total:] == 9.0).all()                                     # rows of no request
    return got, ref


@pytest.mark.parametrize("hd,n_q,n_kv,page", [(256, 16, 2, 16), (256, 8, 1, 64), (128, 8, 2, 32), (128, 32, 8, 128), (64, 6, 2, 256),
                                              (64, 4, 4, 16), (256, 12, 1, 512), (128, 3, 1, 16)])
def test_attend_one_row_each_ragged_lengths(dev, hd, n_q, n_kv, page):
    run_attend(dev, 11 + hd + page, [1, 2, 15, 16, 17, 127, 128, 129, 1000, 383], [1] * 10, n_q, n_kv, hd, page)


@pytest.mark.parametrize("hd,n_q,n_kv,page,rows,max_rows", [
    (256, 16, 2, 32, [5, 1, 0, 2, 3], 5),      # 40 columns a head: eight blocks
    (256, 12, 1, 16, [5, 5, 1, 4], 5),         # 60 columns
    (256, 16, 2, 32, [2, 1, 0, 2, 1], 2),      # 16 columns: two blocks
    (256, 8, 2, 16, [3, 8, 1], 8),             # 32 columns: four blocks
    (128, 8, 1, 64, [4, 2, 7], 7), (128, 4, 2, 16, [1, 9, 16], 16), (128, 4, 2, 16, [3, 4, 2], 4),
    (64, 8, 1, 16, [2, 1, 2], 2), (64, 16, 2, 32, [3, 4, 1], 4), (64, 8, 1, 128, [8, 1, 5], 8),
    (256, 16, 2, 16, [20, 1, 9], 20),          # more columns than one pass holds
    (128, 8, 2, 16, [5, 130, 3], 1),           # the hint says one row: more passes, same rows
    (64, 2, 2, 16, [1, 1, 1], 60),             # and the other way round
])
def test_attend_several_rows_are_causal(dev, hd, n_q, n_kv, page, rows, max_rows):
    g = synth.rng(hd + page)
    lens = [int(x) + max(r, 1) for x, r in zip(g.integers(0, 700, len(rows)), rows)]
    run_attend(dev, 5 + hd, lens, rows, n_q, n_kv, hd, page, gate=True, max_rows=max_rows)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attend_rows_that_see_nothing(dev, hd):
    """No cells at all, and more rows than cells: the first of them see nothing and give zeros."""
    got, ref = run_attend(dev, 3, [0, 3, 0, 40], [1, 5, 4, 2], 8, 2, hd, 16, gate=True)
    assert not got[:3].any() and not got[6:10].any()
    run_attend(dev, 4, [0, 0], [1, 2], 4, 1, hd, 16)
    run_attend(dev, 4, [100, 0, 0], [0, 0, 0], 4, 1, hd, 16, max_rows=1)      # nothing to do


def test_attend_without_row_start_and_in_one_tile(dev):
    """One row a request without a row array; a table of at most 128 cells needs no fold."""
    run_attend(dev, 21, [5, 100, 64], [1, 1, 1], 16, 2, 256, 16, use_row_start=False, extra_rows=0)
    run_attend(dev, 22, [5, 300, 64], [1, 1, 1], 16, 2, 256, 16, use_row_start=False, extra_rows=0)


@pytest.mark.parametrize("n_req,lens_top,page", [(150, 40, 16), (300, 600, 16), (2048, 20, 16)])
def test_attend_many_requests(dev, n_req, lens_top, page):
    g = synth.rng(n_req)
    lens = g.integers(0, lens_top + 1, n_req).tolist()
    rows = [int(x) for x in g.integers(0, 3, n_req)]
    run_attend(dev, 40, lens, rows, 2, 1, 128, page, max_rows=2)


@pytest.mark.parametrize("q_scale,n_kv,n_q", [(1.0, 2, 16), (6.0, 1, 8), (0.0, 1, 4)])
def test_attend_long_flat_and_peaked(dev, q_scale, n_kv, n_q):
    """A row cut into many pieces; flat, peaked and (zero queries) even weights."""
    run_attend(dev, 50, [50001, 7], [1, 1], n_q, n_kv, 256, 64, q_scale=q_scale)
    run_attend(dev, 51, [20000], [3], n_q, n_kv, 128, 16, q_scale=q_scale)


def test_attend_is_bitwise_repeatable_and_takes_any_workspace(dev):
    g = synth.rng(60)
    lens = [5000, 70, 1300]
    planes, table, kv, vv = make_pages(g, dev, lens, 2, 256, 32)
    q = to_dev(synth.normal(g, (3, 16, 256)), dev)
    args = (q, *planes, to_dev(table, dev), to_dev(np.array(lens, np.int32), dev))
    first = ops.attend_paged_kv4(*args, page_size=32)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device=dev)          # NaN everywhere
    for _ in range(3):
        assert torch.equal(first, ops.attend_paged_kv4(*args, page_size=32, workspace=ws))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                                                 # another stream than the tensors' own
        other = ops.attend_paged_kv4(*args, page_size=32)
    torch.cuda.synchronize()
    assert torch.equal(first, other)


def test_attend_masked_cells_do_not_touch_the_rows_that_do_not_see_them(dev):
    """A drafted row's cell holds NaN: the rows before it are as if it were not there, the rows from it on show it."""
    g = synth.rng(70)
    for hd, page in ((256, 16), (128, 32), (64, 16)):
        n, m, n_q, n_kv = 200, 4, 8, 2
        planes, table, kv, vv = make_pages(g, dev, [n, 30], n_kv, hd, page)
        slot = int(slots_of(table, 0, n, page)[n - 2])                          # what row 2 of 4 appended
        q = synth.normal(g, (m + 1, n_q, hd))
        start = to_dev(np.array([0, m, m + 1], np.int32), dev)
        call = lambda: ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(table, dev), to_dev(np.array([n, 30], np.int32), dev),  # noqa: E731
                                            page_size=page, row_start=start, max_rows=m).cpu().numpy()
        clean = call()
        planes[3][:, slot, 1] = 0x7E00                                          # V's second group
        out = call()
        assert np.array_equal(out[[0, 1, 4]], clean[[0, 1, 4]])
        assert np.isnan(out[2:4, :, 32:64]).all() and np.array_equal(out[2:4, :, :32], clean[2:4, :, :32])
        assert np.array_equal(out[2:4, :, 64:], clean[2:4, :, 64:])
        planes[3][:, slot, 1] = 0
        planes[2][:, slot, 0] = 0x7E00                                          # K: the scores of the rows that see it
        out = call()
        assert np.isfinite(out[[0, 1, 4]]).all() and np.isnan(out[2:4]).all()


def test_attend_flags_bad_pages_and_ranges(dev):
    g = synth.rng(80)
    lens, page = [300, 100, 50], 16
    planes, table, kv, vv = make_pages(g, dev, lens, 1, 128, page)
    q = to_dev(synth.normal(g, (3, 4, 128)), dev)
    n_cells = to_dev(np.array(lens, np.int32), dev)
    good = ops.attend_paged_kv4(q, *planes, to_dev(table, dev), n_cells, page_size=page)
    for bad_id in (-1, 10**6, 2**31 - 1):
        t = table.copy()
        t[1, 3] = bad_id
        err = ops.new_err(dev)
        out = ops.attend_paged_kv4(q, *planes, to_dev(t, dev), n_cells, page_size=page, err=err)
        assert int(err.item()) == ops.ERR_PAGES
        assert torch.equal(out[[0, 2]], good[[0, 2]])                            # the others are unaffected
    for cells, start in (([300, -5, 50], [0, 1, 2, 3]), ([300, 10**9, 50], [0, 1, 2, 3]), (lens, [0, 1, 2, 9]), (lens, [0, 2, 1, 3]),
                         (lens, [-3, 1, 2, 3])):
        err = ops.new_err(dev)
        ops.attend_paged_kv4(q, *planes, to_dev(np.where(np.arange(table.shape[1]) < 300, np.maximum(table, 0), 0), dev),
                             to_dev(np.array(cells, np.int32), dev), page_size=page, row_start=to_dev(np.array(start, np.int32), dev), err=err)
        torch.cuda.synchronize()
        assert int(err.item()) == ops.ERR_PAGES


def test_offsets_past_32_bits(dev):
    """Planes of more than 4 GB: the last pages of the last head are written, read and attended."""
    n_kv, hd, page, slots = 2, 256, 16, 20_000_000
    kc, ks = ops.new_kv_cache(slots, n_kv, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(slots, n_kv, hd, dev, fmt="kv4")
    g = synth.rng(90)
    n, n_pages = 100, slots // page
    table = np.array([[n_pages - 1, 3, n_pages - 2, n_pages - 7, n_pages - 9, 1, n_pages - 3, -1]], np.int32)
    slot = slots_of(table, 0, n, page).astype(np.int32)
    q, k, v = (synth.normal(g, (n, h, hd)) for h in (8, n_kv, n_kv))
    q_out = ops.rope_neox_kv4_append(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), to_dev(np.arange(n, dtype=np.int32), dev), n_rot=64,
                                     theta_scale=ops.theta_scale(1e7, 64), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs,
                                     slots=to_dev(slot, dev))
    kr = ops.kv4_read_f32(kc, ks, cells=to_dev(slot, dev)).cpu().numpy().astype(np.float64)
    vr = ops.kv4_read_f32(vc, vs, cells=to_dev(slot, dev)).cpu().numpy().astype(np.float64)
    c, s = kv4_rule(v)
    assert np.array_equal(vr, decode(pack(c), s))
    out = ops.attend_paged_kv4(q_out[n - 1:].contiguous(), kc, vc, ks, vs, to_dev(table, dev), to_dev(np.array([n], np.int32), dev),
                               page_size=page)
    # the same cells in a plane of their own
    own = np.arange(8, dtype=np.int32)[None]
    ref, tol = attend_plain(q_out[n - 1:].cpu().numpy(), np.pad(kr.transpose(1, 0, 2), ((0, 0), (0, 28), (0, 0))),
                            np.pad(vr.transpose(1, 0, 2), ((0, 0), (0, 28), (0, 0))), own, [n], [1], page, hd ** -0.5, None)
    assert (np.abs(out.cpu().numpy() - ref) <= tol).all()


# ---- the set together -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,n_q,n_kv,n_rot", [(256, 16, 2, 64), (128, 8, 4, 128)])
def test_steps_through_a_captured_graph(dev, hd, n_q, n_kv, n_rot):
    """What a serving program does: a prefill step of ragged rows, then decode and draft steps through ONE captured graph
    (lengths, free list and row counts live on the device, rows padded to a fixed capacity), each step's attention
    against 64 bits over the values of the cells."""
    g = synth.rng(100)
    n_req, page, cap = 5, 16, 40
    n_pages = 120
    kc, ks = ops.new_kv_cache(n_pages * page, n_kv, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(n_pages * page, n_kv, hd, dev, fmt="kv4")
    for t in (ks, vs):
        t.fill_(0x7E00)                                                        # never-written cells are NaN
    table = torch.full((n_req, 30), -1, dtype=torch.int32, device=dev)
    free = to_dev(g.permutation(n_pages).astype(np.int32), dev)
    n_cells, head = torch.zeros(n_req, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    n_new = torch.zeros(n_req, dtype=torch.int32, device=dev)
    bufs = [torch.zeros((cap, h, hd), device=dev) for h in (n_q, n_kv, n_kv)]
    gate = torch.zeros((cap, n_q, hd), device=dev)
    q_out, out = torch.full_like(bufs[0], 2.0), torch.full_like(bufs[0], 9.0)
    slots, pos = (torch.zeros(cap, dtype=torch.int32, device=dev) for _ in range(2))
    row_start = torch.zeros(n_req + 1, dtype=torch.int32, device=dev)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    err = ops.new_err(dev)
    ts = ops.theta_scale(1e7, n_rot)

    def step():
        ops.page_tables(table, n_cells, n_new, free, page_size=page, n_pages=n_pages, rows=cap, free_head=head, slots=slots, pos=pos,
                        row_start=row_start, n_cells=n_cells, free_head_out=head, err=err)
        ops.rope_neox_kv4_append(*bufs, pos, n_rot=n_rot, theta_scale=ts, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=slots,
                                 q_out=q_out, err=err)
        ops.attend_paged_kv4(q_out, kc, vc, ks, vs, table, n_cells, page_size=page, row_start=row_start, max_rows=4, gate=gate, out=out,
                             workspace=ws, err=err)

    ops.prepare_device()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens = np.zeros(n_req, np.int64)
    for i, new in enumerate(([13, 1, 0, 17, 9], [1, 1, 1, 1, 1], [4, 1, 0, 2, 3], [1, 0, 30, 1, 1], [0, 0, 0, 0, 0], [3, 1, 1, 1, 15])):
        new = np.array(new)
        n_new.copy_(to_dev(new.astype(np.int32), dev))
        for b in bufs + [gate]:
            b.copy_(to_dev(synth.normal(g, tuple(b.shape)), dev))
        out.fill_(9.0)
        q_out.fill_(2.0)
        graph.replay() if i else step()
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        lens += new
        total = int(new.sum())
        assert np.array_equal(n_cells.cpu().numpy(), lens)
        t = table.cpu().numpy()
        planes = [decode(c.cpu().numpy(), s.cpu().numpy().view(np.float16)) for c, s in ((kc, ks), (vc, vs))]
        ref, tol = attend_plain(q_out[:total].cpu().numpy(), *planes, t, lens.tolist(), new.tolist(), page, hd ** -0.5, gate[:total].cpu().numpy())
        got = out.cpu().numpy()
        assert (np.abs(got[:total] - ref) <= tol).all(), i
        assert (got[total:] == 9.0).all() and bool((q_out[total:] == 2.0).all())
