"""Ways of calling the paged KV4 operators on the GPU: workspaces shared by captured graphs, tables of any width, and the
append over many rows of each head width, against the same statements as the operators' own tests."""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth
from test_gpu_paged_kv4 import attend_plain, decode, kv4_rule, make_pages, pack, to_dev

pytestmark = pytest.mark.gpu


def test_two_captured_graphs_share_a_workspace(dev):
    """Two graphs of different shapes over one workspace, replayed in turn on one stream: neither keeps anything there."""
    g = synth.rng(201)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device=dev)
    ops.prepare_device()
    cases = []
    for hd, n_q, n_kv, page, lens, rows in ((256, 16, 2, 16, [3000, 40, 700], [1, 1, 1]), (128, 8, 2, 32, [900, 5000], [3, 4]),
                                            (256, 16, 2, 32, [400, 2000], [2, 2])):
        planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
        q = to_dev(np.zeros((sum(rows), n_q, hd), np.float32), dev)
        args = (q, *planes, to_dev(table, dev), to_dev(np.array(lens, np.int32), dev))
        start = to_dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32), dev)
        out, err = torch.zeros_like(q), ops.new_err(dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attend_paged_kv4(*args, page_size=page, row_start=start, max_rows=max(rows), out=out, workspace=ws, err=err)
        cases.append((graph, q, out, err, lambda x, a=(kv, vv, table, lens, rows, page, hd ** -0.5, None): attend_plain(x, *a), start, args))
    for _ in range(3):
        fresh = [synth.normal(g, tuple(c[1].shape)) for c in cases]
        for c, x in zip(cases, fresh):
            c[1].copy_(to_dev(x, dev))
        for c in cases:
            c[0].replay()
        torch.cuda.synchronize()
        for c, x in zip(cases, fresh):
            ref, tol = c[4](x)
            assert int(c[3].item()) == 0 and (np.abs(c[2].cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("hd,n_q,n_kv,max_rows", [(256, 16, 2, 1), (128, 8, 2, 3), (64, 4, 4, 1)])
def test_tables_of_any_width_give_the_same_attention(dev, hd, n_q, n_kv, max_rows):
    """A table wide enough for 256 cells keeps requests whole, a wider one cuts them: both within the bound of 64 bits."""
    g = synth.rng(202)
    lens, page = [256, 1, 130, 0, 255], 16
    rows = [min(max_rows, 1 + i % 3) for i in range(5)]
    planes, table, kv, vv = make_pages(g, dev, lens, n_kv, hd, page)
    total = sum(rows)
    q = synth.normal(g, (total, n_q, hd))
    start = to_dev(np.concatenate(([0], np.cumsum(rows))).astype(np.int32), dev)
    ref, tol = attend_plain(q, kv, vv, table, lens, rows, page, hd ** -0.5, None)
    for width in (16, 17, 700):
        wide = np.full((5, width), -1, np.int32)
        wide[:, :16] = table[:, :16]
        err = ops.new_err(dev)
        got = ops.attend_paged_kv4(to_dev(q, dev), *planes, to_dev(wide, dev), to_dev(np.array(lens, np.int32), dev), page_size=page,
                                   row_start=start, max_rows=max_rows, err=err)
        assert int(err.item()) == 0
        assert (np.abs(got.cpu().numpy() - ref) <= tol).all(), width


@pytest.mark.parametrize("rows,n_q,n_kv,hd,n_rot", [(5000, 8, 4, 128, 64), (4097, 8, 8, 64, 32), (3001, 16, 2, 256, 64), (2500, 32, 8, 128, 128)])
def test_append_many_rows(dev, rows, n_q, n_kv, hd, n_rot):
    """Enough rows that every CTA turns its ring of tiles over: codes, scales and rotated queries of every row."""
    g = synth.rng(203 + hd)
    q, k, v = (synth.normal(g, (rows, n, hd)) for n in (n_q, n_kv, n_kv))
    pos = g.integers(0, 1 << 20, rows).astype(np.int32)
    slots = g.permutation(rows + 50)[:rows].astype(np.int32)
    slots[::97] = -1                                                           # padding rows
    kc, ks = ops.new_kv_cache(rows + 50, n_kv, hd, dev, fmt="kv4")
    vc, vs = ops.new_kv_cache(rows + 50, n_kv, hd, dev, fmt="kv4")
    for t in (kc, vc):
        t.fill_(0x3C)
    err, k_f32 = ops.new_err(dev), torch.empty((rows, n_kv, hd), device=dev)
    ts = ops.theta_scale(1e7, n_rot)
    q_out = ops.rope_neox_kv4_append(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), to_dev(pos, dev), n_rot=n_rot, theta_scale=ts,
                                     k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=to_dev(slots, dev), k_f32=k_f32, err=err)
    # queries: the 8-bit append's, which is the same arithmetic before it quantises
    kc8 = torch.zeros((rows + 50, n_kv, hd // 32 * 34), dtype=torch.uint8, device=dev)
    want = ops.rope_neox_q8_0_append(to_dev(q, dev), to_dev(k, dev), to_dev(v, dev), to_dev(pos, dev), n_rot=n_rot, theta_scale=ts,
                                     k_cache=kc8, v_cache=torch.zeros_like(kc8), slots=to_dev(np.where(slots < 0, 0, slots), dev))
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    live = slots >= 0
    assert torch.equal(q_out[torch.from_numpy(live).to(dev)], want[torch.from_numpy(live).to(dev)])
    for codes, scale, src in ((kc, ks, k_f32.cpu().numpy()), (vc, vs, v)):
        code, d = kv4_rule(src[live])
        got_c, got_d = codes.cpu().numpy(), scale.cpu().numpy().view(np.float16)
        assert np.array_equal(got_c[:, slots[live]].transpose(1, 0, 2), pack(code))
        assert np.array_equal(got_d[:, slots[live]].transpose(1, 0, 2), d)
        untouched = np.ones(rows + 50, bool)
        untouched[slots[live]] = False
        assert (got_c[:, untouched] == 0x3C).all()
    assert np.isfinite(decode(kc.cpu().numpy()[:, slots[live]], ks.cpu().numpy().view(np.float16)[:, slots[live]])).all()
