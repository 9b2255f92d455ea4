"""Many steps of a serving program enqueued one after the other with nothing between them, so that each kernel starts under the
end of those before it: block tables, append and attention of every step read what the step before and this one wrote.
Bit for bit what the same steps give when each kernel is waited for; eagerly, and as one captured graph of several steps."""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth

pytestmark = pytest.mark.gpu

STEPS, CAP = 240, 6


class Server:
    def __init__(self, dev, hd, n_q, n_kv, pages, page=16, n_req=3):
        g = synth.rng(hd + pages)
        self.page, self.n_pages, self.n_req = page, n_req * pages + 5, n_req
        self.q, self.k, self.v = (torch.from_numpy(synth.normal(g, (STEPS, CAP, h, hd))).to(dev) for h in (n_q, n_kv, n_kv))
        new = g.integers(0, 3, (STEPS, n_req))
        new[np.cumsum(new, 0) > pages * page] = 0
        self.new = torch.from_numpy(new.astype(np.int32)).to(dev)
        self.free = torch.from_numpy(g.permutation(self.n_pages).astype(np.int32)).to(dev)
        self.pages, self.dev, self.hd, self.n_kv = pages, dev, hd, n_kv
        self.ts = ops.theta_scale(1e7, 64)
        self.ws = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
        self.reset()

    def reset(self):
        slots = self.n_pages * self.page
        self.kc, self.ks = ops.new_kv_cache(slots, self.n_kv, self.hd, self.dev, fmt="kv4")
        self.vc, self.vs = ops.new_kv_cache(slots, self.n_kv, self.hd, self.dev, fmt="kv4")
        i32 = lambda *n: torch.zeros(n, dtype=torch.int32, device=self.dev)  # noqa: E731
        self.table, self.cells, self.head, self.err = i32(self.n_req, self.pages) - 1, i32(self.n_req), i32(1), i32(1)
        self.slots, self.pos, self.start = i32(CAP), i32(CAP), i32(self.n_req + 1)
        self.q_out, self.out = torch.zeros_like(self.q[0]), torch.full_like(self.q, 9.0)

    def step(self, i, wait=False):
        done = torch.cuda.synchronize if wait else lambda: None
        ops.page_tables(self.table, self.cells, self.new[i], self.free, page_size=self.page, n_pages=self.n_pages, rows=CAP,
                        free_head=self.head, free_head_out=self.head, n_cells=self.cells, slots=self.slots, pos=self.pos,
                        row_start=self.start, err=self.err)
        done()
        ops.rope_neox_kv4_append(self.q[i], self.k[i], self.v[i], self.pos, n_rot=64, theta_scale=self.ts, k_cache=self.kc,
                                 v_cache=self.vc, k_scale=self.ks, v_scale=self.vs, slots=self.slots, q_out=self.q_out, err=self.err)
        done()
        ops.attend_paged_kv4(self.q_out, self.kc, self.vc, self.ks, self.vs, self.table, self.cells, page_size=self.page,
                             row_start=self.start, max_rows=2, out=self.out[i], workspace=self.ws, err=self.err)
        done()

    def state(self):
        torch.cuda.synchronize()
        assert int(self.err.item()) == 0
        return [t.clone() for t in (self.out, self.kc, self.ks, self.vc, self.vs, self.table, self.cells, self.head)]


@pytest.mark.parametrize("hd,n_q,n_kv,pages", [(64, 2, 1, 16), (64, 4, 2, 40), (128, 4, 1, 16), (128, 8, 2, 600), (256, 4, 1, 16),
                                               (256, 16, 2, 40), (256, 16, 2, 600)])
def test_steps_without_a_pause(dev, hd, n_q, n_kv, pages):
    s = Server(dev, hd, n_q, n_kv, pages)
    for i in range(STEPS):
        s.step(i, wait=True)
    want = s.state()
    assert int(want[6].max()) > 150                       # cells a request ends with
    for _ in range(3):
        s.reset()
        for i in range(STEPS):
            s.step(i)
        for got, w in zip(s.state(), want):
            assert torch.equal(got, w)
    # eight steps to a graph: no host between them
    s.reset()
    ops.prepare_device()
    graphs = []
    for first in range(0, STEPS, 8):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for i in range(first, first + 8):
                s.step(i)
        graphs.append(graph)
    torch.cuda.synchronize()
    for graph in graphs:
        graph.replay()
    for got, w in zip(s.state(), want):
        assert torch.equal(got, w)
