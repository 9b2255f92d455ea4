"""The norm + RoPE + append pipeline with every arrangement of its producers, over tiles enough to turn its ring over.

Producers work in crews of one or two warps, and one, two or four crews take tiles in turn; which it is follows from the
heads and the number of rows.  Two things are held for each arrangement and cell format: a long launch writes, bit for bit, what
the same tokens give in short launches (one tile a CTA: no stage is used twice); and the give-up path of the bounded waits
(a build whose data-path waits give up after two polls) ends by itself with FNB_ERR_TIMEOUT, leaves no copy in flight, and
the next launch of the production library is right."""
import ctypes as C

import numpy as np
import pytest
import torch

from fnfl_v100_b200 import _lib, ops, synth

pytestmark = pytest.mark.gpu

SHAPES = [
    # query heads, KV heads, head_dim, n_rot, rows
    (24, 8, 64, 64, 148 * 20 + 7),       # four crews of one, tiles of one token
    (8, 4, 128, 64, 148 * 5 * 9 + 3),    # two crews of two, tiles of five tokens
    (2, 1, 64, 0, 148 * 8 * 9 + 5),      # two crews of two, tiles of eight, no angles
    (16, 8, 256, 64, 148 * 9 + 1),       # two crews of one
    (32, 4, 256, 64, 148 * 14 + 1),      # one crew of one
    (16, 2, 256, 64, 148 * 2 * 9 + 1),   # one crew of two
]
FORMATS = ["q8_0", "kv8", "kv4"]


class Step:
    """One append's tensors, and the call through either library."""

    def __init__(self, dev, n_q, n_kv, hd, n_rot, rows, fmt):
        g = synth.rng(n_q * 31 + hd)
        self.fmt, self.n_rot, self.rows, self.slots_n = fmt, n_rot, rows, rows + 9
        self.ts = ops.theta_scale(1e7, n_rot) if n_rot else 1.0
        self.q, self.k, self.v = (torch.from_numpy(synth.normal(g, (rows, n, hd))).to(dev) for n in (n_q, n_kv, n_kv))
        self.w = [torch.from_numpy(1 + 0.1 * synth.normal(g, (hd,))).to(dev) for _ in range(2)]
        self.pos = torch.from_numpy((np.arange(rows) + 1000).astype(np.int32)).to(dev)
        self.slots = torch.from_numpy(g.permutation(self.slots_n)[:rows].astype(np.int32)).to(dev)
        self.err = ops.new_err(dev)
        self.clear()

    def clear(self):
        dev, (rows, n_kv, hd) = self.q.device, self.k.shape
        made = [ops.new_kv_cache(self.slots_n, n_kv, hd, dev, fmt=self.fmt) for _ in range(2)]
        self.k_cache, self.k_scale = made[0] if self.fmt != "q8_0" else (made[0], None)
        self.v_cache, self.v_scale = made[1] if self.fmt != "q8_0" else (made[1], None)
        self.q_out, self.k_f32 = torch.zeros_like(self.q), torch.zeros_like(self.k)

    def written(self):
        return [t.clone() for t in (self.q_out, self.k_f32, self.k_cache, self.v_cache, self.k_scale, self.v_scale) if t is not None]

    def run(self, first=0, end=None):
        end = self.rows if end is None else end
        part = slice(first, end)
        kw = dict(n_rot=self.n_rot, theta_scale=self.ts, k_cache=self.k_cache, v_cache=self.v_cache, slots=self.slots[part],
                  q_norm_w=self.w[0], k_norm_w=self.w[1], q_out=self.q_out[part], k_f32=self.k_f32[part], err=self.err)
        if self.fmt != "q8_0":
            kw.update(k_scale=self.k_scale, v_scale=self.v_scale)
        op = {"q8_0": ops.rope_neox_q8_0_append, "kv8": ops.rope_neox_kv8_append, "kv4": ops.rope_neox_kv4_append}[self.fmt]
        op(self.q[part], self.k[part], self.v[part], self.pos[part], **kw)

    def launch(self, lib):
        at = lambda t: t.data_ptr()  # noqa: E731
        a = _lib.RopeKvArgs(at(self.q), at(self.k), at(self.v), at(self.pos), at(self.slots), at(self.w[0]), at(self.w[1]), at(self.q_out),
                            at(self.k_cache), at(self.v_cache), at(self.k_f32), at(self.err), self.rows, self.slots_n, self.q.shape[1],
                            self.k.shape[1], self.q.shape[2], self.n_rot, self.ts, 1e-6, None)
        if self.fmt != "q8_0":
            a = _lib.RopeKv8Args(a, at(self.k_scale), at(self.v_scale))
        name = "fnb_rope_neox_%s_append" % self.fmt
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
        return fn(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv,hd,n_rot,rows", SHAPES)
def test_long_launch_equals_short_ones(dev, n_q, n_kv, hd, n_rot, rows, fmt):
    s = Step(dev, n_q, n_kv, hd, n_rot, rows, fmt)
    for first in range(0, rows, 148):
        s.run(first, min(rows, first + 148))
    want = s.written()
    for _ in range(3):
        s.clear()
        s.run()
        torch.cuda.synchronize()
        assert int(s.err.item()) == 0
        for got, w in zip(s.written(), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n_q,n_kv,hd,n_rot,rows", SHAPES)
def test_waits_give_up_and_the_next_launch_is_right(dev, shortwait_lib, n_q, n_kv, hd, n_rot, rows, fmt):
    s = Step(dev, n_q, n_kv, hd, n_rot, rows, fmt)
    s.run()                                    # the production build first
    torch.cuda.synchronize()
    assert int(s.err.item()) == 0
    want = s.written()
    assert s.launch(shortwait_lib) == _lib.OK
    torch.cuda.synchronize()                   # returns: nothing is left spinning
    assert int(s.err.item()) & _lib.ERR_TIMEOUT
    s.err.zero_()
    s.clear()
    s.run()
    torch.cuda.synchronize()
    assert int(s.err.item()) == 0
    for got, w in zip(s.written(), want):
        assert torch.equal(got, w)
