"""The give-up path of the SwiGLU pipeline does not hang on chance: in the build whose data-path waits give up after two
polls, every launch gives up, the smallest too, whose consumers set up their exponential table before they look for the one
tile there is."""
import ctypes as C

import pytest
import torch

from fnfl_v100_b200 import _lib, ops, synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 512), (256, 512), (148 * 8, 512)])
def test_every_launch_of_the_two_poll_build_gives_up(dev, shortwait_lib, rows, cols):
    g = synth.rng(rows)
    gate, up = (torch.from_numpy(synth.normal(g, (rows, cols), 0.5)).to(dev) for _ in range(2))
    err = ops.new_err(dev)
    want = ops.swiglu_q8_1(gate, up, err=err)          # the production build first
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    out = torch.zeros_like(want)
    at = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    for _ in range(10):
        err.zero_()
        assert shortwait_lib.fnb_swiglu_q8_1(at(gate), at(up), at(out), None, rows, cols, at(err),
                                             C.c_void_p(torch.cuda.current_stream().cuda_stream)) == _lib.OK
        torch.cuda.synchronize()                       # returns: nothing is left spinning
        assert int(err.item()) == _lib.ERR_TIMEOUT
    err.zero_()
    assert torch.equal(ops.swiglu_q8_1(gate, up, out=out, err=err), want)
    assert int(err.item()) == 0
