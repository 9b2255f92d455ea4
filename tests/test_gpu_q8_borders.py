"""8-bit codes of values on the border between two codes and a few ulps to either side, against the CPU definition: there a
product x id that is not rounded before the rounding of the code would show."""
import numpy as np
import pytest
import torch

from fnfl_v100_b200 import ops, synth

pytestmark = pytest.mark.gpu


def borders(seed, blocks):
    """Blocks of 32 values: the first is the block's largest, the others lie within three ulps of (k + 1/2) d."""
    g = synth.rng(seed)
    amax = np.exp2(g.uniform(-100, 100, blocks)).astype(np.float32)
    d = (amax / np.float32(127)).astype(np.float32)
    x = ((g.integers(0, 127, (blocks, 32)) + 0.5) * d[:, None]).astype(np.float32)
    x = (x.view(np.int32) + g.integers(-3, 4, x.shape).astype(np.int32)).view(np.float32)
    x = np.minimum(x, amax[:, None]) * g.choice(np.array([-1, 1], np.float32), x.shape)
    x[:, 0] = amax
    return np.ascontiguousarray(x, np.float32)


@pytest.mark.parametrize("seed", [1, 2])
def test_quantisers(dev, oracle, seed):
    x = borders(seed, 1 << 16).reshape(-1, 2048)
    dx = torch.from_numpy(x).to(dev)
    assert np.array_equal(ops.quantize_q8_0(dx).cpu().numpy().reshape(-1), oracle.quantize_q8_0(x))
    assert np.array_equal(ops.quantize_q8_1(dx).cpu().numpy().reshape(-1), oracle.quantize_q8_1(x))
    codes, scales = ops.act_quantize(dx)
    want = oracle.act_quantize(x)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


@pytest.mark.parametrize("hd,n_rot", [(256, 64), (128, 64), (64, 64), (256, 32)])
def test_cells(dev, oracle, hd, n_rot):
    """V passes through the append's quantiser alone; n_rot 32 takes the row-per-warp kernel."""
    v = borders(hd, 1 << 13).reshape(-1, 2, hd)
    rows = v.shape[0]
    kc, vc = (ops.new_kv_cache(rows, 2, hd, dev) for _ in range(2))
    zero = torch.zeros((rows, 2, hd), device=dev)
    ops.rope_neox_q8_0_append(zero, zero, torch.from_numpy(v).to(dev), torch.arange(rows, dtype=torch.int32, device=dev), n_rot=n_rot,
                              theta_scale=0.5, k_cache=kc, v_cache=vc)
    assert np.array_equal(vc.cpu().numpy().reshape(-1), oracle.quantize_q8_0(v))
