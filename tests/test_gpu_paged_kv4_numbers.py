"""Numbers that the paged KV4 operators have to refuse instead of taking their low 32 bits or failing in an allocation."""
import pytest
import torch

from fnfl_v100_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", [dict(page_size=2**32 + 16), dict(n_pages=2**32 + 8), dict(page_size=-2**32 + 16), dict(rows=0), dict(rows=-1),
                                    dict(rows=2**32 + 4), dict(n_pages=2**31)])
def test_page_tables(dev, change):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.full((2, 4), -1, dtype=torch.int32, device=dev)
    kw = dict(page_size=16, n_pages=8, rows=4)
    outs = dict(slots=i32(9, 9, 9, 9), pos=i32(9, 9, 9, 9), row_start=i32(9, 9, 9), n_cells=i32(9, 9))
    given = outs if change.get("rows", 4) == 4 else {}
    with pytest.raises(ValueError):
        ops.page_tables(table, i32(0, 0), i32(1, 1), i32(0, 1, 2, 3), **{**kw, **change}, **given)
    torch.cuda.synchronize()
    assert all(bool((t == 9).all()) for t in outs.values()) and bool((table == -1).all())
    t = ops.page_tables(table, i32(0, 0), i32(1, 1), i32(0, 1, 2, 3), **kw)
    assert t.slots.tolist() == [0, 16, -1, -1]


@pytest.mark.parametrize("change", [dict(page_size=2**32 + 16), dict(max_rows=2**32), dict(max_rows=2**31), dict(max_rows=-1)])
def test_attend(dev, change):
    (kc, ks), (vc, vs) = (ops.new_kv_cache(64, 1, 64, dev, fmt="kv4") for _ in range(2))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q, out = torch.ones((1, 1, 64), device=dev), torch.full((1, 1, 64), 9.0, device=dev)
    args = (q, kc, vc, ks, vs, i32(0).view(1, 1), i32(5))
    with pytest.raises(ValueError):
        ops.attend_paged_kv4(*args, out=out, **{**dict(page_size=16, max_rows=1), **change})
    torch.cuda.synchronize()
    assert bool((out == 9.0).all())
    assert not bool(ops.attend_paged_kv4(*args, out=out, page_size=16).any())


@pytest.mark.parametrize("kw", [dict(cell0=65), dict(cell0=64), dict(rows=0), dict(rows=-3), dict(rows=2**40), dict(rows=65), dict(cell0=-1), dict(cells=torch.zeros(0, dtype=torch.int32))])
def test_read(dev, kw):
    codes, scale = ops.new_kv_cache(64, 2, 128, dev, fmt="kv4")
    assert ops.kv4_read_f32(codes, scale, cell0=63).shape == (1, 2, 128)
    with pytest.raises(ValueError):
        ops.kv4_read_f32(codes, scale, **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})


def test_append(dev):
    (kc, ks), (vc, vs) = (ops.new_kv_cache(8, 1, 128, dev, fmt="kv4") for _ in range(2))
    q = torch.ones((2, 1, 128), device=dev)
    pos = torch.arange(2, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.rope_neox_kv4_append(q, q, q, pos, n_rot=2**32 + 64, theta_scale=0.5, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert not bool(ks.any()) and not bool(vs.any())
