"""That the bound which 4-bit attention is held to tells a lost or a doubled tile
of 32 places, without a GPU."""
import pytest
import torch

from tests import _kv4, _read


@pytest.mark.parametrize("n, tile", [(20000, 0), (20000, 312), (20000, 624), (700, 3)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [0.0, 0.3])
def test_a_lost_or_doubled_tile_breaks_the_bound(n, tile, dt, size):
    g = torch.Generator().manual_seed(n)
    q = (size * torch.randn(1, 4, 128, generator=g)).to(dt)
    k = torch.randn(n, 1, 128, generator=g)
    v = _kv4.markers([n], 1, 128)
    kp, vp, table = _kv4.streams(k, v, [n], 16, device="cpu")
    want, limit = _kv4.attend(q, kp, vp, table, [n])
    x = _read.values(k)[:, 0]
    w = torch.softmax(128 ** -0.5 * q[0].double() @ x.T, -1)
    part = w[:, tile * 32:tile * 32 + 32]
    part = part.sum(-1, keepdim=True) * _read.values(v)[tile * 32, 0]
    for wrong in (want[0] - part, want[0] + part):
        assert bool(((wrong - want[0]).abs() > limit[0]).any(-1).all())


def test_layout_of_the_helper():
    """What the helper lays out is read back as what was put in."""
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(37, 2, 64, generator=g), torch.randn(37, 2, 64, generator=g)
    kp, vp, table = _kv4.streams(k, v, [21, 0, 16], 8, gap=2, device="cpu")
    assert kp.shape == (7, 2, 8, 40) and table.shape == (3, 3)
    got = _read.read_cache(kp, 64)[table[0].long()].transpose(1, 2).reshape(24, 2, 64)[:21]
    assert torch.equal(got, _read.values(k[:21]))
    got = _read.read_cache(vp, 64)[table[2, :2].long()].transpose(1, 2).reshape(16, 2, 64)
    assert torch.equal(got, _read.values(v[21:]))
