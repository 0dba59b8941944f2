"""One-token attention over a 4-bit cache where values are large, small or of
very unequal size, against a bound in which each place counts by its weight; and
that every tile of a stream counts once, whichever warps take it."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _kv4, _seq

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _rand(shape, seed, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return scale * torch.randn(shape, generator=g, device="cuda")


def _check(q, k, v, lens, size=16, scale=None):
    kp, vp, table = _kv4.streams(k, v, lens, size)
    got = attention.kv4_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=scale)
    _seq.check(got, *_kv4.attend(q, kp, vp, table, lens, scale))


HEADS = [(8, 2, 128), (16, 1, 64), (5, 1, 96), (3, 3, 32), (4, 2, 256), (9, 1, 160)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk, d", HEADS)
@pytest.mark.parametrize("lens", [[20000], [700, 0, 33, 1, 32], [(i * 131) % 400 for i in range(70)]])
def test_every_tile_counts_once(cuda_ok, dt, hq, hk, d, lens):
    for size in (0.0, 0.3):
        k = _rand((sum(lens), hk, d), 1)
        v = _kv4.markers(lens, hk, d).to("cuda").contiguous()
        _check(_rand((len(lens), hq, d), 2, size).to(dt), k, v, lens)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk, d", HEADS)
@pytest.mark.parametrize("scale", [1e-4, 1e-3, 1.0, 20.0, 1e3, 1.2e4])
def test_sizes_of_values(cuda_ok, dt, hq, hk, d, scale):
    lens = [3000, 7, 200, 0, 61]
    _check(_rand((len(lens), hq, d), 1, 2.0).to(dt), _rand((sum(lens), hk, d), 2), _rand((sum(lens), hk, d), 3, scale), lens)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk, d", [(8, 2, 128), (16, 1, 64), (2, 1, 224)])
@pytest.mark.parametrize("wide", [50.0, 3000.0, 60000.0])
@pytest.mark.parametrize("at", [0, 15, 33, 1500, 20000, 39999])
def test_one_wide_group(cuda_ok, dt, hq, hk, d, wide, at):
    """One element far outside the others: in the first, a middle and the last
    tile, of a part of its own or not; only its own stream and group may lose by it."""
    lens = [40000, 100, 31]
    k, v = _rand((sum(lens), hk, d), 1), _rand((sum(lens), hk, d), 2)
    v[at, :, 40] = wide
    _check(_rand((len(lens), hq, d), 3).to(dt), k, v, lens)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq", [1, 8, 16])
@pytest.mark.parametrize("orders", [-60.0, -20.0, 0.0])
@pytest.mark.parametrize("at", [5, 9000, 16380])
def test_wide_groups_of_little_weight(cuda_ok, dt, hq, orders, at):
    """A place with an element of 60000 whose weight is 2^orders of the others', and
    a key 10 binary orders above them: the others' small weights still count."""
    n, d = 16384, 128
    k, v = 0.02 * _rand((n, 1, d), 1), _rand((n, 1, d), 2)
    q = torch.zeros(1, hq, d, device="cuda")
    q[:, :, :32] = 1.0  # a group of its own, so that its steps do not coarsen the others
    k[at, :, :32] = orders * 0.6931 * d ** 0.5 / 32
    k[n // 3, :, :32] = 10 * 0.6931 * d ** 0.5 / 32
    v[at, :, 3] = 60000.0
    _check(q.to(dt), k, v, [n])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk, d", [(8, 2, 128), (12, 1, 64)])
def test_wide_groups_come_and_go(cuda_ok, dt, hq, hk, d):
    """Many short streams to a warp, wide values in some of them, by turns with narrow
    ones, and scores that grow along a stream, so that what was wide loses its weight."""
    lens = [(i * 53) % 300 for i in range(900)]
    k, v = _rand((sum(lens), hk, d), 1), _rand((sum(lens), hk, d), 2)
    at = torch.arange(sum(lens), device="cuda")
    v *= torch.where(at % 700 < 350, 1.0, torch.where(at % 3 == 0, 900.0, 0.002))[:, None, None]
    _check(_rand((len(lens), hq, d), 3).to(dt), k, v, lens)
    n = 5000
    k, v = _rand((n, hk, d), 4, 0.1), _rand((n, hk, d), 5)
    k[..., 0] = torch.linspace(-3, 3, n, device="cuda")[:, None]
    v[:2000:7] *= 5000.0
    q = _rand((1, hq, d), 6)
    q[..., 0] = 30.0
    _check(q.to(dt), k, v, [n])


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk", [(8, 8), (72, 8)])
def test_wide_groups_in_long_parts(cuda_ok, dt, hq, hk):
    """The same where a warp has many tiles one after the other (more than 30): an
    element of 60000 at weight 2^-60 ahead of a key 14.1 binary orders above the
    others, whose own value is 0, so that the result is what the others' weights leave."""
    n, b, d = 4096, 64, 64
    k, v = 0.02 * _rand((b * n, hk, d), 1), 2.0 + _rand((b * n, hk, d), 2)
    q = torch.zeros(b, hq, d, device="cuda")
    q[:, :, :32] = 1.0
    at = torch.arange(b * n, device="cuda")
    k[at % 1024 == 3, :, :32] = -60 * 0.6931 * d ** 0.5 / 32
    k[at % 512 == 9, :, :32] = 14.1 * 0.6931 * d ** 0.5 / 32
    v[at % 1024 == 3, :, 3] = 60000.0
    v[at % 512 == 9] = 0.0
    _check(q.to(dt), k, v, [n] * b)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hq, hk, d", [(1, 1, 64), (8, 2, 128), (9, 1, 96), (2, 1, 256)])
@pytest.mark.parametrize("b, n", [(1, 5000), (150, 3000)])
def test_sizes_change_from_tile_to_tile(cuda_ok, dt, hq, hk, d, b, n):
    """Tiny, ordinary and huge values in turn, tile by tile, where a warp has one tile and
    where it has many; tiles without any range among them."""
    lens = [n - 7 * i % 400 for i in range(b)]
    at = torch.arange(sum(lens), device="cuda")
    sizes = torch.tensor([1e-3, 1.0, 2000.0, 1e-3, 1e4, 0.0, 1e-3, 30.0], device="cuda")
    k, v = _rand((len(at), hk, d), 1), _rand((len(at), hk, d), 2) * sizes[at // 40 % 8][:, None, None]
    _check(_rand((b, hq, d), 3).to(dt), k, v, lens)
