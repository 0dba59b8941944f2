"""Tokens over states and one token over the 4-bit cache where scores are far larger
than a norm leaves: as long as they are finite in f32, the largest one's value results."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _kv4, _read, _seq

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _keys(n, d, seed):
    """Keys of one value each, 2% or more apart, in random order; which is the largest and which the least."""
    size = 1.02 ** -torch.arange(n, dtype=torch.float64, device="cuda")
    size[1::2] *= -1
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).cuda()
    k = size[order, None, None].expand(n, 1, d).contiguous()
    return k, int(k[:, 0, 0].argmax()), int(k[:, 0, 0].argmin())


SIZES = [1e5, 1e8, 3e9, 1e12, 1e20, 1e30, 4e34, 2e36]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("n", [5, 130, 300])
@pytest.mark.parametrize("hq", [2, 10])
def test_one_hot_over_4_bits(cuda_ok, size, n, hq):
    d = 64
    k, top, least = _keys(n, d, n)
    v = torch.randn(n, 1, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    q = torch.full((1, hq, d), size, device="cuda", dtype=BF16)
    q[:, 1::2] *= -1
    kp, vp, table = _kv4.streams(k, v, [n], 8)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    x = _read.values(v)[:, 0]
    got = attention.kv4_attention(q, kp, vp, table, lens)[0]
    for h in range(hq):
        want = x[least if h % 2 else top]
        _seq.check(got[h], want, _seq.UNIT[BF16] * want.abs() + 2.0 ** -9 * (x - x.min()).abs().max() * torch.ones_like(want))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", [F16, BF16])
def test_keys_of_zero(cuda_ok, size, dt):
    """Scores of zero, whatever the queries are: the values' mean."""
    n, d = 300, 64
    if dt == F16:
        size = min(size, 65504.0)
    k, v = torch.zeros(n, 2, d, device="cuda"), torch.randn(n, 2, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    q = torch.full((1, 4, d), size, device="cuda", dtype=dt)
    kp, vp, table = _kv4.streams(k, v, [n], 8)
    got = attention.kv4_attention(q, kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    _seq.check(got, *_kv4.attend(torch.zeros_like(q), kp, vp, table, [n]))
    k, v = k.to(dt), v.to(dt)
    got = attention.cross_attention(q, k, v, _read.starts([n]))
    _seq.check(got, *_read.cross(torch.zeros_like(q), k, v, [1], [n]))


@pytest.mark.parametrize("dt, size", [(F16, 1e3), (F16, 65504.0), (BF16, 1e5), (BF16, 1e8), (BF16, 3e9), (BF16, 1e12), (BF16, 1e20), (BF16, 1e30),
                                      (BF16, 2e36)])
@pytest.mark.parametrize("n", [5, 130, 300, 20000])
@pytest.mark.parametrize("hq, d", [(2, 64), (10, 128), (2, 200)])
def test_one_hot_over_states(cuda_ok, dt, size, n, hq, d):
    k, top, least = _keys(min(n, 300), d, n)
    k = torch.cat([k, torch.zeros(n - k.shape[0], 1, d, device="cuda", dtype=k.dtype)])
    k = (k * (60000.0 if dt == F16 else 1.0)).to(dt)  # finite scores in f32, 2% apart
    v = torch.randn(n, 1, d, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(dt)
    q = torch.full((1, hq, d), size, device="cuda", dtype=dt)
    q[:, 1::2] *= -1
    got = attention.cross_attention(q, k, v, _read.starts([n]))[0]
    if size * d >= 2.0 ** 128:  # 200 products of 2e36 are 4e38: infinite in f32, and inf - inf no number
        assert bool(torch.isnan(got).all())
        return
    for h in range(hq):
        assert torch.equal(got[h], v[least if h % 2 else top, 0])


@pytest.mark.parametrize("dt, size", [(F16, 1.0), (F16, 1e3), (F16, 65504.0), (BF16, 1e5), (BF16, 1e8), (BF16, 3e9), (BF16, 1e20), (BF16, 1e30),
                                      (F32, 1e9), (F32, 1e30)])
@pytest.mark.parametrize("n", [5, 300, 20000])
@pytest.mark.parametrize("rows", [1, 3, 70, 300])
@pytest.mark.parametrize("hq, d", [(2, 64), (8, 128), (2, 200)])
def test_one_hot_of_packed_tokens(cuda_ok, dt, size, n, rows, hq, d):
    """Beside them tokens of another sequence, whose scores are ordinary."""
    k, top, least = _keys(min(n, 300), d, n)
    k = torch.cat([k, torch.zeros(n - k.shape[0], 1, d, device="cuda", dtype=k.dtype)])
    k = (k * (60000.0 if dt == F16 else 1.0)).to(dt)
    g = torch.Generator("cuda").manual_seed(1)
    v = torch.randn(n, 1, d, generator=g, device="cuda").to(dt)
    q = torch.full((rows, hq, d), size, device="cuda", dtype=dt)
    q[:, 1::2] *= -1
    q1, k1, v1 = (torch.randn(m, h, d, generator=g, device="cuda").to(dt) for m, h in ((9, hq), (50, 1), (50, 1)))
    got = attention.cross_attention(torch.cat([q, q1]), torch.cat([k, k1]), torch.cat([v, v1]), _read.starts([n, 50]),
                                    cu_q=_read.starts([rows, 9]))
    want = v[[least if h % 2 else top for h in range(hq)], 0]
    assert torch.equal(got[:rows], want.expand(rows, -1, -1))
    _seq.check(got[rows:], *_read.cross(q1, k1, v1, [9], [50]))
