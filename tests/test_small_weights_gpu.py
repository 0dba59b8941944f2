"""Contexts in which one key outweighs many small equal ones that add up: the
weights' rounding to 16 bits must not lose them."""
import math

import pytest
import torch

from ai_engine_b200 import attention
from tests import _seq

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _heads(n, d, dt, first, orders):
    """One query direction, n keys of which number `first` has a score (scale 1)
    `orders` binary orders above the others'; values 0 for it, about 1 for those."""
    top = math.sqrt(orders * math.log(2))
    q, k = torch.zeros(1, 1, d, dtype=dt, device="cuda"), torch.zeros(n, 1, d, dtype=dt, device="cuda")
    q[0, 0, 0] = top
    k[first, 0, 0] = top
    g = torch.Generator("cuda").manual_seed(n)
    v = (1 + 0.25 * torch.rand(n, 1, d, generator=g, device="cuda")).to(dt)
    v[first] = 0
    return q, k, v


def _check(got, q, k, v, n):
    """_seq.attend's bound, the weights' rounding tighter: f16 weights are held
    2^7 times as large as the row's largest makes them, so that half the
    spacing of their subnormals, 2^-25, is 2^-32 of it, once a key."""
    dt = q.dtype
    want, lim = _seq.attend(q[:, 0], k[:, 0], v[:, 0], torch.tensor([n], device="cuda"), 1.0, dt)
    low = _seq.TINY[dt] * n * float(v.double().abs().max())
    _seq.check(got.view(1, -1), want, lim - low + low * 2.0 ** -7)


ORDERS = [(F16, 22.6), (F16, 24.3), (F16, 25.5), (F16, 16.0), (BF16, 24.3)]


@pytest.mark.parametrize("dt, orders", ORDERS)
@pytest.mark.parametrize("first", [5, 20000])
def test_prompt(cuda_ok, dt, orders, first):
    n, d = 32768, 64
    q, k, v = _heads(n, d, dt, first, orders)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = attention.prompt_attention(q.expand(n, 1, d).contiguous(), k, v, cu, scale=1.0)
    _check(got[n - 1], q, k, v, n)


@pytest.mark.parametrize("dt, orders", ORDERS)
@pytest.mark.parametrize("shared, n, first", [(0, 32768, 7), (0, 32768, 30000), (32768, 32768, 7), (30000, 40000, 35000),
                                              (8000, 40000, 7), (20000, 40001, 12345)])
def test_prefix(cuda_ok, dt, orders, shared, n, first):
    """All keys the stream's own, all in the prefix, or some in either, the
    outstanding one in either."""
    d, size = 128, 64
    q, k, v = _heads(n, d, dt, first, orders)
    pages = -(-n // size)
    kv = torch.zeros(2, pages, size, 1, d, dtype=dt, device="cuda")
    kv[0].view(-1, 1, d)[:n], kv[1].view(-1, 1, d)[:n] = k, v
    row = torch.arange(pages, dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = attention.prefix_attention(q, kv[0], kv[1], row, shared, row[None], lens, scale=1.0)
    _check(got, q, k, v, n)
