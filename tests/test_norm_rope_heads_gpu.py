"""Norm and rotation of so many heads that a lane takes four of a token."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _seq
from tests.test_attention_gpu import _rand, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens, hq, hk, d, rot, interleaved", [
    (2000, 9, 3, 64, 64, False), (2001, 10, 2, 64, 32, True), (1300, 25, 5, 96, 48, True), (700, 32, 8, 128, 128, False),
    (1301, 15, 5, 128, 64, False), (300, 6, 3, 256, 256, False), (301, 7, 7, 512, 256, True), (900, 18, 6, 80, 0, False),
])
@pytest.mark.parametrize("cached", [True, False])
def test_four_heads_a_lane(cuda_ok, dt, tokens, hq, hk, d, rot, interleaved, cached):
    lanes = 4 if d <= 64 else 8 if d <= 128 else 32
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert tokens * (hq + 2 * hk) * lanes > 128 * 5 * sms  # as many threads as run at once
    x = _rand((tokens, hq + 2 * hk, d), dt, 5, 2.0)
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    wq, wk = _rand((d,), torch.float32, 3), _rand((d,), torch.float32, 4)
    table = _table(500, rot) if rot else torch.zeros(500, 0, device="cuda")
    pos = torch.randint(0, 500, (tokens,), device="cuda", dtype=torch.int32)
    want_q = _seq.norm_rope(q, wq, pos, table, rot, interleaved, 1e-6)
    want_k = _seq.norm_rope(k, wk, pos, table, rot, interleaved, 1e-6)
    opts = dict(q_weight=wq, k_weight=wk, interleaved=interleaved)
    if not cached:
        qo, ko = attention.qk_norm_rope(q, k, pos, table, **opts)
        _seq.check_norm_rope(qo, *want_q)
        _seq.check_norm_rope(ko, *want_k)
        return
    size = 16
    n = -(-tokens // size) + 2
    pages = torch.zeros(2, n, size, hk, d, dtype=dt, device="cuda")
    slots = torch.randperm(n * size, device="cuda")[:tokens]
    slots[3], slots[tokens - 2] = -1, n * size
    keep = (slots >= 0) & (slots < n * size)
    at = slots[keep]
    v0 = v.clone()
    # in place
    qo, ko = attention.qk_norm_rope(q, k, pos, table, v=v, k_pages=pages[0], v_pages=pages[1], slots=slots, q_out=q, k_out=k, **opts)
    _seq.check_norm_rope(qo, *want_q)
    _seq.check_norm_rope(ko, *want_k)
    assert torch.equal(v, v0)
    rest = torch.zeros_like(pages)
    rest[0].view(-1, hk, d)[at], rest[1].view(-1, hk, d)[at] = ko[keep], v[keep]
    assert torch.equal(pages, rest)
