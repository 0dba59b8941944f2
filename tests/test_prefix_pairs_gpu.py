"""One-token attention with more (stream, key head) pairs than blocks run at
once: a block goes through several."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _seq
from tests.test_attention_gpu import _prefix_case, _prefix_want

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

# 0, fewer places than the prefix, as many, and up to several tiles of 64 more
MORE = [0, -3, 1, 130, -1, 64, 700, 63, -60, 65, 0, 200]


@pytest.mark.parametrize("b, hq, hk, d, size, shared, dt", [
    (301, 6, 3, 64, 16, 0, F16), (301, 6, 3, 128, 16, 0, BF16), (301, 6, 3, 64, 16, 100, F16), (301, 6, 3, 128, 8, 100, BF16),
    (301, 6, 3, 64, 24, 300, BF16), (607, 8, 1, 128, 64, 100, F16), (150, 40, 2, 64, 16, 77, F16), (150, 40, 2, 128, 16, 0, F16),
])
def test_more_pairs_than_blocks(cuda_ok, b, hq, hk, d, size, shared, dt):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert b * hk * -(-hq // hk // 16) > 2 * sms
    lens = [0 if i % 29 == 5 else max(shared + MORE[i % len(MORE)], 0) for i in range(b)]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, dt, 3)
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    _seq.check(got, *_prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5))
    for _ in range(3):
        assert torch.equal(got, attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln))
