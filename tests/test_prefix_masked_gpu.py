"""Shared-prefix attention where places carry no weight."""
import math

import pytest
import torch

from ai_engine_b200 import attention
from tests import _seq
from tests.test_attention_gpu import _prefix_case

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _places(kv, prefix, table, i, n, shared):
    """Keys and values of stream i's first n places."""
    size = kv.shape[2]
    j = torch.arange(n, device="cuda")
    row = table[i].long()
    page = torch.where(j < shared, prefix.long()[(j // size).clamp(max=prefix.numel() - 1)], row[j // size])
    return kv[0][page, j % size], kv[1][page, j % size]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d, size", [(64, 16), (128, 64)])
@pytest.mark.parametrize("lo, hi, own", [(128, 256, False), (0, 1200, False), (256, 640, True), (1100, 1200, True), (0, 1200, True)])
def test_scores_of_minus_infinity(cuda_ok, dt, d, size, lo, hi, own):
    """Keys lo .. hi - 1 of the prefix, whole pieces of it among them, and all
    of one stream's own, have scores of -inf: no weight.  A stream of such
    scores alone is NaN, as the formula says."""
    b, hq, hk, shared = 3, 4, 2, 1200
    lens = [1200, 1277, 1300]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, dt, 3)
    q[..., 0] = 1
    at = torch.arange(lo, hi, device="cuda")
    kv[0, prefix.long()[at // size], at % size, :, 0] = -math.inf
    if own:
        at = torch.arange(shared, lens[1], device="cuda")
        kv[0, table[1].long()[at // size], at % size, :, 0] = -math.inf
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    for i, n in enumerate(lens):
        k, v = _places(kv, prefix, table, i, n, shared)
        keep = torch.isfinite(k[:, 0, 0])
        if not keep.any():
            assert torch.isnan(got[i]).all()
            continue
        k, v = k[keep], v[keep]
        for h in range(hq):
            # -inf adds nothing: the softmax over the other keys
            want, lim = _seq.attend(q[i, h:h + 1], k[:, h // 2], v[:, h // 2], torch.tensor([len(k)], device="cuda"), d ** -0.5, dt)
            _seq.check(got[i, h:h + 1], want, lim)
