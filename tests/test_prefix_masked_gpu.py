"""Shared-prefix attention where places carry no weight: scores of -inf, and
values that a stream does not see."""
import math

import pytest
import torch

from ai_engine_b200 import attention
from tests import _seq
from tests.test_attention_gpu import _prefix_case, _prefix_want

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


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("b, hq, hk, d, size, shared, cut", [
    (9, 4, 2, 64, 16, 1000, 650), (9, 8, 2, 128, 24, 1000, 650), (9, 40, 2, 64, 64, 700, 640), (9, 4, 1, 128, 8, 90, 33),
    (9, 4, 2, 64, 12, 200, 150), (301, 6, 3, 64, 16, 300, 200), (301, 3, 3, 128, 16, 130, 100),
])
def test_values_behind_a_short_stream(cuda_ok, dt, bad, b, hq, hk, d, size, shared, cut):
    """Values of the prefix from place `cut` on are not finite.  Streams that
    end there or before do not see them; those that see one are not finite."""
    few = [0, 1, cut, cut - 1, shared, cut // 2, shared + 70, cut + 1, 3]
    lens = [few[i % len(few)] for i in range(b)]
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, lens, dt, 3)
    want, lim = _prefix_want(q, kv, prefix, table, ln, shared, d ** -0.5)
    at = torch.arange(cut, shared, device="cuda")
    kv[1, prefix.long()[at // size], at % size] = bad
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    short = ln <= cut
    _seq.check(got[short], want[short], lim[short])
    assert not torch.isfinite(got[~short]).any()
    assert torch.equal(got[short], attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)[short])
    # bounded lengths: nothing behind the bound is seen either
    got = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln, max_len=cut)
    one = (ln <= cut) | (ln > shared)
    want, lim = _prefix_want(q, kv, prefix, table, ln.clamp(max=cut), shared, d ** -0.5)
    _seq.check(got[one], want[one], lim[one])


def test_values_behind_a_short_stream_in_a_graph(cuda_ok):
    """Which streams are short changes between replays."""
    b, hq, hk, d, size, shared, cut = 40, 8, 2, 128, 16, 520, 300
    q, kv, prefix, table, ln = _prefix_case(b, hq, hk, d, size, shared, [shared + 3 * i for i in range(b)], F16, 5)
    at = torch.arange(cut, shared, device="cuda")
    clean = kv.clone()
    attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = attention.prefix_attention(q, kv[0], kv[1], prefix, shared, table, ln)
    kv[1, prefix.long()[at // size], at % size] = math.nan
    lens = ln.clone()
    for first in (0, 1):
        ln.copy_(torch.where(torch.arange(b, device="cuda") % 2 == first, torch.arange(b, device="cuda") * 7, lens))
        g.replay()
        torch.cuda.synchronize()
        want, lim = _prefix_want(q, clean, prefix, table, ln, shared, d ** -0.5)
        short = ln <= cut
        assert short.sum() == b // 2
        _seq.check(out[short], want[short], lim[short])
        assert torch.isnan(out[~short]).all()
