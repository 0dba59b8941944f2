"""One f32 token each of very many sequences over a few states: a sequence's cost does
not grow with how many stand before it."""
import pytest
import torch

from ai_engine_b200 import attention
from tests import _read, _seq

pytestmark = pytest.mark.gpu


def _inputs(seqs, hq, hk, d):
    g = torch.Generator("cuda").manual_seed(seqs)
    lens = torch.randint(0, 4, (seqs,), generator=torch.Generator().manual_seed(seqs)).tolist()
    q, k, v = (torch.randn(n, h, d, generator=g, device="cuda") for n, h in ((seqs, hq), (sum(lens), hk), (sum(lens), hk)))
    return lens, q, k, v


@pytest.mark.parametrize("hq, hk, d", [(2, 1, 16), (70, 1, 32), (130, 2, 24), (4, 4, 128)])
def test_right_for_each(cuda_ok, hq, hk, d):
    lens, q, k, v = _inputs(300, hq, hk, d)
    _seq.check(attention.cross_attention(q, k, v, _read.starts(lens)), *_read.cross(q, k, v, [1] * 300, lens))


def _time(seqs):
    lens, q, k, v = _inputs(seqs, 1, 1, 32)
    cu = _read.starts(lens)
    run = lambda: attention.cross_attention(q, k, v, cu)  # noqa: E731
    run()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    run()
    b.record()
    b.synchronize()
    return a.elapsed_time(b)


def test_cost_of_many_sequences(cuda_ok):
    """32 times as many: less than 200 times the time (the square would be 1024)."""
    assert _time(128000) < 200 * max(_time(4000), 0.02)
