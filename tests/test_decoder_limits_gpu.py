"""The example decoder at the ends of what its cache holds."""
import pytest
import torch

from ai_engine_b200.decoder import StreamDecoder

pytestmark = pytest.mark.gpu


def _decoder(max_len):
    return StreamDecoder(2, 64, 2, 1, 64, streams=2, pages_=20, max_len=max_len, dtype=torch.float16)


def _feats(n, seed):
    return torch.randn(n, 64, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").half()


def test_length_that_ends_inside_a_page(cuda_ok):
    """Every token that the cache accepts is attended, as in a longer cache."""
    short, wide = _decoder(40), _decoder(200)
    for m in (short, wide):
        m.prompt(_feats(38, 1))
        m.fork([1, 2])
    for i in range(10):  # tokens 38 .. 47: the row's third page is full then
        x = _feats(2, 10 + i)
        a, b = short.step([1, 2], x), wide.step([1, 2], x)
        assert short.status() == 0 and torch.equal(a, b), i
    short.step([1, 2], x)
    assert short.status() == 1 and short.state.lens.tolist() == [38, 48, 48]
