"""The example decoder at the ends of what its cache holds."""
import pytest
import torch

from ai_engine_b200.decoder import StreamDecoder
from tests.test_decoder_gpu import Plain, _near

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


def test_second_prompt_is_refused(cuda_ok):
    m = _decoder(100)
    m.fork([1])  # of nothing
    m.prompt(_feats(20, 1))
    m.fork([2])
    for ended in ([], [0], [1]):
        if ended:
            m.end(ended)
        before = m.state.lens.tolist()
        with pytest.raises(ValueError):
            m.prompt(_feats(5, 2))
        assert m.state.lens.tolist() == before
    m.end([2])
    m.step([1], _feats(1, 4))  # a stream behind nothing
    with pytest.raises(ValueError):
        m.prompt(_feats(5, 2))
    m.end([1])
    y = m.prompt(_feats(30, 3))
    assert torch.equal(y, _decoder(100).prompt(_feats(30, 3)))
    assert m.state.lens.tolist() == [30, 0, 0] and m.status() == 0


def test_streams_outlive_the_prompt_row(cuda_ok):
    """The prompt's row ends while streams behind it go on."""
    m = _decoder(100)
    p = Plain(m)
    _near(m.prompt(_feats(37, 1)), p.run(0, _feats(37, 1).double(), 0), 2)
    m.fork([1, 2])
    for r in (1, 2):
        p.rows[r] = list(p.rows[0])
    for i in range(6):
        if i == 2:
            m.end([0])
        x = _feats(2, 10 + i)
        want = torch.cat([p.run(r, x[r - 1:r].double(), 37 + i) for r in (1, 2)])
        _near(m.step([1, 2], x), want, 2)
    assert m.status() == 0 and m.state.lens.tolist() == [0, 43, 43]
