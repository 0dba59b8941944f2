"""Scratch of the one-token attention, by the C ABI without a GPU: a warp leaves two
partial results at most, so it does not grow with the streams by more than their list."""
import pytest

from ai_engine_b200 import _lib
from ai_engine_b200.build import build
from tests.test_read_abi import cross_args, step


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


@pytest.mark.parametrize("d, hq, hk", [(128, 32, 8), (64, 8, 8), (256, 16, 2)])
def test_workspace_of_many_streams(lib, d, hq, hk):
    cache = (1 << 20, 1 << 20, hk * 16 * d * 5 // 8, 8, 16, hk, d)
    few, many = (lib.aie_kv4_attn_workspace(step(cache=cache, batch=n, hq=hq)) for n in (1, 65535))
    assert 0 < few <= many < few + 65535 * 4 + 128
    few, many = (lib.aie_cross_attn_workspace(cross_args(cu_q=0, tokens=n, seqs=n, hq=hq, hk=hk, d=d, keys=1 << 20)) for n in (1, 1 << 20))
    assert 0 < few <= many < few + 4 * (1 << 20) + 128
