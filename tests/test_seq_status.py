"""Waits that give up in the sequence operators' kernels, beside the conv path's."""
import ctypes as C

import pytest

from ai_engine_b200 import _lib
from ai_engine_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def test_selftest_rejects_bad_timeout(lib):
    assert lib.aie_seq_selftest_wait_timeout(0, None) == -2
    assert lib.aie_seq_selftest_wait_timeout(10_000_000, None) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("seq_first", [True, False])
def test_both_codes_are_reported(lib, cuda_ok, seq_first):
    """Both words set: one call reports one code, the next the other, a third none."""
    import torch
    stream, code = C.c_void_p(torch.cuda.current_stream().cuda_stream), C.c_uint32(0)
    assert lib.aie_device_status(stream, C.byref(code)) == 0
    tests = [lib.aie_selftest_wait_timeout, lib.aie_seq_selftest_wait_timeout]
    for test in reversed(tests) if seq_first else tests:
        assert test(20_000, stream) == 0  # 20 ms limit
    got = []
    for _ in range(2):
        assert lib.aie_device_status(stream, C.byref(code)) == -6  # AIE_E_DEVICE_TIMEOUT
        got.append(code.value)
    assert sorted(got) == [0x7F000001, 0x7F000002]
    assert lib.aie_device_status(stream, C.byref(code)) == 0 and code.value == 0
