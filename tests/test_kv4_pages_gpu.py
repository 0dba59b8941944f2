"""The pages' upkeep takes byte caches of 4 bits, in their layout, and no others."""
import pytest
import torch

from ai_engine_b200 import pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 2, 8, 16, 4, 64), (1, 2, 8, 16, 2, 40), (1, 2, 8, 2, 16, 48), (1, 2, 8, 2, 12, 40),
                                   (1, 2, 8, 1, 8, 180), (1, 2, 8, 2, 16, 0), (1, 2, 8, 2, 0, 40)])
def test_bytes_in_another_layout_are_refused(cuda_ok, shape):
    kv, st = torch.zeros(shape, dtype=torch.uint8, device="cuda"), pages.new_state(8, 4, 2)
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
    for call in (lambda: pages.fork(kv, st, src, dst), lambda: pages.copy(kv, src, dst), lambda: pages.compact(kv, st)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("size, hk, d", [(8, 1, 32), (16, 4, 64), (64, 2, 256)])
def test_4_bit_caches_are_taken(cuda_ok, size, hk, d):
    kv, st = pages.new_cache4(2, 8, size, hk, d), pages.new_state(8, 4, 2)
    src, dst = (torch.tensor([i], dtype=torch.int32, device="cuda") for i in (0, 1))
    kv[:, :, 0] = 7
    pages.copy(kv, src, dst)
    assert torch.equal(kv[:, :, 1], kv[:, :, 0]) and not bool(kv[:, :, 2:].any())
    grown = torch.tensor([size + 3], dtype=torch.int32, device="cuda")
    pages.grow(st, size, src, grown, size + 3)
    pages.fork(kv, st, src, dst)
    pages.compact(kv, st)
    assert int(st.status) == 0 and st.lens[:2].tolist() == [size + 3] * 2
