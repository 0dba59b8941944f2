"""What the decoder that reads frames refuses before it needs a GPU."""
import pytest
import torch

from ai_engine_b200 import decoder


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.int8, torch.float8_e4m3fn])
def test_types_that_a_step_cannot_take(dtype):
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        decoder.FrameDecoder(1, 96, 4, 2, 64, streams=3, pages_=60, dtype=dtype, device="cpu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_types_that_it_takes(dtype):
    m = decoder.FrameDecoder(1, 96, 4, 2, 64, streams=3, pages_=60, dtype=dtype, device="cpu")
    assert m.wqkv[0].dtype == dtype
