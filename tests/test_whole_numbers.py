"""CPU checks of how the entry points take whole numbers."""
import pytest
import torch

from specdec import _lib


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8])
def test_numbers_that_32_bits_hold_stay_as_they_are(dtype):
    x = torch.tensor([0, 1, 127], dtype=dtype)
    y = _lib.as_int32("x", x)
    assert y.dtype == torch.int32 and y.tolist() == [0, 1, 127]
    assert (y is x) == (dtype is torch.int32)
    z = _lib.as_int32("x", torch.arange(6, dtype=dtype).view(2, 3).t())
    assert z.is_contiguous() and z.tolist() == [[0, 3], [1, 4], [2, 5]]


def test_numbers_past_32_bits_stay_out_of_range():
    x = [-2 ** 31, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, -2 ** 32, 2 ** 63 - 1, -2 ** 63, -1]
    want = [max(-2 ** 31, min(2 ** 31 - 1, v)) for v in x]
    assert _lib.as_int32("x", torch.tensor(x)).tolist() == want


def test_only_whole_numbers_are_taken():
    z = torch.zeros(2)
    for dtype in (torch.int64, torch.int32, torch.uint8, torch.int16, torch.uint32):
        assert _lib.as_int64("keep", z.to(dtype)).dtype == torch.int64
    for dtype in (torch.float32, torch.float64, torch.float16, torch.bfloat16, torch.bool, torch.complex64):
        for take in (_lib.as_int64, _lib.as_int32, _lib.whole):
            with pytest.raises(TypeError, match="keep must be whole numbers"):
                take("keep", z.to(dtype))
