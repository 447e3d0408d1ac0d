"""Layer normalisation on the CPU: types."""
import pytest
import torch

from distributed_tensorflow_amd.ops import functional as F


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint8, torch.bool])
def test_whole_numbers_are_refused(dtype):
    # (the result, cast back to x's type, would be cut to whole numbers)
    with pytest.raises(ValueError, match="floating-point"):
        F.layer_norm(torch.ones(2, 4).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64])
def test_floating_point_types_are_kept(dtype):
    x = torch.arange(8.0).view(2, 4).to(dtype)
    y = F.layer_norm(x, eps=0.0)
    want = torch.tensor([-1.5, -0.5, 0.5, 1.5], dtype=torch.float64) / 1.25 ** 0.5
    assert y.dtype == dtype   # one rounding, and four of fp32 before it
    assert ((y.double() - want).abs() <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22)).all()
