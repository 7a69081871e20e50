"""quantize_w4 at the ends of the types' ranges, and W4Weight.to."""
import pytest
import torch

from kernel_pocs_b200.w4 import W4Weight, quantize_w4
from tests.test_w4 import random_parts, weight64


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-37), (torch.bfloat16, 1e-38), (torch.bfloat16, 3e-39),
                                        (torch.bfloat16, 1e38), (torch.float16, 1e-3), (torch.float16, 2e-5),
                                        (torch.float16, 2e-6), (torch.float16, 6e4)])
@pytest.mark.parametrize("zero_points", [False, True])
def test_weights_whose_scale_leaves_the_normal_range(dtype, size, zero_points):
    g = torch.Generator().manual_seed(0)
    weight = ((torch.rand(6, 70, generator=g) * 2 - 1) * size).to(dtype)
    weight[:, ::9] = 0.0
    weight[3] = 0.0
    w = quantize_w4(weight, 32, zero_points)
    got = weight64(w.packed, w.scales, w.zeros, 70, 32)
    which = torch.arange(70) // 32
    step = w.scales.double()[:, which]
    # Half a step; at the ends of the range up to 15 times what the scale's own rounding took off: half a unit of it, which
    # below the normal range is half the type's smallest number.  With zero points half a step more, the zero's rounding.
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    scale_error = torch.maximum(step * eps / 2, torch.full_like(step, tiny / 2))
    # products with the inverse are off by a few parts of 2^24
    bound = step * (0.5 + 0.5 * zero_points + 2.0 ** -18) + 15 * scale_error
    err = (got - weight.double()).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    assert not bool(got[3].any())
    assert not zero_points or not bool(got[:, ::9].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1.0), (torch.bfloat16, 1e-38), (torch.float16, 2e-6)])
@pytest.mark.parametrize("zero_points", [False, True])
def test_the_device_gives_the_codes_of_the_host(dtype, size, zero_points):
    g = torch.Generator().manual_seed(1)
    weight = ((torch.rand(40, 300, generator=g) * 2 - 1) * size).to(dtype)
    host, device = quantize_w4(weight, 64, zero_points), quantize_w4(weight.cuda(), 64, zero_points)
    assert torch.equal(device.scales.cpu(), host.scales)
    # a product may be rounded to the other side of half a step by the last bit of an inverse, no further
    off = (weight64(device.packed, device.scales, device.zeros, 300, 64) - weight64(host.packed, host.scales, host.zeros, 300, 64)).abs()
    assert bool((off <= host.scales.double()[:, torch.arange(300) // 64]).all()) and float((off > 0).double().mean()) < 0.01


def test_to_moves_and_does_not_convert():
    w = W4Weight(*random_parts(20, 70, 32, True, torch.bfloat16), in_features=70, group_size=32)
    assert w.to("cpu") is w and w.to(torch.device("cpu")) is w and w.to(device="cpu") is w
    meta = w.to("meta")
    assert meta.device.type == "meta" and meta.blocks.dtype == torch.uint8 and meta.shape == w.shape
    for other in (torch.float16, torch.uint8, torch.zeros(1, dtype=torch.float16), None):
        with pytest.raises(TypeError, match="device"):
            w.to(other)
