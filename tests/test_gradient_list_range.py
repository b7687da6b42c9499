"""Norms of gradient lists at the end of fp32's range."""
import math

import pytest
import torch

import dlvk_b200 as dl

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_norm_above_fp32_scales_nothing(device, dtype, strided, given):
    """Sixteen elements of 3e38 have a norm of 1.2e39, which the caller gets as infinity: like every norm
    that is not finite it scales by 1."""
    def tensors():
        t = torch.full((4, 8), 3e38, device=device).to(dtype)
        return [t[:, ::2] if strided else t[:, :4].contiguous(), torch.ones(3, device=device)]

    grads, out = tensors(), [torch.zeros(4, 4, device=device), torch.zeros(3, device=device)] if given else None
    norm = dl.GradientClipping.clip_global_norm(grads, 1.0, out)
    assert math.isinf(norm.item()) and math.isinf(dl.GradientClipping.global_norm(tensors()).item())
    for got, had in zip(out or grads, tensors()):
        assert torch.equal(got.float(), had.float())


@pytest.mark.parametrize("device", DEVICES)
def test_a_norm_just_below_it_scales(device):
    """sqrt(2) 2e38 = 2.83e38 is finite.  Its scale of 3.5e-39 lies among fp32's smallest numbers, 2^-149
    apart: off by 2^-150 / 3.5e-39 = 2^-22.3 of itself, and the product by 2^-24."""
    t = torch.full((2,), 2e38, device=device)
    norm = dl.GradientClipping.clip_global_norm([t], 1.0)
    want = float(torch.tensor(2e38)) * math.sqrt(2.0)
    assert abs(norm.item() - want) <= 2.0 ** -23 * want
    assert abs(t[0].item() - math.sqrt(0.5)) <= 2.0 ** -21.5 * math.sqrt(0.5) and t[0].item() == t[1].item()
