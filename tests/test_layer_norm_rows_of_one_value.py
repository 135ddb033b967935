"""Rows of one value: variance 0, so the result is the bias, whatever the value, the number of columns and its reciprocal's rounding."""
import numpy as np
import pytest
import torch


def test_a_sum_times_the_reciprocal_is_not_the_mean():
    """why the kernel takes the mean twice: 41 times 1, summed exactly, times fl(1 / 41) is the float below 1, and 1 / sqrt(eps) enlarges that"""
    one = np.float32(41) * (np.float32(1) / np.float32(41))
    assert one < 1 and (1 - float(one)) / 1e-5 ** 0.5 > 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('cols', [3, 41, 49, 98, 103, 107, 196, 392, 1000, 1531, 2049, 5003, 16383])
def test_the_bias_comes_out(cols, dtype):
    """The first mean is off by at most some dozen steps, the differences from it are equal whole numbers of steps, their sums below 2^24 steps and
    exact, so that the second mean is the value itself: no tolerance.  Backward: h = 0, so dx = r (gh - mean gh), dw = 0."""
    from mr3d_amd.detector.layers import layer_norm
    g = torch.Generator().manual_seed(cols)
    value = torch.cat([torch.tensor([1.0, -1.0, 1000.0, 0.1, 3.0e-5, -7777.7]), 100 * torch.randn(26, generator=g)])
    x = value.to(dtype)[:, None].expand(32, cols).contiguous().cuda().requires_grad_(True)
    w, b = torch.randn(cols, generator=g).cuda().requires_grad_(True), torch.randn(cols, generator=g).cuda()
    y = layer_norm(x, w, b)
    assert torch.equal(y, b.to(dtype).expand(32, cols))
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert not dw.any() and torch.isfinite(dx).all()
