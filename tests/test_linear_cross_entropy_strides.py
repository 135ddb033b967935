"""linear_cross_entropy on tensors whose strides say less than they seem to: an axis of one element may carry any stride."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_axes_of_one_element(dtype):
    """one class, one row, one feature, as transposes and slices of something larger; the same values stored plainly give the same bits"""
    from mr3d_amd.core import linear_cross_entropy
    g = torch.Generator().manual_seed(0)
    big = torch.randn(64, 64, generator=g).to(dtype).cuda()
    col = torch.randn(8, 1, generator=g).to(dtype).cuda()
    cases = [(big[:5, :8], col.t()), (col.t(), big[:7, :8]), (big[:5, 3:4], big[9:20, 7:8]), (big[:5, 3:4].t().contiguous().t(), big[:1, :1]),
             (big[:1, :8], big[:1, 8:16]), (big[:5, :8], big[:8, 5:6].t())]
    assert col.t().stride() == (1, 1) and col.t().is_contiguous()
    for x, w in cases:
        label = torch.zeros(x.shape[0], dtype=torch.int64, device='cuda')
        res = []
        for xs, ws in ((x, w), (torch.empty_like(x, memory_format=torch.contiguous_format).copy_(x), torch.zeros(w.shape, dtype=dtype, device='cuda').copy_(w))):
            leaves = [xs.detach().requires_grad_(True), ws.detach().requires_grad_(True)]
            loss = linear_cross_entropy(leaves[0], leaves[1], label)
            res.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
        assert all(torch.equal(p, q) and bool(torch.isfinite(p).all()) for p, q in zip(*res)), (x.shape, w.shape)
