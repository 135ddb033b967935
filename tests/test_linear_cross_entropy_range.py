"""linear_cross_entropy where probabilities span many orders of magnitude: the gradients of unlikely classes are small, and as exact as the others."""
import pytest
import torch

from test_linear_cross_entropy import _check, _reference


def _spread(n, k, v, dtype, nats, seed=0):
    """logits that fall by `nats` over the classes, in an order that puts likely and unlikely classes side by side"""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g).to(dtype)
    w = (torch.randn(v, k, generator=g) / k ** 0.5).to(dtype)
    b = -nats * torch.arange(v) / v
    b = b[torch.randperm(v, generator=g)]
    label = torch.randint(0, v, (n,), generator=g)
    label[::9] = -100
    return x, w, b, label, 0.25 + torch.rand(n, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize('n,k,v', [(1, 8, 500), (200, 16, 1500), (700, 40, 9000)])
def test_unlikely_classes_bf16(n, k, v):
    """Class by class against 64 bits: an entry of g is off by 2^-8 + 2^-10 of itself (its own rounding, the stored exponential's), t x by another 2^-8, however
    small the entry -- the bound is the one of the even case, which has no absolute part."""
    from mr3d_amd.core import linear_cross_entropy
    x, w, b, label, rw = _spread(n, k, v, torch.bfloat16, 50.0)
    label[0] = int(b.argmin())
    ref, bound = _reference(x, w, b, label, rw)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], label.cuda(), rw.cuda(), leaves[2])
    for name, t in zip(('loss', 'dx', 'dw', 'db'), (loss,) + torch.autograd.grad(loss, leaves)):
        _check(t, ref[name], bound[name], (name, n, k, v))
