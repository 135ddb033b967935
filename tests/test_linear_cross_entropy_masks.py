"""linear_cross_entropy where the bias masks: every class with the type's lowest value, the label among the masked, masked classes with any weights."""
import math

import pytest
import torch

from test_linear_cross_entropy import _check, _inputs


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('v', [1, 2, 50, 700])
def test_every_class_at_the_lowest_value(dtype, v):
    """Logits of size 1 vanish beside 3e38, in 64 bits too: all classes are equally likely, the loss is log v (as torch's cross entropy, which takes the
    difference from the maximum first, gives it).  bf16's own lowest value the same way"""
    x, w, _, label, rw = _inputs(40, 24, v, dtype)
    for low in (torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min):
        b = torch.full((v,), low)
        # the logits are exactly equal, so that the bound's share of their size (3e38) does not apply: exponentials and sums, g's planes or its rounding
        p = torch.full((40, v), 1.0 / v, dtype=torch.float64)
        p[torch.arange(40), label.clamp(min=0)] -= 1
        n = int((label != -100).sum())
        g = p * ((label != -100).double() * rw.double() / n)[:, None]
        loss64 = (rw.double() * (label != -100)).sum().reshape(1) * math.log(v) / n
        want = dict(loss=loss64, dx=g @ w.double(), dw=g.t() @ x.double(), db=g.sum(0))
        step = 2.0 ** -18 if dtype == torch.float32 else 2.0 ** -7 + 2.0 ** -9
        size = dict(loss=loss64, dx=g.abs() @ w.double().abs(), dw=g.abs().t() @ x.double().abs(), db=g.abs().sum(0))
        from mr3d_amd.core import linear_cross_entropy
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], label.cuda(), rw.cuda(), leaves[2])
        for name, t in zip(('loss', 'dx', 'dw', 'db'), (loss,) + torch.autograd.grad(loss, leaves)):
            _check(t, want[name], (2.0 ** -18 if name == 'loss' else step) * size[name], (name, v, low, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_labels_that_are_masked(dtype):
    """a label of the lowest value has a loss of 3e38 and p = 0: its row's gradient is that of p = softmax of the others and -1; one of -infinity an infinite loss"""
    from mr3d_amd.core import linear_cross_entropy
    x, w, b, label, _ = _inputs(12, 16, 90, dtype, dead=0.0)
    b = b.float()
    label[:] = 7
    for low in (torch.finfo(torch.float32).min, float('-inf')):
        b[7] = low
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], label.cuda(), bias=leaves[2])
        dx, dw, db = torch.autograd.grad(loss, leaves)
        assert float(loss) == -low or abs(float(loss) / -low - 1) <= 2.0 ** -20
        z = x.double() @ w.double().t() + b.double()
        p = torch.softmax(z, 1)
        p[:, 7] -= 1
        g = p / 12
        step = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -6
        for got, ref in ((dx, g @ w.double()), (dw, g.t() @ x.double()), (db, g.sum(0))):
            assert float((got.double().cpu() - ref).norm()) <= step * float(ref.norm())


@pytest.mark.gpu
@pytest.mark.parametrize('low', [float('-inf'), torch.finfo(torch.float32).min])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_masked_classes_may_have_any_finite_weights(dtype, low):
    """weights of 1e-30 to 1e30 in classes that the bias takes out: the others' loss and gradients have the bits of the same call with zeros there"""
    from mr3d_amd.core import linear_cross_entropy
    x, w, b, label, rw = (t.cuda() for t in _inputs(60, 40, 500, dtype, dead=0.1))
    keep = torch.ones(500, dtype=torch.bool, device='cuda')
    keep[::5], keep[256:384] = False, False
    kept = keep.nonzero().squeeze(1)
    label = torch.where(label < 0, label, kept[label % len(kept)])
    b = b.float().masked_fill(~keep, low)
    out = []
    for junk in (0.0, 1e-30, 1.0, 1e8, 1e30):
        wj = torch.where(keep[:, None], w, torch.randn(500, 40, generator=torch.Generator().manual_seed(1)).cuda().to(dtype) * junk)
        leaves = [t.detach().requires_grad_(True) for t in (x, wj, b)]
        loss = linear_cross_entropy(leaves[0], leaves[1], label, rw, leaves[2])
        out.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
        assert all(bool(torch.isfinite(t).all()) for t in out[-1]) and not out[-1][2][~keep].any(), junk
        assert all(torch.equal(p, q) for p, q in zip(out[0], out[-1])), junk
