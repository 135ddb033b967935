"""linear_cross_entropy at the largest number of rows that it takes."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_four_million_rows(dtype):
    """2^22 rows against 33 classes, every gradient wanted.  bf16: g is off by 2^-8 + 2^-10 of each entry to either side, which averages out in db over the
    rows; what is left of db is taken as 2^-12 of the sum of |g|, of the loss as 2^-18."""
    from mr3d_amd.core import linear_cross_entropy
    rows, k, v = 1 << 22, 8, 33
    g = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(rows, k, generator=g, device='cuda').to(dtype).requires_grad_(True)
    w = torch.randn(v, k, generator=g, device='cuda').to(dtype).requires_grad_(True)
    b = torch.randn(v, generator=g, device='cuda').requires_grad_(True)
    label = torch.randint(0, v, (rows,), generator=g, device='cuda')
    label[::5] = -100
    loss = linear_cross_entropy(x, w, label, bias=b)
    dx, dw, db = torch.autograd.grad(loss, [x, w, b])
    n = int((label >= 0).sum())
    total, wdw, wdb, mag = 0.0, 0, 0, 0
    for s in range(0, rows, 1 << 19):
        sl = slice(s, s + (1 << 19))
        keep = label[sl] >= 0
        xd, lab = x[sl].detach().double(), label[sl].clamp(min=0)
        z = xd @ w.detach().double().t() + b.detach().double()
        logp = torch.log_softmax(z, 1)
        total -= float(logp.gather(1, lab[:, None])[keep].sum())
        p = logp.exp().scatter_add(1, lab[:, None], torch.full((len(lab), 1), -1.0, dtype=torch.float64, device='cuda')) * (keep[:, None] / n)
        wdw, wdb, mag = wdw + p.t() @ xd, wdb + p.sum(0), mag + p.abs().sum(0)
        want = p @ w.detach().double()
        step = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -14
        assert float((dx[sl].double() - want).norm()) <= step * float(want.norm())
    assert abs(float(loss.detach()) - total / n) <= 2.0 ** -18 * total / n
    assert bool(((db.double() - wdb).abs() <= 2.0 ** -12 * mag).all())
    assert float((dw.double() - wdw).norm()) <= (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -14) * float(wdw.norm()) + 2.0 ** -12 * float(mag.norm())
