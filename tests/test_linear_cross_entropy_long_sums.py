"""linear_cross_entropy, bf16: sums of one sign over many rows, classes or features.  A matrix instruction that cut what it adds always downwards would let
them drift with their length (8 u an instruction, u = 2^-24: 1 % of 655360 rows).  The tolerances do not grow with the length: DRIFT, a
quarter of the largest rounding to bf16, for what is rounded to bf16; 2^-18 of the logits for the fp32 loss."""
import pytest
import torch

U = 2.0 ** -24
DRIFT = 2.0 ** -10


def _grads(x, w, label, **kw):
    from mr3d_amd.core import linear_cross_entropy
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    loss = linear_cross_entropy(x, w, label, **kw)
    return (loss.detach(),) + torch.autograd.grad(loss, leaves)


def _exact(x, w, label, avg):
    x, w = x.detach().double(), w.detach().double()
    z = x @ w.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    at = torch.arange(len(x), device=x.device)
    loss = (lse.squeeze(1) - z[at, label]).sum() / avg
    g = torch.exp(z - lse)
    g[at, label] -= 1
    return loss, g / avg, x, w


@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,v', [(655360, 16, 100), (1000003, 40, 7), (70001, 300, 33)])
def test_dw_of_many_rows(rows, k, v):
    """Positive features and classes that are never a label: every product of their rows of dW has the same sign.  Roundings of g and t x are off to
    either side and average out over the rows; a result's own rounding (2^-8 at most) averages out over the entries, 6 / sqrt(3 n) of it.  What is left of the mean
    relative error is a drift."""
    g = torch.Generator(device='cuda').manual_seed(rows)
    x = torch.rand(rows, k, generator=g, device='cuda').add_(0.25).bfloat16()
    w = torch.randn(v, k, generator=g, device='cuda').mul_(0.05).bfloat16()
    label = torch.randint(0, 2, (rows,), generator=g, device='cuda')
    loss, dx, dw = _grads(x, w, label)
    want = torch.zeros(v, k, dtype=torch.float64, device='cuda')
    total = 0.0
    for s in range(0, rows, 1 << 16):
        l, gg, xd, _ = _exact(x[s:s + (1 << 16)], w, label[s:s + (1 << 16)], rows)
        want += gg.t() @ xd
        total += float(l)
    assert abs(float(loss) - total) <= (2 * 17 * (k // 32 + 1) * U * 3 + 2.0 ** -19) * total + 1e-6
    rel = (dw.double() / want - 1)[2:]
    n = rel.numel()
    assert abs(float(rel.mean())) <= DRIFT + 6 * 2.0 ** -8 / (3 * n) ** 0.5
    assert float(rel.abs().max()) <= 2.0 ** -8 + 2 * DRIFT
    lab = dw[:2].double()
    assert float((lab - want[:2]).norm()) <= 2.0 ** -7 * float(want[:2].norm()) + 2.0 ** -8 * float((x.double().sum(0) / rows).norm())


@pytest.mark.gpu
def test_dx_of_many_classes():
    """16 x 16 large tiles, one part of 65600 classes each.  Class 0 is everybody's label and has no weights, so dx is the mean of the others' weights"""
    g = torch.Generator(device='cuda').manual_seed(1)
    v, k, rows = 65600, 4096, 4096
    x = torch.randn(rows, k, generator=g, device='cuda').bfloat16()
    w = torch.randn(v, k, generator=g, device='cuda').mul_(0.01).add_(0.02).bfloat16()
    w[0] = 0
    label = torch.zeros(rows, dtype=torch.int64, device='cuda')
    _, dx, _ = _grads(x, w, label)
    for s in (slice(0, 24), slice(2047, 2063), slice(4080, 4096)):
        _, gg, _, wd = _exact(x[s], w, label[s], rows)
        want = gg @ wd
        # two roundings of g over 65600 entries of random error, far below the drift; the result's rounding
        assert float((dx[s].double() - want).norm()) <= (2.0 ** -8 + DRIFT) * float(want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize('rows,k,v', [(70, 40000, 300), (1, 65536, 65), (300, 8200, 1000)])
def test_logits_of_many_features(rows, k, v):
    """positive features and weights: a logit's products have one sign.  The loss is a difference of two of them"""
    g = torch.Generator(device='cuda').manual_seed(k)
    x = torch.rand(rows, k, generator=g, device='cuda').add_(0.5).bfloat16()
    w = torch.rand(v, k, generator=g, device='cuda').mul_(40.0 / k).add_(20.0 / k).bfloat16()
    label = torch.randint(0, v, (rows,), generator=g, device='cuda')
    loss, dx, dw = _grads(x, w, label)
    want, gg, xd, wd = _exact(x, w, label, rows)
    z = float((xd @ wd.t()).max())
    ez = 2.0 ** -18 * z
    assert abs(float(loss) - float(want)) <= 2 * ez + 2.0 ** -20 + 8 * U * float(want), (float(loss), float(want), z)
    for got, ref, mag in ((dx, gg @ wd, gg.abs() @ wd.abs()), (dw, gg.t() @ xd, gg.abs().t() @ xd.abs())):
        bound = (2 * ez + 2.0 ** -7 + 2.0 ** -10 + DRIFT) * mag + 2.0 ** -8 * ref.abs()
        assert bool(((got.double() - ref).abs() <= bound).all())
