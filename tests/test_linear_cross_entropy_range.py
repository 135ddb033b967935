"""linear_cross_entropy where probabilities span many orders of magnitude: the gradients of unlikely classes are small, and as exact as the others."""
import pytest
import torch

from test_linear_cross_entropy import U, _check, _reference


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


def _run(x, w, b, label, rw):
    from mr3d_amd.core import linear_cross_entropy
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], label.cuda(), rw.cuda(), leaves[2])
    return [t.detach().double().cpu() for t in (loss,) + torch.autograd.grad(loss, leaves)]


def _fp32(x, w, b, label, rw):
    """64-bit values (1 - p_label as a sum over the others) and bounds.  E as in test_linear_cross_entropy: a logit is off by Z, a probability by E = 2 Z +
    2^-19 of itself.  dx: g relative to its row's 1 - p_label, 2^-22 of the value or 2^-39 (half a step of the lower plane).  dW: the same relative to the
    class's largest g |x|_max among 128 rows.  db: fp32 sums.  Products: 2^-21 + (204 + n / 128) u."""
    x, w, b, rw = (t.double() for t in (x, w, b, rw))
    n, v = len(x), len(w)
    rows = (label != -100).nonzero().squeeze(1)
    xl, ll, rl = x[rows], label[rows], rw[rows]
    m = len(rows)
    at = torch.arange(m)
    z = xl @ w.t() + b
    others = z.clone()
    others[at, ll] = float('-inf')
    so, zl = torch.logsumexp(others, 1), z[at, ll]
    ce = torch.logaddexp(so, zl) - zl
    ce = torch.where(zl > so, torch.log1p(torch.exp(so - zl)), ce)
    rest = torch.exp(so - torch.logaddexp(so, zl))
    gp = torch.softmax(others, 1)
    gp[at, ll] = -1
    t = (rest * rl / m)[:, None]
    g = gp * t
    prod = lambda k: 2.0 ** -21 + (204 + k / 128) * U
    ez = prod(x.shape[1]) * xl.norm(dim=1, keepdim=True) * w.norm(dim=1).max() + 2 * U * z.abs().amax(1, keepdim=True)
    e = 2 * ez + 2.0 ** -19
    eg = e * g.abs()
    dx, ex = torch.zeros_like(x), torch.zeros_like(x)
    dx[rows] = g @ w
    ex[rows] = ((e + 2.0 ** -22) * g.abs() + 2.0 ** -39 * t) @ w.abs() + prod(v) * (g.abs() @ w.abs())
    top = torch.zeros(v, dtype=torch.float64)
    for s in range(0, m, 128):
        top += (g[s:s + 128].abs() * xl[s:s + 128].abs().amax(1, keepdim=True)).amax(0) * min(128, m - s)
    ew = ((e + 2.0 ** -22) * g.abs()).t() @ xl.abs() + 2.0 ** -38 * top[:, None] + prod(m) * (g.abs().t() @ xl.abs())
    loss = (ce * rl).sum() / m
    el = (torch.minimum(2 * ez.squeeze(1) + 2.0 ** -20, e.squeeze(1) * ce.clamp(max=1) + (2 * ez.squeeze(1) + 2.0 ** -20) * (ce > 1)) * rl).sum() / m
    return (loss.reshape(1), dx, g.t() @ xl, g.sum(0)), ((el + 6 * U * loss).reshape(1), ex, ew, eg.sum(0) + 300 * U * g.abs().sum(0))


def _all_within(got, ref, bound, what):
    for name, t, r, e in zip(('loss', 'dx', 'dw', 'db'), got, ref, bound):
        assert torch.isfinite(t).all(), (name,) + what
        over = float(((t - r).abs() / (e + 2 * U * r.abs() + 1e-36)).max())
        assert over <= 1, (name, over) + what


@pytest.mark.gpu
@pytest.mark.parametrize('nats', [5.0, 25.0, 50.0])
@pytest.mark.parametrize('n,k,v', [(1, 8, 500), (2, 3, 40), (200, 16, 1500), (700, 40, 9000), (20000, 20, 130)])
def test_unlikely_classes_fp32(n, k, v, nats):
    x, w, b, label, rw = _spread(n, k, v, torch.float32, nats)
    label[0] = int(b.argmin())
    ref, bound = _fp32(x, w, b, label, rw)
    _all_within(_run(x, w, b, label, rw), ref, bound, (n, k, v, nats))


@pytest.mark.gpu
@pytest.mark.parametrize('margin', [0.0, 14.0, 25.0, 40.0])
def test_certain_rows_beside_uncertain_ones_fp32(margin):
    """a third of the rows gives its label all but exp(-margin), and rows differ by 2^20 in size: each row of dx is right relative to its own gradient"""
    n, v = 300, 700
    x, w, b, label, rw = _spread(n, 16, v, torch.float32, 3.0, seed=3)
    label = torch.arange(n) % v
    x[:, 8:] = 0
    w[:, 8:] = 0
    for i in range(0, n, 3):                                 # features 8.. lift the label of every third row
        x[i, 8 + i % 8] = 1.0
    w[label[::3], 8 + torch.arange(0, n, 3) % 8] = margin + 8.0
    scale = 2.0 ** torch.randint(-20, 1, (n,), generator=torch.Generator().manual_seed(0))
    x[1::3] *= scale[1::3, None]
    ref, bound = _fp32(x, w, b, label, rw)
    got = _run(x, w, b, label, rw)
    _all_within(got, ref, bound, (margin,))


@pytest.mark.gpu
@pytest.mark.parametrize('want', [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)])
@pytest.mark.parametrize('rows,live', [(300, 300), (300, 0), (260, 129)])
def test_each_gradient_alone_has_the_same_bits(want, rows, live):
    """dx alone, dW alone and db alone take other routes through memory; rows that do not count leave no trace in them"""
    from mr3d_amd.core import linear_cross_entropy
    x, w, b, label, rw = (t.cuda() for t in _spread(rows, 24, 333, torch.float32, 10.0))
    label = torch.where(torch.arange(rows, device='cuda') < live, label.clamp(min=0), torch.full_like(label, -100))
    res = []
    for w3 in ((1, 1, 1), want):
        leaves = [t.clone().requires_grad_(bool(q)) for t, q in zip((x, w, b), w3)]
        loss = linear_cross_entropy(leaves[0], leaves[1], label, rw, leaves[2])
        g = iter(torch.autograd.grad(loss, [t for t in leaves if t.requires_grad]))
        res.append([loss.detach()] + [next(g) if q else None for q in w3])
    for p, q in zip(*res):
        assert q is None or torch.equal(p, q)
    if not live:
        assert all(not t.any() for t in res[0])
