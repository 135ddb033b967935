"""layer_norm (csrc/norm.hip) against the formulas in 64 bits.

Tolerances: u = 2^-24 is half a step of fp32 relative to the value.  A row sum has at most 16 terms per lane, 6 shuffle levels and 16 waves one
after the other: D = 40 roundings.  With rho = mean|x| / std of the row the error of h is at most u (D rho + (D + 8) |h|), and every bound
below follows from it term by term; results in bf16 add half a step of bf16 (2^-8 of the value)."""
import numpy as np
import pytest
import torch

U = 2.0 ** -24
D = 40


def _reference(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits, and the elementwise error bounds of an fp32 evaluation"""
    x, dy = x.double(), dy.double()
    c = x.shape[1]
    w = torch.ones(c, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(c, dtype=torch.float64) if b is None else b.double()
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + eps)
    h = (x - m) * r
    gh = dy * w
    c1, c2 = gh.mean(1, keepdim=True), (gh * h).mean(1, keepdim=True)
    out = dict(y=h * w + b, dx=r * (gh - c1 - h * c2), dw=(dy * h).sum(0), db=dy.sum(0))
    rho = x.abs().mean(1, keepdim=True) * r
    eh = U * (D * rho + (D + 8) * h.abs())
    bound = dict(
        y=eh * w.abs() + 4 * U * ((h * w).abs() + b.abs()),
        dx=r * (U * (8 * gh.abs() + (D + 4) * gh.abs().mean(1, keepdim=True) + 2 * (D + 4) * h.abs() * (gh * h).abs().mean(1, keepdim=True)) +
                eh * c2.abs() + h.abs() * (gh.abs() * eh).mean(1, keepdim=True) + (D + 8) * U * (gh - c1 - h * c2).abs()))
    # a column sum: one lane adds the rows of its workgroup one after the other, at most 32 groups meet in LDS, the rest is double
    depth = x.shape[0] // 1024 + 2 + 32
    bound['dw'] = ((dy * h).abs() * (depth + 2) * U + dy.abs() * eh).sum(0)
    bound['db'] = dy.abs().sum(0) * depth * U
    return out, bound


def _check(got, ref, bound, what):
    got = got.detach().double().cpu()
    half = 0.0 if what[1] == torch.float32 else torch.finfo(what[1]).eps / 2
    tol = bound * (1 + half) + half * ref.abs() + 1e-30
    over = ((got - ref).abs() / tol).max()
    assert float(over) <= 1, f'{what}: {float(over):.3g} times the bound'


def _inputs(rows, cols, dtype, pdtype, seed=0, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * (0.5 + 2 * torch.rand(rows, 1, generator=g)) + offset).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(pdtype)
    b = (0.3 * torch.randn(cols, generator=g)).to(pdtype)
    dy = torch.randn(rows, cols, generator=g).to(dtype)
    return x, w, b, dy


def _run(x, w, b, dy, eps=1e-5, dev='cuda'):
    from mr3d_amd.detector.layers import layer_norm
    leaves = [None if t is None else t.detach().to(dev).requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy.to(dev)))
    return [y] + [None if t is None else next(grads) for t in leaves]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,pdtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 2), (5, 7), (33, 8), (257, 31), (300, 64), (70, 65), (40, 128), (19, 250), (64, 257), (513, 512),
                                       (1, 1024), (31, 1531), (9, 2048), (7, 2049), (5, 4100), (3, 8191), (2, 16383), (3, 16384), (40000, 64),
                                       (5001, 300)])
def test_forward_and_gradients(rows, cols, dtype, pdtype):
    x, w, b, dy = _inputs(rows, cols, dtype, pdtype, seed=rows + cols)
    ref, bound = _reference(x, w, b, dy, 1e-5)
    y, dx, dw, db = _run(x, w, b, dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == pdtype
    for name, t in (('y', y), ('dx', dx), ('dw', dw), ('db', db)):
        _check(t, ref[name], bound[name], (name, t.dtype, rows, cols))


@pytest.mark.gpu
@pytest.mark.parametrize('which', ['none', 'weight', 'bias'])
def test_absent_parameters(which):
    x, w, b, dy = _inputs(50, 96, torch.float32, torch.float32)
    w, b = (w if which == 'weight' else None), (b if which == 'bias' else None)
    ref, bound = _reference(x, w, b, dy, 1e-3)
    got = _run(x, w, b, dy, eps=1e-3)
    for name, t in zip(('y', 'dx', 'dw', 'db'), got):
        if t is not None:
            _check(t, ref[name], bound[name], (name, t.dtype, which))


@pytest.mark.gpu
def test_large_offset_keeps_its_variance():
    x, w, b, dy = _inputs(20, 1000, torch.float32, torch.float32, offset=3000.0)
    ref, bound = _reference(x, w, b, dy, 1e-5)
    for name, t in zip(('y', 'dx', 'dw', 'db'), _run(x, w, b, dy)):
        _check(t, ref[name], bound[name], (name, t.dtype))


@pytest.mark.gpu
def test_strided_rows_voxel_views_and_broadcast_gradients():
    from mr3d_amd.detector.layers import layer_norm
    x, w, b, dy = _inputs(24, 200, torch.float32, torch.float32)
    ref, bound = _reference(x[:, 3:67], w[3:67], b[3:67], dy[:, 1:65], 1e-5)
    xd = x.cuda().requires_grad_(True)
    y = layer_norm(xd[:, 3:67], w[3:67].cuda(), b[3:67].cuda())
    (gx,) = torch.autograd.grad(y, xd, dy.cuda()[:, 1:65])
    _check(y, ref['y'], bound['y'], ('y', torch.float32))
    _check(gx[:, 3:67], ref['dx'], bound['dx'], ('dx', torch.float32))
    assert float(gx[:, :3].abs().max()) == 0 and float(gx[:, 67:].abs().max()) == 0
    # transposed storage: no view with a contiguous last axis exists
    yt = layer_norm(x.cuda().t().contiguous().t()[:, 3:67], w[3:67].cuda(), b[3:67].cuda())
    assert torch.equal(yt, y.detach())
    # the voxels of a channels-last map
    m = torch.randn(2, 16, 3, 4, 5, generator=torch.Generator().manual_seed(5)).cuda().contiguous(memory_format=torch.channels_last_3d)
    v = layer_norm(m.permute(0, 2, 3, 4, 1))
    rv, bv = _reference(m.permute(0, 2, 3, 4, 1).reshape(-1, 16).cpu(), None, None, torch.zeros(120, 16), 1e-5)
    assert v.shape == (2, 3, 4, 5, 16)
    _check(v.reshape(-1, 16), rv['y'], bv['y'], ('y', torch.float32))
    # the gradient of a sum is one value expanded over the result
    xs = x.cuda().requires_grad_(True)
    ws = w.cuda().requires_grad_(True)
    layer_norm(xs, ws).sum().backward()
    rs, bs = _reference(x, w, None, torch.ones_like(x), 1e-5)
    _check(xs.grad, rs['dx'], bs['dx'], ('dx', torch.float32))
    _check(ws.grad, rs['dw'], bs['dw'], ('dw', torch.float32))


@pytest.mark.gpu
def test_rows_of_nan_and_infinity_stay_in_their_rows():
    x, w, b, dy = _inputs(40, 64, torch.float32, torch.float32)
    ref, bound = _reference(x, w, b, dy, 1e-5)
    x2 = x.clone()
    x2[7, 3], x2[20] = float('nan'), float('inf')
    y, dx, dw, db = _run(x2, w, b, dy)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[7, 20]] = False
    assert torch.isnan(y[7]).all() and torch.isnan(y[20]).all() and torch.isnan(dx[7]).all()
    _check(y[keep.cuda()], ref['y'][keep], bound['y'][keep], ('y', torch.float32))
    _check(dx[keep.cuda()], ref['dx'][keep], bound['dx'][keep], ('dx', torch.float32))
    _check(db, ref['db'], bound['db'], ('db', torch.float32))
    assert torch.isnan(dw).all()
    # a constant row: variance 0, y is the bias
    xc = torch.full((3, 64), 2.5)
    assert torch.equal(_run(xc, w, b, dy[:3])[0].cpu(), b.expand(3, 64))


@pytest.mark.gpu
def test_second_derivatives_are_refused_and_a_changed_input_is_noticed():
    from mr3d_amd.detector.layers import layer_norm
    x = torch.randn(4, 8, device='cuda', requires_grad=True)
    (g,) = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='second derivatives'):
        g.sum().backward()
    h = x * 1
    y = layer_norm(h)
    h.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()


@pytest.mark.gpu
def test_no_rows():
    from mr3d_amd.detector.layers import layer_norm
    x = torch.zeros(0, 32, device='cuda', requires_grad=True)
    w = torch.ones(32, device='cuda', requires_grad=True)
    y = layer_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 32) and x.grad.shape == (0, 32) and float(w.grad.abs().max()) == 0


@pytest.mark.gpu
def test_gradient_against_differences():
    """central differences of sum(y * cot) along random directions.  Step 2^-7 of inputs of size about 1: the third-order term is at most
    step^2 times a few units of |cot| |v| (1e-4 relative to 1), the rounding of y over the step about u sqrt(n) / step = 1e-4; both are
    taken against sqrt(n) |.| with a factor of 8."""
    from mr3d_amd.detector.layers import layer_norm
    x, w, b, dy = _inputs(12, 80, torch.float32, torch.float32, seed=3)
    _, dx, dw, db = _run(x, w, b, dy)
    g = torch.Generator().manual_seed(9)
    e = 2.0 ** -7
    f = lambda *a: float((layer_norm(*(t.cuda() for t in a)).double().cpu() * dy.double()).sum())
    for i, grad in ((0, dx), (1, dw), (2, db)):
        p = [x, w, b]
        v = torch.randn(p[i].shape, generator=g)
        hi, lo = list(p), list(p)
        hi[i], lo[i] = p[i] + e * v, p[i] - e * v
        diff = (f(*hi) - f(*lo)) / (2 * e)
        want = float((grad.double().cpu() * v.double()).sum())
        assert abs(diff - want) <= 8 * 2e-4 * np.sqrt(x.numel()), (i, diff, want)


@pytest.mark.gpu
def test_same_bits_every_run_on_another_stream_and_in_a_graph():
    from mr3d_amd.detector.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in _inputs(3000, 96, torch.bfloat16, torch.float32))

    def both():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    first = both()
    assert all(torch.equal(p, q) for p, q in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(k)).to(x.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, both())), k


def test_refusals_need_no_gpu():
    from abi import lib
    from mr3d_amd.detector.layers import layer_norm
    x = torch.zeros(4, 8)
    with pytest.raises(NotImplementedError):
        layer_norm(x)
    with pytest.raises(TypeError):
        layer_norm(x.half())
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        layer_norm(x.bfloat16(), torch.ones(8), torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        layer_norm(x, eps=-1.0)
    with pytest.raises(NotImplementedError):
        layer_norm(torch.zeros(1, 16385))
    with pytest.raises(NotImplementedError):
        layer_norm(torch.zeros(3, 0))
    L = lib()
    p = 64                                                    # never read: every call below is refused on the host
    assert L.mr3d_layer_norm_forward(None, 8, p, p, p, p, p, 4, 8, 1e-5, 0, 0, None) == 1
    assert L.mr3d_layer_norm_forward(p, 8, p, p, p, p, None, 4, 8, 1e-5, 0, 0, None) == 1
    assert L.mr3d_layer_norm_forward(p, 8, p, p, p, p, p, 0, 8, 1e-5, 0, 0, None) == 1
    assert L.mr3d_layer_norm_forward(p, 8, p, p, p, p, p, 4, 8, float('nan'), 0, 0, None) == 1
    assert L.mr3d_layer_norm_forward(p, 8, p, p, p, p, p, 4, 8, 1e-5, 2, 2, None) == 4
    assert L.mr3d_layer_norm_forward(p, 8, p, p, p, p, p, 4, 8, 1e-5, 0, 1, None) == 4
    assert L.mr3d_layer_norm_forward(p, 16385, p, p, p, p, p, 4, 16385, 1e-5, 0, 0, None) == 4
    assert L.mr3d_layer_norm_backward(p, 8, p, 8, p, p, p, p, p, p, 4, 8, 0, 0, None, 0, None) == 2
    assert L.mr3d_layer_norm_backward(p, 8, p, 8, p, None, p, p, p, p, 4, 8, 0, 0, p, 1 << 20, None) == 1
    assert L.mr3d_layer_norm_workspace_bytes(1, 8, 0) == 64 and L.mr3d_layer_norm_workspace_bytes(0, 8, 0) == 0
