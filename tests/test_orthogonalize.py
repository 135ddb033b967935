"""orthogonalize (csrc/ortho.hip) against the same iteration in 64 bits.

Tolerance.  Up to 64 rows the iteration is in double.  Above: the factors carry 22 bits (rounding 2^-23 of the value at most, lo * lo of at most 2^-22 of a
term is dropped), and a matrix instruction cuts each of its 32 products 2 bits below the last place of the largest.  Taken as independent, these
errors perturb a product by 2^-23 of the product of its factors' norms or less, and one step -- three products of factors with spectral norms
below 1.3, weighted 1, b = 4.8, c = 2 and 1 -- perturbs X by at most about d = 2^-20 |X|_F.  The map's slope is largest at 0 (a = 3.4445), so an
error of step k is amplified by a^(steps-1-k) at most while |X|_F itself grows towards sqrt(m):
|error| <= d sum_k a^(steps-1-k) |X_k|_F, with the norms of the iterates taken from the reference.
Results in bf16 add half a step, 2^-8 of each value."""
import pytest
import torch

C = (3.4445, -4.7750, 2.0315)


def _reference(g, steps=5, c=C, eps=1e-7):
    x = g.double().reshape(g.shape[0], -1)
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    norms = []
    for _ in range(steps):
        norms.append(float(x.norm()))
        a = x @ x.t()
        x = c[0] * x + (c[1] * a + c[2] * a @ a) @ x
    tol = 2.0 ** -20 * sum(abs(c[0]) ** (steps - 1 - k) * n for k, n in enumerate(norms))
    return (x.t() if tall else x).reshape(g.shape), tol


def _check(got, g, **kw):
    ref, tol = _reference(g.cpu(), **kw)
    assert got.shape == g.shape and got.dtype == g.dtype
    got = got.double().cpu()
    if g.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * float(ref.norm())
    err = float((got - ref).norm())
    assert err <= tol, (tuple(g.shape), g.dtype, err / max(float(ref.norm()), 1e-30), tol / max(float(ref.norm()), 1e-30))


def _gauss(m, n, seed=0, dtype=torch.float32):
    return torch.randn(m, n, generator=torch.Generator().manual_seed(seed + 1000 * m + n)).mul_(1e-3).to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('m,n', [(1, 1), (1, 5), (7, 1), (2, 3), (16, 1029), (31, 33), (33, 31), (64, 64), (64, 1728), (100, 129), (128, 128), (129, 127),
                                 (130, 257), (1000, 64), (257, 300), (500, 40), (333, 1301), (640, 640), (20, 9000)])
def test_matrix(m, n, dtype):
    from mr3d_amd.core import orthogonalize
    g = _gauss(m, n, dtype=dtype)
    _check(orthogonalize(g), g)


@pytest.mark.gpu
def test_list_of_mixed_shapes_types_and_axes_equals_the_single_calls():
    from mr3d_amd.core import orthogonalize
    shapes = [(64, 64), (16, 1029), (300, 200), (5, 7), (200, 3000), (1, 1), (128, 512)] * 4
    mats = [_gauss(m, n, k, torch.bfloat16 if k % 3 == 1 else torch.float32) for k, (m, n) in enumerate(shapes)]
    mats.append(_gauss(32, 16 * 27).reshape(32, 16, 3, 3, 3))
    mats.append(torch.empty(0, 5, device='cuda'))
    out = orthogonalize(mats)
    for g, o in zip(mats, out):
        if g.numel():
            _check(o, g)
    assert out[-1].shape == (0, 5) and orthogonalize([]) == []
    again = orthogonalize(mats)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.gpu
@pytest.mark.parametrize('count', [15, 16, 47])
def test_long_lists(count):
    """more matrices than one launch takes as arguments, small and large ones mixed, runs of either"""
    from mr3d_amd.core import orthogonalize
    g = torch.Generator().manual_seed(count)
    mats = []
    for k in range(count):
        lo, hi = ((1, 64) if k % 20 < 8 else (65, 200) if k % 20 < 16 else (1, 200))
        m, n = (int(v) for v in torch.randint(lo, hi + 1, (2,), generator=g))
        mats.append(_gauss(m, n, k, torch.bfloat16 if k % 5 == 4 else torch.float32))
    for got, want in zip(orthogonalize(mats), mats):
        _check(got, want)


@pytest.mark.gpu
def test_spectra():
    """low rank, decaying spectrum, duplicated rows, one dominant direction, zeros"""
    from mr3d_amd.core import orthogonalize
    g = torch.Generator().manual_seed(7)
    q = torch.linalg.qr(torch.randn(200, 200, generator=g, dtype=torch.float64))[0]
    p = torch.linalg.qr(torch.randn(300, 300, generator=g, dtype=torch.float64))[0][:200]
    cases = [q @ torch.diag(torch.logspace(0, -6, 200, dtype=torch.float64)) @ p,
             torch.randn(200, 4, generator=g, dtype=torch.float64) @ torch.randn(4, 300, generator=g, dtype=torch.float64),
             torch.randn(1, 300, generator=g, dtype=torch.float64).expand(200, 300).clone(),
             torch.randn(200, 300, generator=g, dtype=torch.float64) + 1e4]
    for t in cases:
        t = t.float().cuda()
        _check(orthogonalize(t), t)
    z = torch.zeros(50, 70, device='cuda')
    assert torch.equal(orthogonalize(z), z)


@pytest.mark.gpu
def test_scales_of_the_input():
    """the norm is taken in double: neither squares that overflow fp32 nor values near its smallest change the result"""
    from mr3d_amd.core import orthogonalize
    g = _gauss(60, 90)
    for s in (2.0 ** 100, 2.0 ** -60):
        _check(orthogonalize(g * s, eps=0.0), g * s, eps=0.0)
    _check(orthogonalize(g, eps=0.5), g, eps=0.5)
    _check(orthogonalize(g, steps=1), g, steps=1)
    _check(orthogonalize(g, steps=8, coefficients=(1.875, -1.25, 0.375)), g, steps=8, c=(1.875, -1.25, 0.375))


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_matrix():
    from mr3d_amd.core import orthogonalize
    mats = [_gauss(40, 60), _gauss(64, 64), _gauss(130, 50), _gauss(40, 60, 5), _gauss(200, 300), _gauss(300, 100), _gauss(150, 150), _gauss(200, 300, 6)]
    for i, v in ((1, 'nan'), (2, 'inf'), (5, 'inf'), (6, 'nan')):
        mats[i][3, 5] = float(v)
    out = orthogonalize(mats)
    for i in (0, 3, 4, 7):
        _check(out[i], mats[i])
    for i in (1, 2, 5, 6):
        assert torch.isnan(out[i]).all(), i


@pytest.mark.gpu
def test_strided_inputs_and_given_outputs():
    from mr3d_amd.core import orthogonalize
    big = _gauss(200, 300)
    for v in (big[10:90, 7:250], big.t(), big[::2, ::3], big[:, 5:6], big.t()[3:, 2:9]):
        _check(orthogonalize(v), v)
    g = _gauss(70, 140)
    ref = orthogonalize(g)
    o = torch.full((71, 140), 9.0, device='cuda')
    assert orthogonalize(g, out=o[:70]) is not None and torch.equal(o[:70], ref) and bool((o[70] == 9).all())
    h = g.clone()
    orthogonalize(h, out=h)
    assert torch.equal(h, ref)
    big = _gauss(200, 300)
    ref = orthogonalize(big)
    orthogonalize(big, out=big)
    assert torch.equal(big, ref)
    with pytest.raises(ValueError, match='overlaps'):
        orthogonalize([g, g], out=[o[:70], o[:70]])
    with pytest.raises(ValueError, match='overlaps'):
        orthogonalize([h, g], out=[o[:70], h])
    saved = _gauss(70, 140).requires_grad_(True)
    kept = (saved * o[:70]).sum()
    orthogonalize(g, out=o[:70])
    with pytest.raises(RuntimeError, match='inplace'):
        kept.backward()
    sq = _gauss(64, 64)
    with pytest.raises(ValueError, match='overlaps'):
        orthogonalize(sq.t(), out=sq)
    with pytest.raises(ValueError, match='contiguous'):
        orthogonalize(g, out=torch.empty(140, 70, device='cuda').t())


@pytest.mark.gpu
def test_other_stream_and_replayed_graph():
    from mr3d_amd.core import orthogonalize
    mats = [_gauss(64, 1728), _gauss(200, 100), _gauss(300, 2000)]
    ref = orthogonalize(mats)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = orthogonalize(mats)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = orthogonalize(mats)
    for k in range(3):
        for m in mats:
            m.copy_(torch.randn(m.shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        eager = orthogonalize(mats)
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_refusals_need_no_gpu():
    from abi import Matrix, lib
    from mr3d_amd.core import orthogonalize
    g = torch.zeros(4, 8)
    with pytest.raises(NotImplementedError):
        orthogonalize(g)
    with pytest.raises(TypeError):
        orthogonalize(torch.zeros(8))
    with pytest.raises(TypeError):
        orthogonalize([g, g.half()])
    for kw in (dict(steps=0), dict(steps=101), dict(eps=-1.0), dict(eps=float('nan')), dict(coefficients=(17, 0, 0)), dict(coefficients=(float('nan'), 0, 0))):
        with pytest.raises(ValueError):
            orthogonalize(g, **kw)
    with pytest.raises(NotImplementedError):
        orthogonalize(torch.zeros(1, 1).expand(1, (1 << 20) + 1))
    L = lib()
    mk = lambda **kw: (Matrix * 1)(Matrix(**{**dict(in_=256, out=256, rows=4, cols=8, in_row_stride=8, in_col_stride=1, dtype=0), **kw}))
    need = L.mr3d_orthogonalize_workspace_bytes(mk(), 1)
    call = lambda t, n=1, steps=5, a=1.0, eps=0.0, ws=256, by=need: L.mr3d_orthogonalize(t, n, steps, a, 0.0, 0.0, eps, ws, by, None)
    assert need > 0 and need % 256 == 0
    assert call(None) == 1 and call(mk(), 0) == 1 and call(mk(), steps=0) == 1 and call(mk(), a=17.0) == 1 and call(mk(), a=float('nan')) == 1
    assert call(mk(), eps=-1.0) == 1 and call(mk(in_=None)) == 1 and call(mk(rows=0)) == 1 and call(mk(cols=(1 << 20) + 1)) == 1
    assert call(mk(dtype=2)) == 4 and call(mk(), ws=None) == 2 and call(mk(), ws=128) == 2 and call(mk(), by=need - 1) == 2
    assert L.mr3d_orthogonalize_workspace_bytes(mk(dtype=2), 1) == 0
