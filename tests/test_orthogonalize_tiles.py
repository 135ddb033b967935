"""orthogonalize: the tiles and splits that large matrices and lists take.  What each list is here for is asserted from its shapes (on the host, without a GPU), so
that another estimate of the times cannot take a path out of the tests unseen; then the results are compared with 64 bits."""
import ctypes

import pytest
import torch

from abi import Matrix, lib
from test_orthogonalize import _reference


class Tiles(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int * 3) for n in ('width', 'whole', 'split', 'parts')]


def _tiles(shapes):
    fn = lib().mr3d_orthogonalize_tiles
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    a = (Matrix * len(shapes))(*[Matrix(rows=m, cols=n, in_row_stride=n, in_col_stride=1) for m, n in shapes])
    t = Tiles()
    assert fn(a, len(shapes), ctypes.byref(t)) == 0
    return [list(getattr(t, n)) for n in ('width', 'whole', 'split', 'parts')]


def _detector():
    """the weight matrices of a 50-layer backbone with a 16-channel stem, its four-level neck and the two shared layers of a bbox head"""
    out, cin = [(16, 3 * 343)], 16
    for stage, blocks in enumerate((3, 4, 6, 3)):
        planes = 16 * 2 ** stage
        for b in range(blocks):
            out += [(planes, cin), (planes, planes * 27), (planes * 4, planes)] + ([(planes * 4, cin)] if b == 0 else [])
            cin = planes * 4
    for c in (64, 128, 256, 512):
        out += [(64, c), (64, 64 * 27)]
    return out + [(1024, 64 * 3 * 7 * 7), (1024, 1024)]


# per product (Gram, square, apply): tile width, and whether tiles are computed whole, shared, or both (the leftovers of full rounds of workgroups)
LISTS = {
    'square_full_round_and_leftovers': ([(4096, 4096)], [(128, 'both'), (128, 'both'), (128, 'whole')]),
    'ragged_leftovers_everywhere': ([(4100, 4200)], [(128, 'both'), (128, 'both'), (128, 'both')]),
    'tall_leftovers_of_the_last_product': ([(2950, 2900)], [(128, 'whole'), (128, 'whole'), (128, 'both')]),
    'wide_tiles_whole': ([(2560, 2560)], [(128, 'whole'), (128, 'whole'), (128, 'whole')]),
    'long_axis': ([(1024, 9408)], [(128, 'shared'), (64, 'whole'), (128, 'both')]),
    'long_axis_odd': ([(2049, 5000)], [(128, 'shared'), (64, 'whole'), (128, 'both')]),
    'narrow_tiles_shared': ([(1000, 3000 + 1)], [(64, 'shared'), (64, 'whole'), (64, 'whole')]),
    'list_with_a_carrier': ([(1024, 9408), (200, 300), (512, 13824), (40, 50)], [(128, 'both'), (64, 'whole'), (128, 'both')]),
    'detector': (_detector(), [(128, 'both'), (64, 'whole'), (128, 'whole')]),
}


@pytest.mark.parametrize('name', LISTS)
def test_the_list_takes_its_path(name):
    shapes, want = LISTS[name]
    width, whole, split, parts = _tiles(shapes)
    for i, (w, how) in enumerate(want):
        got = 'both' if whole[i] and split[i] else 'shared' if split[i] else 'whole'
        assert (width[i], got) == (w, how), (i, width, whole, split, parts)
        assert (parts[i] > 1) == (split[i] > 0)


def test_refused_lists_have_no_tiles():
    fn = lib().mr3d_orthogonalize_tiles
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p]
    t, good = Tiles(), (Matrix * 1)(Matrix(rows=4, cols=8))
    assert fn(None, 1, ctypes.byref(t)) == 1 and fn(good, 0, ctypes.byref(t)) == 1 and fn(good, 1, None) == 1
    assert fn((Matrix * 1)(Matrix(rows=0, cols=8)), 1, ctypes.byref(t)) == 1
    assert fn((Matrix * 1)(Matrix(rows=4, cols=8, dtype=2)), 1, ctypes.byref(t)) == 4
    assert fn(good, 1, ctypes.byref(t)) == 0 and not any(t.whole) and not any(t.split)


def _matrix(m, n, k, dtype):
    """a decaying spectrum under noise, made on the GPU"""
    g = torch.Generator(device='cuda').manual_seed(1000 * m + n + k)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')
    q = max(1, min(m, n) // 8)
    return ((r(m, q) @ r(q, n)) * (1e-3 / q ** 0.5) + 5e-4 * r(m, n)).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('name', LISTS)
def test_against_64_bits(name, dtype):
    """norm-wise with the bound of test_orthogonalize; and tile by tile: every 64 x 64 block of the result, corner and edge blocks among them, with the error that
    the bound of the whole would let it have if spread evenly, times 8 -- a tile that is missing or in the wrong place is off by its own size"""
    from mr3d_amd.core import orthogonalize
    mats = [_matrix(m, n, k, dtype) for k, (m, n) in enumerate(LISTS[name][0])]
    outs = orthogonalize(mats)
    for g, o in zip(mats, outs):
        ref, tol = _reference(g)
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        err = (o.double() - ref).abs()
        assert float(err.norm()) <= tol + half * float(ref.norm()), (tuple(g.shape), float(err.norm()), tol)
        m, n = g.shape
        pad = torch.nn.functional.pad((err - half * ref.abs()).clamp(min=0), (0, -n % 64, 0, -m % 64))
        blocks = pad.view(pad.shape[0] // 64, 64, pad.shape[1] // 64, 64).square().sum((1, 3)).sqrt()
        assert float(blocks.max()) <= 8 * tol / blocks.numel() ** 0.5 + 2.0 ** -8 * half, (tuple(g.shape), float(blocks.max()))
    assert all(torch.equal(a, b) for a, b in zip(outs, orthogonalize(mats)))
