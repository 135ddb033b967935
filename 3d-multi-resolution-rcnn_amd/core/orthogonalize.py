"""Orthogonalised updates of weight matrices (csrc/ortho.hip); `dist_utils.ArenaMuon` steps a whole detector with them."""
import torch

from .. import _hip

COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # singular values from 1e-2 .. 1 to 0.7 .. 1.2 in five steps


def _matrix(t, i):
    if not torch.is_tensor(t) or t.dim() < 2:
        raise TypeError(f'orthogonalize: matrix {i} is a tensor of two or more axes')
    if t.dtype not in _hip.STORAGE_DTYPES:
        raise TypeError(f'orthogonalize: matrix {i} is float32 or bfloat16, got {t.dtype}')
    t = t.detach()
    return t if t.dim() == 2 else t.reshape(t.shape[0], -1)


def orthogonalize(mats, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """Newton-Schulz orthogonalisation of a matrix or a list of matrices (fp32 / bf16, on one GPU; a weight of more axes counts as
    [shape[0], rest]):  X = G / (|G|_F + eps), then `steps` times  X <- a X + (b A + c A A) X  with A = X X^T (X^T X where that is smaller).
    Returns X in G's shape and type; a list shares the launches of every stage, which is what makes small matrices cheap, and its
    results are views of one buffer per type.  out: contiguous tensors to write to (G itself is allowed).  Not differentiable."""
    single = torch.is_tensor(mats)
    given = [mats] if single else list(mats)
    flat = [_matrix(t, i) for i, t in enumerate(given)]
    a, b, c = (float(v) for v in coefficients)
    if not 1 <= int(steps) <= 100 or not float(eps) >= 0 or not all(-16 <= v <= 16 for v in (a, b, c)):
        raise ValueError('orthogonalize: 1 to 100 steps, eps at least 0, coefficients within 16')
    if any(max(t.shape) > 1 << 20 for t in flat):
        raise NotImplementedError('orthogonalize: up to 2^20 rows and columns')
    if any(t.device != flat[0].device for t in flat):
        raise ValueError('orthogonalize: the matrices of a list are on one device')
    if flat and not flat[0].is_cuda:
        raise NotImplementedError('orthogonalize has no CPU fallback')
    if out is None:
        outs = [None] * len(flat)
        for dt in {t.dtype for t in flat}:
            at = [i for i, t in enumerate(flat) if t.dtype == dt]
            sizes = [-(-flat[i].numel() // 64) * 64 for i in at]                  # every result starts on its own 128 bytes
            for i, buf in zip(at, torch.empty((sum(sizes),), dtype=dt, device=flat[0].device).split(sizes)):
                outs[i] = buf[:flat[i].numel()].view(given[i].shape)
    else:
        outs = [out] if torch.is_tensor(out) else list(out)
        if len(outs) != len(flat):
            raise ValueError('orthogonalize: one out per matrix')
        for g, o in zip(given, outs):
            if o.shape != g.shape or o.dtype != g.dtype or o.device != g.device or not o.is_contiguous():
                raise ValueError('orthogonalize: an out is contiguous and has its matrix\'s shape, type and device')
    work = [(t, o) for t, o in zip(flat, outs) if t.numel()]
    if work:
        _hip.orthogonalize([t for t, _ in work], [o.detach() for _, o in work], int(steps), (a, b, c), float(eps))
    return outs[0] if single else outs
