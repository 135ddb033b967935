"""Orthogonalised updates of weight matrices (csrc/ortho.hip); `dist_utils.ArenaMuon` steps a whole detector with them."""
import torch

from .. import _hip

COEFFICIENTS = (3.4445, -4.7750, 2.0315)      # singular values from 1e-2 .. 1 to 0.7 .. 1.2 in five steps


def orthogonalize(mats, steps=5, coefficients=COEFFICIENTS, eps=1e-7, out=None):
    """Newton-Schulz orthogonalisation of a matrix or a list of matrices (fp32 / bf16, on one GPU; a weight of more axes counts as
    [shape[0], rest]):  X = G / (|G|_F + eps), then `steps` times  X <- a X + (b A + c A A) X  with A = X X^T (X^T X where that is smaller).
    Returns X in G's shape and type; a list shares the launches of every stage, which is what makes small matrices cheap, and its
    results are views of one buffer per type.  out: contiguous tensors to write to (G itself is allowed, another overlap with a matrix or an out is not).  Not differentiable."""
    single = torch.is_tensor(mats)
    a, b, c = coefficients
    if out is not None and torch.is_tensor(out):
        out = [out]
    res = _hip.train_ops().orthogonalize([mats] if single else list(mats), steps, a, b, c, eps, out)
    return res[0] if single else res
