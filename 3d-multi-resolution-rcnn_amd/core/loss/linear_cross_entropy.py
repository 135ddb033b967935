"""Softmax cross entropy of a linear classifier over many classes (csrc/linear_ce.hip): `layers.linear` + `weighted_cross_entropy`
without the [rows, classes] logits between them."""
import torch
from torch.autograd.function import once_differentiable

from ... import _hip


def _rows(t):
    """[rows, k] with a contiguous last axis and rows that do not overlap: a view where the strides allow it, else a copy"""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


class _LinearCrossEntropyFn(torch.autograd.Function):
    """the forward call leaves the gradients too; backward multiplies them by the incoming one, in place and once"""

    @staticmethod
    def forward(ctx, x, weight, bias, run):
        want = ctx.needs_input_grad[:3]
        ctx.shape = x.shape
        loss, *ctx.grads = run(x.detach(), weight.detach(), None if bias is None else bias.detach(), want)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if ctx.grads is None:
            raise RuntimeError('linear_cross_entropy: a second backward through the same loss (its gradients were handed over by the first); '
                               'call linear_cross_entropy again')
        g = g.float().contiguous()
        dx, dw, db = (t if t is None or t.numel() == 0 else _hip.scale_by(t, g) for t in ctx.grads)
        ctx.grads = None
        return (None if dx is None else dx.reshape(ctx.shape)), dw, db, None


def linear_cross_entropy(x, weight, label, row_weight=None, bias=None, avg_factor=None, valid_rows=None, ignore_index=-100):
    """sum_i row_weight_i * cross_entropy(x_i @ weight.T + bias, label_i) / avg -> loss [1] (fp32), differentiable in x, weight and bias.

    x [..., K] and weight [C, K]: both fp32 or both bf16; bias [C] in their type or fp32; label [...] int64; row_weight [...] (None: 1).
    A row counts when its weight is not 0, its label is not ignore_index and it lies before valid_rows (a device int32 scalar: static
    shapes with padding).  The others take no part, whatever they hold, and get zero gradients.  avg_factor: a number, a device scalar, or None for
    max(number of counted rows with a positive weight, 1), as `weighted_cross_entropy` divides.  A counted label outside [0, C) makes the loss NaN.
    The memory beside the gradients is bounded (2 GiB of exponentials, rows go through in pieces).  fp32: products carry 22 bits of
    each factor.  One backward per call."""
    if not torch.is_tensor(x) or x.dim() < 1 or not torch.is_tensor(weight) or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError('linear_cross_entropy: x is [..., K] and weight [C, K]')
    if x.dtype not in _hip.STORAGE_DTYPES or weight.dtype != x.dtype:
        raise TypeError(f'linear_cross_entropy: x and weight are both float32 or both bfloat16, got {x.dtype} and {weight.dtype}')
    classes, k = weight.shape
    if not 1 <= classes <= 1 << 20 or not 1 <= k <= 1 << 16 or x.numel() // max(k, 1) > 1 << 22:
        raise NotImplementedError('linear_cross_entropy: 1 to 2^20 classes, 1 to 2^16 features, up to 2^22 rows')
    if bias is not None and (tuple(bias.shape) != (classes,) or bias.dtype not in (torch.float32, x.dtype)):
        raise ValueError(f'linear_cross_entropy: bias is [{classes}], float32 or {x.dtype}')
    if label.shape != x.shape[:-1] or label.dtype != torch.int64:
        raise ValueError(f'linear_cross_entropy: label is {tuple(x.shape[:-1])}, int64')
    if row_weight is not None:
        if row_weight.shape != label.shape:
            raise ValueError(f'linear_cross_entropy: row_weight is {tuple(label.shape)}')
        if row_weight.requires_grad:
            raise NotImplementedError('linear_cross_entropy is not differentiable in row_weight')
        row_weight = row_weight.reshape(-1).float().contiguous()
    if torch.is_tensor(avg_factor):
        if avg_factor.numel() != 1 or avg_factor.device != x.device:
            raise ValueError('linear_cross_entropy: avg_factor is a number or one value on the device of x')
        avg_factor = avg_factor.detach().float().reshape(1)
    elif avg_factor is not None:
        avg_factor = float(avg_factor)
        if not avg_factor > 0:
            raise ValueError(f'linear_cross_entropy: avg_factor is positive, got {avg_factor}')
    if valid_rows is not None and (valid_rows.numel() != 1 or valid_rows.dtype != torch.int32):
        raise ValueError('linear_cross_entropy: valid_rows is one int32 value on the device')
    for t in (weight, bias, label, row_weight, valid_rows):
        if t is not None and t.device != x.device:
            raise ValueError('linear_cross_entropy: all tensors are on one device')
    if not x.is_cuda:
        raise NotImplementedError('linear_cross_entropy has no CPU fallback')
    label = label.reshape(-1).contiguous()

    def run(x, weight, bias, want):
        if label.numel() == 0:
            return [torch.zeros((1,), dtype=torch.float32, device=x.device)] + [torch.zeros_like(t) if w else None for t, w in zip((x, weight, bias), want)]
        return _hip.linear_cross_entropy(_rows(x.reshape(-1, k)), _rows(weight), None if bias is None else bias.contiguous(), label, row_weight,
                                         avg_factor, valid_rows, int(ignore_index), *want)

    return _LinearCrossEntropyFn.apply(x, weight, bias, run)
