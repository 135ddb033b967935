"""Softmax cross entropy of a linear classifier over many classes (csrc/linear_ce.hip): `layers.linear` + `weighted_cross_entropy`
without the [rows, classes] logits between them."""
import torch

from ... import _hip


def linear_cross_entropy(x, weight, label, row_weight=None, bias=None, avg_factor=None, valid_rows=None, ignore_index=-100):
    """sum_i row_weight_i * cross_entropy(x_i @ weight.T + bias, label_i) / avg -> loss [1] (fp32), differentiable in x, weight and bias.

    x [..., K] and weight [C, K]: both fp32 or both bf16; bias [C] in their type or fp32; label [...] int64; row_weight [...] (None: 1).
    A row counts when its weight is not 0, its label is not ignore_index and it lies before valid_rows (a device int32 scalar: static
    shapes with padding).  The others take no part, whatever they hold, and get zero gradients.  avg_factor: a number, a device scalar, or None for
    max(number of counted rows with a positive weight, 1) (`weighted_cross_entropy` counts every positive weight, also of rows behind valid_rows:
    the same where those rows have weight 0, as the samplers leave them).  A counted label outside [0, C) makes the loss NaN.
    Beside copies of x and weight the memory is bounded (2 GiB of exponentials, rows go through in pieces).  fp32: products carry 22 bits of
    each factor, relative to the largest of its row (x, and g for dx), of its class (g for dW) or of all (weight, but classes
    whose bias is -1e30 or less).  bf16 gradients are rounded once more when the incoming gradient is no power of two.  One backward per call; under
    graph capture both are captured (as `torch.cuda.make_graphed_callables` does) or neither."""
    on_device = torch.is_tensor(avg_factor)
    return _hip.train_ops().linear_cross_entropy(x, weight, label, row_weight, bias, avg_factor if on_device else None,
                                                 None if on_device else avg_factor, valid_rows, ignore_index)
