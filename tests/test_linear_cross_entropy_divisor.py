"""What linear_cross_entropy divides by, beside weighted_cross_entropy: rows that do not count are not in its divisor, whatever their weight."""
import pytest
import torch


@pytest.mark.gpu
def test_padding_rows_of_positive_weight():
    """Both losses sum the same rows; weighted_cross_entropy divides by all positive weights, this one by the counted ones, or by avg_factor.  Each is good to some
    2^-18 (fp32 products of 64 features, logits of size 2, a mean over rows)."""
    from mr3d_amd.core import linear_cross_entropy, weighted_cross_entropy
    from mr3d_amd.detector import layers
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g).cuda() for s in ((60, 64), (40, 64), (40,)))
    w = w / 4
    label = torch.randint(0, 40, (60,), generator=g).cuda()
    rw = (0.5 + torch.rand(60, generator=g)).cuda()
    rw[::4] = 0
    valid = torch.tensor([37], dtype=torch.int32, device='cuda')
    counted, positive = int((rw[:37] > 0).sum()), int((rw > 0).sum())
    assert counted < positive
    beside = float(weighted_cross_entropy(layers.linear(x, w, b), label, rw, valid_rows=valid))
    own = float(linear_cross_entropy(x, w, label, rw, b, valid_rows=valid))
    given = float(linear_cross_entropy(x, w, label, rw, b, valid_rows=valid, avg_factor=float(positive)))
    assert abs(given - beside) <= 2.0 ** -17 * beside
    assert abs(own - beside * positive / counted) <= 2.0 ** -17 * own
    # padding of weight 0: the same divisor
    rw[37:] = 0
    beside = float(weighted_cross_entropy(layers.linear(x, w, b), label, rw, valid_rows=valid))
    assert abs(float(linear_cross_entropy(x, w, label, rw, b, valid_rows=valid)) - beside) <= 2.0 ** -17 * beside
    # ignored rows are not in it either
    label[3] = -100
    counted = int(((rw > 0) & (label != -100)).sum())
    own, given = (float(linear_cross_entropy(x, w, label, rw, b, avg_factor=a)) for a in (None, float(counted)))
    assert own == given
