"""ArenaMuon's treatment of parameters that have never received a gradient (dist_utils.py), on the CPU: an arena without matrices calls no kernel."""
import torch
import torch.nn as nn


class _Two(nn.Module):
    def __init__(self):
        super().__init__()
        self.used, self.late = nn.Linear(3, 2), nn.Linear(3, 2)


def _arena():
    from mr3d_amd.dist_utils import ArenaMuon, DetectorArena
    torch.manual_seed(0)
    net = _Two()
    arena = DetectorArena(net, engine_attr=None)
    return net, arena, ArenaMuon(arena, lr=0.1, momentum=0.5, weight_decay=0.01, other_lr=1.0, min_rows=1 << 30)


def test_a_foreign_write_to_an_untouched_gradient_leaves_no_momentum():
    net, arena, opt = _arena()
    assert opt._mats == []
    start = net.late.weight.detach().clone()
    for _ in range(3):
        arena.zero_grad()
        net.used(torch.ones(1, 3)).sum().backward()
        for lo, hi in arena.untouched_ranges():
            arena.flat_grads[lo:hi] = 7.0
        opt.step()
    assert len(arena.untouched_ranges()) == 2 and torch.equal(net.late.weight.detach(), start)
    for lo, hi in arena.untouched_ranges():
        assert not opt.momentum_buffer[lo:hi].any()
    # the first gradient: v = grad, d = grad + momentum v, and nothing of what was written before.  Every product and sum below is exact but the
    # update itself, three roundings of values below 1
    arena.zero_grad()
    net.late(torch.ones(1, 3)).sum().backward()
    opt.step()
    want = start.double() * (1 - 0.1 * 0.01) - 0.1 * 1.5
    assert float((net.late.weight.detach().double() - want).abs().max()) <= 4 * 2.0 ** -24
