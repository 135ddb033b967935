"""The training operators together: a classification head over many classes -- linear, layer norm, linear cross entropy -- stepped by ArenaMuon
on a DetectorArena, against the same step in 64 bits; and ArenaMuon over the whole detector's arena."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
C = (3.4445, -4.7750, 2.0315)


class Head(nn.Module):
    """what a detector hands to train_step: forward_train -> losses, total_loss"""

    def __init__(self, features=96, hidden=64, classes=500):
        super().__init__()
        self.fc = nn.Linear(features, hidden)
        self.norm_weight = nn.Parameter(torch.ones(hidden))
        self.norm_bias = nn.Parameter(torch.zeros(hidden))
        self.fc_cls = nn.Linear(hidden, classes)
        self.unused = nn.Linear(32, 32)

    def forward_train(self, x, label, weight):
        from mr3d_amd.core import linear_cross_entropy
        from mr3d_amd.detector import layers
        h = layers.layer_norm(layers.linear(x, self.fc.weight, self.fc.bias, relu=True), self.norm_weight, self.norm_bias)
        return dict(loss_cls=linear_cross_entropy(h, self.fc_cls.weight, label, weight, bias=self.fc_cls.bias))

    @staticmethod
    def total_loss(losses):
        return sum(v.sum() for v in losses.values())


def _ns(g, steps=5):
    x = g / (g.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    for _ in range(steps):
        a = x @ x.t()
        x = C[0] * x + (C[1] * a + C[2] * a @ a) @ x
    return x.t() if tall else x


def _reference_grads(p, x, label, weight):
    leaves = {k: v.clone().requires_grad_(True) for k, v in p.items()}
    h = torch.relu(x @ leaves['fc.weight'].t() + leaves['fc.bias'])
    h = torch.nn.functional.layer_norm(h, h.shape[1:], leaves['norm_weight'], leaves['norm_bias'])
    z = h @ leaves['fc_cls.weight'].t() + leaves['fc_cls.bias']
    live = (label != -100) & (weight != 0)
    ce = torch.nn.functional.cross_entropy(z[live], label[live], reduction='none')
    ((ce * weight[live]).sum() / max(int((live & (weight > 0)).sum()), 1)).backward()
    return {k: v.grad for k, v in leaves.items()}


def test_head_gradients_and_steps_follow_the_formulas():
    """Gradients: every operator alone is within about 1e-5 of 64 bits (their own tests), the fp32 linear layer within 1e-4 of the largest value
    (tests/test_gpu_heads.py), and these compose with factors of a few: 1e-3 in norm.  The update of a matrix is a function of its gradient
    whose slope is at most a^5 = 485 in the directions of the smallest singular values and below 10 in those that make up its norm: 1e-2
    of the update in norm, and the same of the parameters' change."""
    from mr3d_amd.dist_utils import ArenaMuon, DetectorArena, train_step
    torch.manual_seed(0)
    det = Head().cuda()
    start = {k: v.detach().double().cpu().clone() for k, v in det.named_parameters()}
    arena = DetectorArena(det, engine_attr=None)
    opt = ArenaMuon(arena, lr=0.02, momentum=0.9, weight_decay=0.1, other_lr=0.5)
    assert [tuple(m.shape) for m in opt._mats] == [(64, 96), (500, 64), (32, 32)]
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(200, 96, generator=gen)
    label = torch.randint(0, 500, (200,), generator=gen)
    label[::7] = -100
    weight = 0.5 + torch.rand(200, generator=gen)
    batch = ((x.cuda(), label.cuda(), weight.cuda()), {})
    p = {k: v.clone() for k, v in start.items() if not k.startswith('unused')}
    v = {k: torch.zeros_like(t) for k, t in p.items()}
    for it in range(3):
        # each step is compared from the parameters that it started from
        p = {k: t.detach().double().cpu().clone() for k, t in det.named_parameters() if k in p}
        grads = _reference_grads(p, x.double(), label, weight.double())
        train_step(det, arena, opt, batch, world_size=1, grad_clip=None)
        now = dict(det.named_parameters())
        for k, g in grads.items():
            got = now[k].grad.double().cpu()
            assert float((got - g).norm()) <= 1e-3 * float(g.norm()), (it, k)
            v[k] = 0.9 * v[k] + got
            d = got + 0.9 * v[k]
            if d.dim() > 1:
                want = -0.02 * (max(1, d.shape[0] / d.shape[1]) ** 0.5 * _ns(d) + 0.1 * p[k])
            else:
                want = -0.02 * (0.5 * d + 0.1 * p[k])
            change = now[k].detach().double().cpu() - p[k]
            assert float((change - want).norm()) <= 1e-2 * float(want.norm()) + 2.0 ** -23 * float(p[k].norm()), (it, k)
    assert torch.equal(det.unused.weight.detach().double().cpu(), start['unused.weight'])           # never received a gradient
    saved = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state_dict().items()}
    opt.momentum_buffer.zero_()
    opt.load_state_dict(saved)
    assert torch.equal(opt.momentum_buffer, saved['momentum_buffer']) and float(opt.momentum_buffer.norm()) > 0


def test_training_runs_and_is_reproducible():
    """five steps twice from the same start: the same bits (every operator sums in a fixed order)"""
    from mr3d_amd.dist_utils import ArenaMuon, DetectorArena, train_step
    out = []
    for _ in range(2):
        torch.manual_seed(4)
        det = Head().cuda()
        arena = DetectorArena(det, engine_attr=None)
        opt = ArenaMuon(arena, lr=0.02)
        gen = torch.Generator().manual_seed(2)
        for _ in range(5):
            x = torch.randn(64, 96, generator=gen).cuda()
            label = torch.randint(0, 500, (64,), generator=gen).cuda()
            total, _ = train_step(det, arena, opt, ((x, label, torch.ones(64).cuda()), {}), world_size=1)
            assert torch.isfinite(total)
        out.append(arena.flat_params.detach().clone())
    assert torch.equal(*out)


def test_arena_of_a_detector_lists_its_matrices():
    from mr3d_amd.detector import ExtractFeat3D
    from mr3d_amd.dist_utils import ArenaMuon, DetectorArena

    class Det(nn.Module):
        def __init__(self):
            super().__init__()
            self.extract = ExtractFeat3D(device='cuda')
            self.head = nn.Linear(64, 2).cuda()

    det = Det()
    arena = DetectorArena(det)
    mats = arena.matrices()
    assert (arena.engine.num_trainable, (2, 64)) in mats and len(mats) == len(arena.engine.specs) + 1
    for off, shape in mats[:-1]:
        n = 1
        for k in shape:
            n *= k
        assert off + n <= arena.engine.num_trainable
    opt = ArenaMuon(arena, lr=0.01)
    g = torch.Generator(device='cuda').manual_seed(0)
    before = arena.flat_params.clone()
    arena.flat_grads.copy_(torch.randn(arena.flat_grads.shape, generator=g, device='cuda') * 1e-3)
    arena.engine.grads_touched = True
    arena.heads._touch(0)
    arena.heads._touch(1)
    grads = arena.flat_grads.clone()
    opt.step()
    for off, shape in mats[:-1:9]:
        n = 1
        for k in shape:
            n *= k
        d = (grads[off:off + n].double() * (1 + 0.95)).view(shape[0], -1)
        want = -0.01 * max(1, shape[0] ** 2 / n) ** 0.5 * _ns(d)
        got = (arena.flat_params[off:off + n].double() - before[off:off + n].double()).view(shape[0], -1)
        # the change is read off parameters of size up to 1: half a step of those, twice
        assert float((got - want).norm()) <= 1e-4 * float(want.norm()) + 2.0 ** -23 * float(before[off:off + n].norm()), shape
