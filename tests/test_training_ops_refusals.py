"""What layer_norm, linear_cross_entropy and orthogonalize refuse because they would answer it wrongly: forward-mode tangents, traces, function
transforms, views whose sign is kept outside of their memory.  All of it is refused before the device is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def _calls():
    from mr3d_amd.core import linear_cross_entropy, orthogonalize
    from mr3d_amd.detector.layers import layer_norm
    w, lab = torch.ones(5, 8), torch.zeros(4, dtype=torch.int64)
    return [lambda t: layer_norm(t), lambda t: layer_norm(torch.zeros(4, 8), t[0]), lambda t: linear_cross_entropy(t, w, lab),
            lambda t: linear_cross_entropy(torch.zeros(4, 8), t, lab), lambda t: linear_cross_entropy(torch.zeros(4, 8), w, lab, avg_factor=t[0, :1]),
            lambda t: orthogonalize(t), lambda t: orthogonalize([w, t]), lambda t: orthogonalize(torch.zeros(4, 8), out=t)]


@pytest.mark.parametrize('which', range(8))
def test_tangents_traces_transforms_and_negated_views(which):
    call = _calls()[which]
    x = torch.zeros(4, 8)
    with fwad.dual_level():
        for dual in (fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(x.clone().requires_grad_(True), torch.ones_like(x))):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call(dual)
    with pytest.raises(NotImplementedError, match='trace'):
        torch.jit.trace(call, x)
    with pytest.raises(NotImplementedError, match='transforms'):
        torch.vmap(call)(x.expand(3, 4, 8))
    with pytest.raises(NotImplementedError, match='negated'):
        call(torch.conj(torch.zeros(4, 8, dtype=torch.complex64)).imag)
    with pytest.raises(NotImplementedError, match='no CPU fallback'):
        call(x)


def test_function_gradient_and_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from mr3d_amd.detector.layers import layer_norm
    with pytest.raises(NotImplementedError, match='transforms'):
        torch.func.grad(lambda t: layer_norm(t).sum())(torch.zeros(4, 8))
    with FakeTensorMode():
        with pytest.raises(NotImplementedError, match='transforms'):
            layer_norm(torch.empty(4, 8, device='cuda'))
    with pytest.raises(NotImplementedError, match='dense'):
        layer_norm(torch.zeros(4, 8).to_sparse())


@pytest.mark.gpu
def test_incoming_gradients_are_held_to_the_same():
    from mr3d_amd.core import linear_cross_entropy
    from mr3d_amd.detector.layers import layer_norm
    x = torch.randn(4, 8, device='cuda', requires_grad=True)
    y = layer_norm(x)
    with pytest.raises(RuntimeError, match='transforms'):
        torch.autograd.grad(y, x, torch.ones(3, 4, 8, device='cuda'), is_grads_batched=True, retain_graph=True)
    with fwad.dual_level():
        dual = fwad.make_dual(torch.ones(4, 8, device='cuda'), torch.ones(4, 8, device='cuda'))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.autograd.grad(y, x, dual, retain_graph=True)
    with pytest.raises(NotImplementedError, match='negated'):
        torch.autograd.grad(y, x, torch.conj(torch.zeros(4, 8, dtype=torch.complex64, device='cuda')).imag, retain_graph=True)
    loss = linear_cross_entropy(x, torch.randn(5, 8, device='cuda'), torch.zeros(4, dtype=torch.int64, device='cuda'))
    with fwad.dual_level():
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.autograd.grad(loss, x, fwad.make_dual(torch.ones(1, device='cuda'), torch.ones(1, device='cuda')), retain_graph=True)
    # refused calls leave the node as it was
    assert torch.isfinite(torch.autograd.grad(loss, x)[0]).all() and torch.isfinite(torch.autograd.grad(y, x, torch.ones_like(y))[0]).all()
