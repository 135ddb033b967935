"""layer_norm, linear_cross_entropy and orthogonalize called side by side: on two streams, from two threads, in two graphs replayed in turn, with results that a
caller keeps.  Every answer has the bits of the same call made alone."""
import threading

import pytest
import torch


def _data(seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(700, 520, generator=g).to(dtype).cuda()
    lw = (1 + 0.1 * torch.randn(520, generator=g)).to(dtype).cuda()
    w = (torch.randn(3001, 520, generator=g) / 20).to(dtype).cuda()
    b = torch.randn(3001, generator=g).to(dtype).cuda()
    label = torch.randint(0, 3001, (700,), generator=g).cuda()
    label[::6] = -100
    return [x, lw, w, b, label]


def _step(s):
    from mr3d_amd.core import linear_cross_entropy, orthogonalize
    from mr3d_amd.detector.layers import layer_norm
    x, lw, w, b, label = s
    leaves = [t.detach().requires_grad_(True) for t in (x, lw, w, b)]
    h = layer_norm(leaves[0], leaves[1])
    loss = linear_cross_entropy(h, leaves[2], label, bias=leaves[3])
    grads = torch.autograd.grad(loss, leaves)
    return [loss.detach(), *grads, *orthogonalize([grads[0], grads[2], grads[2][:40]])]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_streams(dtype):
    data = [_data(k, dtype) for k in range(2)]
    alone = [_step(s) for s in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    kept = [[], []]
    for _ in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                kept[k].append(_step(data[k]))
    torch.cuda.synchronize()
    assert all(_same(r, alone[k]) for k in range(2) for r in kept[k])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_threads(dtype):
    data = [_data(k, dtype) for k in range(2)]
    alone = [_step(s) for s in data]
    torch.cuda.synchronize()
    out, errors = [[], []], []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(4):
                    out[k].append(_step(data[k]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                               # shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(len(out[k]) == 4 and all(_same(r, alone[k]) for r in out[k]) for k in range(2))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_graphs_in_turn(dtype):
    """replays of two graphs alternate with each other and with eager calls on changed inputs"""
    data = [_data(k, dtype) for k in range(2)]
    for s in data:
        _step(s)
    torch.cuda.synchronize()
    graphs, held = [], []
    for s in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(_step(s))
        graphs.append(g)
    for turn in range(3):
        for k in (0, 1) if turn % 2 else (1, 0):
            fresh = _data(10 * turn + k, dtype)
            for t, f in zip(data[k], fresh):
                t.copy_(f)
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert _same(held[k], _step(data[k])), (turn, k)
