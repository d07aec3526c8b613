"""GPU: the calibration step around int8 experts captured as a whole, forward and backward, and run on two streams at once."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _calibration, _step

pytestmark = pytest.mark.gpu


def _eager(layer, tensors, target, fns):
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    loss, _ = _step(layer, *leaves, target, fns)
    return [loss.detach()] + [g.clone() for g in torch.autograd.grad(loss, leaves)]


def test_a_captured_step_is_the_eager_one():
    layer, x, gate, adapter, target, fns = _calibration(True)
    held = [t.clone().requires_grad_(True) for t in (x, gate, adapter)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss, _ = _step(layer, *held, target, fns)
        torch.autograd.grad(loss, held)
        del loss                                                    # torch captures no backward beside a living eager graph of the leaves
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = _step(layer, *held, target, fns)
        grads = torch.autograd.grad(loss, held)
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        new = [torch.randn(t.shape, generator=g).mul(t.detach().float().std().item()).to(t.dtype).to(DEV) for t in held]
        with torch.no_grad():
            for h, n in zip(held, new):
                h.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.detach().clone()] + [t.clone() for t in grads]
        want = _eager(layer, new, target, fns)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    layer.close()


def test_steps_on_two_streams():
    layer, x, gate, adapter, target, fns = _calibration(True)
    want = _eager(layer, (x, gate, adapter), target, fns)
    other = [x.flip(0).contiguous(), gate, adapter]
    want2 = _eager(layer, other, target, fns)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, t in enumerate(((x, gate, adapter), other)):
            with torch.cuda.stream(streams[i]):
                got[i].append(_eager(layer, t, target, fns))
    torch.cuda.synchronize()
    for run, ref in zip(got, (want, want2)):
        assert all(torch.equal(a, b) for r in run for a, b in zip(r, ref))
    layer.close()
