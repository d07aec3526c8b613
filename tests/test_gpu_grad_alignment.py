"""GPU: gradients as torch hands them over: contiguous views that begin anywhere (the backward of cat and of flat views cuts
them out of larger tensors)."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _layer, _setup

pytestmark = pytest.mark.gpu


def _off(t):
    """The same values in a contiguous view one element behind a 16-byte boundary."""
    v = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    assert v.is_contiguous() and v.data_ptr() % 16 != 0
    return v.copy_(t)


def test_a_gradient_that_is_cut_out_of_a_flat_tensor():
    from moe_gen_b200 import combine_rows, sort_rows
    T, k, H = 20, 2, 256
    layer, idx, counts, pad, dst, rows, live = _setup(T, 8, k, H)
    x = torch.randn(T, H, device=DEV).to(torch.bfloat16).requires_grad_(True)
    out = torch.randn(rows, H, device=DEV).to(torch.bfloat16).requires_grad_(True)
    w = torch.rand(T, k, device=DEV).requires_grad_(True)
    sh = torch.randn(T, H, device=DEV).to(torch.bfloat16).requires_grad_(True)
    one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
    for make, leaves, n in ((lambda: sort_rows(layer, x, dst, rows, counts, pad), [x], rows * H),
                            (lambda: combine_rows(layer, out, dst, idx, w, counts, pad, sh), [out, w, sh], T * H)):
        g = torch.randn(n, device=DEV).to(torch.bfloat16)
        want = torch.autograd.grad(make(), leaves, g.view(-1, H))
        got = torch.autograd.grad(torch.cat([one, make().reshape(-1)]), leaves, torch.cat([one, g]))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    layer.close()


@pytest.mark.parametrize("gating", (0, 2))
def test_logits_that_begin_off_a_boundary(gating):
    from moe_gen_b200 import route
    layer = _layer(E=64, k=6, gating=gating)
    if gating == 2:
        layer.bias = torch.zeros(64, device=DEV)
    lg = torch.randn(33, 64, device=DEV)
    g = torch.randn(33, 6, device=DEV)
    a, b = lg.clone().requires_grad_(True), _off(lg).requires_grad_(True)
    (ia, wa), (ib, wb) = route(layer, a), route(layer, b)
    assert torch.equal(ia, ib) and torch.equal(wa, wb)
    assert torch.equal(torch.autograd.grad(wa, a, g)[0], torch.autograd.grad(wb, b, _off(g))[0])
    layer.close()
