"""GPU: a batch without tokens through the steps around the experts, forward and backward."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gating,combine", [(0, 0), (1, 1), (2, 0), (3, 2)])
def test_the_chain_of_no_tokens(gating, combine):
    from moe_gen_b200 import combine_rows, route, sort_rows
    E, k, H = 8, 2, 256
    layer = _layer(E=E, k=k, H=H, gating=gating, n_group=4, topk_group=2, norm=True, combine=combine)
    layer.bias = torch.zeros(E, device=DEV) if gating == 2 else None
    logits = torch.zeros(0, E, device=DEV, requires_grad=True)
    x = torch.zeros(0, H, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    shared = torch.zeros(0, H, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    idx, w = route(layer, logits)
    assert idx.shape == (0, k) and w.shape == (0, k)
    counts, offsets, pad, dst = layer.permute_plan(idx)
    assert dst.shape == (0, k) and not counts.any() and not offsets.any() and not pad.any()
    for n in (layer.padded_rows(0), 0):
        rows = sort_rows(layer, x, dst, n, counts, pad)
        assert rows.shape == (n, H) and not rows.any() and not layer.permute_rows(x.detach(), dst, n).any()
        y = combine_rows(layer, rows, dst, idx, w, counts, pad, shared)
        assert y.shape == (0, H)
        got = torch.autograd.grad(y.float().sum(), (logits, x, shared), retain_graph=True)
        assert [g.shape for g in got] == [(0, E), (0, H), (0, H)]
        out = torch.ones(n, H, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        assert not torch.autograd.grad(combine_rows(layer, out, dst, idx, w, counts, pad).float().sum(), out)[0].any()
    torch.cuda.synchronize()
    assert layer.device_status() == (0, 0)
    layer.close()
