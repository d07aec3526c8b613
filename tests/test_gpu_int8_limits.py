"""GPU: 8-bit integer rows and products at the ends of what they take, compared bit for bit with the restatements of
test_gpu_int8."""

import pytest
import torch

from tests.test_gpu_int8 import DEV, _check_mlp, _layer, _load, _staged

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ inner sizes beyond what a block keeps in registers
@pytest.mark.parametrize("inter,T", [(16384, 9), (16512, 1), (16512, 9), (16512, 700), (20480, 130)])
def test_experts_of_large_inner_size(inter, T):
    """Rows between the products of more than 16384 elements, some experts empty, rows of no pick left alone."""
    layer = _layer(E=4, k=2, H=256, I=inter)
    mats = _load(layer, inter + T)
    g = torch.Generator().manual_seed(T)
    x = (torch.randn(T, 256, generator=g) * 0.05).to(torch.bfloat16).to(DEV)
    idx = (torch.rand(T, 4, generator=g) + torch.tensor([1.0, 0.5, 0.0, -2.0])).topk(2, dim=1)[1].int().to(DEV)
    counts, _, pad, dst = layer.permute_plan(idx)
    xq, xs = layer.quantize_rows(x)
    pq, ps = layer.permute_rows_int8(xq, xs, dst, layer.padded_rows(T * 2))
    h, out = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    c, p = counts.cpu().tolist(), pad.cpu().tolist()
    for e in range(4):
        r = slice(p[e], p[e] + c[e])
        if c[e]:
            _check_mlp(pq[r].cpu().long(), ps[r].cpu(), mats[e], h[r].cpu(), out[r].cpu())
    flat = torch.zeros(out.shape[0], dtype=torch.bool, device=DEV)
    flat[dst.reshape(-1).long()] = True
    assert not out[~flat].any()
    logits = torch.randn(T, 4, generator=g).to(DEV)
    y = layer.forward_from_logits(x, logits)
    idx, w = layer.route_topk(logits)
    counts, _, pad, dst = layer.permute_plan(idx)
    pq, ps = layer.permute_rows_int8(xq, xs, dst, layer.padded_rows(T * 2))
    assert torch.equal(y, layer.combine(layer.expert_ffn_int8(pq, ps, pad, counts, dst)[1], dst, idx, w))
    layer.close()


@pytest.mark.parametrize("T", (5, 129))
def test_a_layer_of_large_hidden_size(T):
    """Tokens of more than 16384 elements: quantised by the plan that copies the rows up to 128 tokens, by rows beyond."""
    layer = _layer(E=4, k=2, H=16640, I=128, Is=128)
    _load(layer, T)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, 16640, generator=g).to(torch.bfloat16).to(DEV)
    logits = torch.randn(T, 4, generator=g).to(DEV)
    y = layer.forward_from_logits(x, logits)
    assert torch.equal(y, _staged(layer, x, logits)) and layer.device_status() == (0, 0)
    layer.close()
