"""GPU: rows that reach the layer's products from torch are what the products take them for, or refused."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _setup

pytestmark = pytest.mark.gpu


def test_rows_of_another_type_or_width_are_refused():
    layer, idx, counts, pad, dst, rows, live = _setup(10, 8, 2, 256)
    layer.set_router(torch.zeros(8, 256))
    x = torch.zeros(10, 256, dtype=torch.bfloat16, device=DEV)
    perm = layer.permute_rows(x, dst, rows)
    for call, good in ((layer.gate_logits, x), (layer.gate_route, x), (layer.shared_ffn, x), (lambda t: layer.expert_ffn(t, pad, counts), perm)):
        for bad in (good.float(), good[:, :128].contiguous(), good.repeat(1, 2), good[:, ::2], good.view(-1), good.cpu()):
            with pytest.raises(ValueError):
                call(bad)
    for c, p in ((counts.long(), pad), (counts, pad.long()), (counts[:4].contiguous(), pad), (counts, pad[:-1].contiguous()),
                 (counts.cpu(), pad)):
        with pytest.raises(ValueError):
            layer.expert_ffn(perm, p, c)
    assert not layer.expert_ffn(perm, pad, counts)[1].any()
    layer.close()
