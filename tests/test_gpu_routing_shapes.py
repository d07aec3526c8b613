"""GPU: logits and picks of other layers' shapes, whose rows the kernels would read past, are refused."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(10, 16), (10, 4), (80,), (2, 5, 8)])
def test_logits_of_another_shape(shape):
    from moe_gen_b200 import route
    layer = _layer(E=8, k=2)
    for call in (layer.route_topk, lambda t: route(layer, t)):
        with pytest.raises(ValueError, match="logits"):
            call(torch.zeros(shape, device=DEV))
    layer.close()


@pytest.mark.parametrize("shape", [(10, 4), (10, 1), (20,), (2, 5, 2)])
def test_picks_of_another_shape(shape):
    layer = _layer(E=8, k=2)
    with pytest.raises(ValueError, match="topk_idx"):
        layer.permute_plan(torch.zeros(shape, dtype=torch.int32, device=DEV))
    layer.close()
