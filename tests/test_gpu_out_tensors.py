"""GPU: tensors that are handed over for the results."""
import pytest
import torch

from tests.test_gpu_int8 import DEV, FORWARD, _ready

pytestmark = pytest.mark.gpu


def test_results_into_given_tensors():
    layer, _ = _ready(FORWARD[0])
    T, H = 12, layer.H
    x = torch.randn(3, 4, H, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    norm = torch.ones(H, dtype=torch.bfloat16, device=DEV)
    lg = torch.randn(T, layer.E, device=DEV)
    calls = {"forward": lambda out: layer.forward(x, out=out), "logits": lambda out: layer.forward_from_logits(x, lg, out=out),
             "norm": lambda out: layer.rmsnorm(x, norm, out=out), "block": lambda out: layer.block_forward(x, norm, out=out)}
    wrong = [torch.zeros(T, H, device=DEV), torch.zeros(T - 1, H, dtype=torch.bfloat16, device=DEV),
             torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, 2 * H, dtype=torch.bfloat16, device=DEV)[:, ::2],
             torch.zeros(T, 2 * H, dtype=torch.bfloat16, device=DEV)[:, :H]]
    for name, call in calls.items():
        want = call(None)
        for shape in ((T, H), (3, 4, H)):
            out = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
            got = call(out)
            assert got.shape == x.shape and got.data_ptr() == out.data_ptr() and torch.equal(out.view(-1), want.view(-1)), name
        for bad in wrong:
            with pytest.raises(ValueError, match="out"):
                call(bad)
    layer.close()
