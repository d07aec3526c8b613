"""GPU: what the differentiable calls refuse before their forward pass, because their backward pass could not follow."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


@pytest.mark.parametrize("with_residual", (True, False))
def test_rows_longer_than_the_norms_gradient_takes(layer, with_residual):
    from moe_gen_b200 import add_norm
    for cols in (16384, 16385, 20000):
        rows = [torch.randn(2, cols, device=DEV).to(torch.bfloat16) for _ in range(2)]
        w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
        res = rows[1] if with_residual else None
        want = layer.add_rmsnorm(rows[0], res, w)
        frozen = add_norm(layer, rows[0], res, w)                       # nothing to differentiate: any length
        assert torch.equal(frozen[1], want[0]) and torch.equal(frozen[0], want[1])
        for k in range(3):
            leaves = [rows[0].clone(), None if res is None else res.clone(), w.clone()]
            if leaves[k] is None:
                continue
            leaves[k].requires_grad_(True)
            with torch.no_grad():
                assert torch.equal(add_norm(layer, *leaves)[1], want[0])
            if cols <= 16384:
                h, y = add_norm(layer, *leaves)
                assert torch.autograd.grad(y.float().sum(), leaves[k])[0].isfinite().all()
            else:
                with pytest.raises(ValueError, match="16384"):
                    add_norm(layer, *leaves)


def test_adapters_of_rows_without_a_plan(layer):
    """Ids that change between the passes would give another batch's gradients: a plan is made once and only read."""
    from moe_gen_b200 import adapt_rows
    g = torch.Generator(device=DEV).manual_seed(1)
    x, y, down, up = (torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16) for s in ((40, 64), (40, 32), (3, 16, 64), (3, 32, 16)))
    ids = torch.randint(-1, 3, (40,), generator=g, device=DEV, dtype=torch.int32)
    plan = layer.adapter_plan(ids, 3)
    for frozen in (True, False):
        leaf = x.clone().requires_grad_(not frozen)
        with pytest.raises(ValueError, match="plan"):
            adapt_rows(layer, y, leaf, down, up, ids, 0.5)
    out, s = layer.adapter_add(y, x, down, up, plan, 0.5, keep=True)
    want = layer.adapter_grad(y, x, down, up, plan, 0.5, s)
    got = adapt_rows(layer, y, leaf, down, up, plan, 0.5)
    ids.fill_(1)
    assert torch.equal(got, out) and torch.equal(torch.autograd.grad(got, leaf, y)[0], want[0])
