"""GPU: infinities in the rows and in their gradients.  Each reaches what the formulas say, as an infinity of its sign where no other term makes a NaN
of it: s and gs have a second part beside their first, and zeros of it times an infinity are no part of the sum."""
import pytest
import torch

from tests.test_gpu_adapters import DEV, _adapters, _near, _realign, _reference, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


def _same(got, ref):
    """Infinities and NaN where the formula has them, the rest within the bounds."""
    want, tol = ref
    odd = ~want.isfinite()
    assert torch.equal(got.double()[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), want[odd].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))
    return bool(((got.double() - want).abs()[~odd] <= tol[~odd]).all())


@pytest.mark.parametrize("n,G", [(20, 3), (600, 3), (3000, 1), (3000, 200), (6000, 2)])
@pytest.mark.parametrize("r", (8, 12, 40, 128))
def test_infinities_of_rows_and_of_gradients(layer, n, G, r):
    """Of adapter 0 one row has an infinity in x, and another one in its gradient; in the sums over rows each meets finite s and gs."""
    K, N = 72, 40
    x, y, go = _rows(n, K, 1), _rows(n, N, 2), _rows(n, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    ids = (torch.arange(n, device=DEV) % G).int()
    clean = _reference(x, y, down, up, scale, ids, go)
    plan = layer.adapter_plan(ids, G)
    x, go = _realign(x), _realign(go)
    x[0, 5] = float("inf")
    x[2 * G, 9] = float("-inf")
    _, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
    gx, gd, gu = layer.adapter_grad(go, x, down, up, plan, scale, s)
    refs = _reference(x, y, down, up, scale, ids, go)
    assert _near(gx, clean[1])                                   # x is no part of it
    assert _same(gd, refs[2]) and gd[0, :, 5].isinf().all() and gd[0, :, 9].isinf().all() and gd.isfinite().sum() == gd.numel() - 2 * r
    assert _same(gu, refs[3]) and not gu[0].isfinite().any()

    x = _rows(n, K, 1)
    go[0, 7] = float("inf")
    _, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
    gx, gd, gu = layer.adapter_grad(go, x, down, up, plan, scale, s)
    refs = _reference(x, y, down, up, scale, ids, go)
    assert _same(gu, refs[3]) and gu[0, 7].isinf().all() and gu.isfinite().sum() == gu.numel() - r
    assert _same(gx, refs[1]) and not gx[0].isfinite().any() and gx[1:].isfinite().all()
    assert _same(gd, refs[2]) and not gd[0].isfinite().any()
