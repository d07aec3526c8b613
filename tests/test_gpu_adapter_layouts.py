"""GPU: contiguous adapters whose rows begin off 16-byte boundaries, by their rank, their width or their address: the same bits as for views of
rows that lie on them."""
import pytest
import torch

from tests.test_gpu_adapters import DEV, _adapters, _ids, _near, _reference, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


def _whole_at(t, off):
    """t's numbers one behind another, from `off` elements behind a boundary on."""
    flat = torch.full((t.numel() + off + 8,), float("nan"), dtype=t.dtype, device=DEV)
    return flat[off:off + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("n", (1, 40, 700))
@pytest.mark.parametrize("K,N,r,G", [(64, 72, 4, 3), (64, 72, 12, 3), (136, 64, 100, 2), (128, 128, 1, 5), (100, 33, 16, 4), (101, 1, 7, 1), (8, 64, 16, 3)])
@pytest.mark.parametrize("off", (0, 1, 4))
def test_contiguous_adapters(layer, n, K, N, r, G, off):
    x, y, go = _rows(n, K, 1), _rows(n, N, 2), _rows(n, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    ids = _ids(n, G, 5)
    d, u = _whole_at(down, off), _whole_at(up, off)
    assert d.is_contiguous() and u.is_contiguous()
    for who in (ids, layer.adapter_plan(ids, G)):
        want = layer.adapter_add(y, x, down, up, who, scale, keep=True)
        got = layer.adapter_add(y, x, d, u, who, scale, keep=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and _near(got[0], _reference(x, y, down, up, scale, ids)[0])
        grads = layer.adapter_grad(go, x, d, u, who, scale, got[1])
        assert all(torch.equal(a, b) for a, b in zip(grads, layer.adapter_grad(go, x, down, up, who, scale, want[1])))


def test_the_copies_live_as_long_as_the_call_needs_them(layer):
    """Results of the copies' own sizes: an allocation behind the copy must not get its memory."""
    n, K, N, r, G = 256, 96, 104, 12, 16                   # down's copy: 36864 bytes, up's 53248 bytes, as are those of n rows of N
    x, y = _rows(n, K, 1), _rows(n, N, 2)
    down, up, scale = _adapters(G, r, K, N, 4)
    d, u, ids = down.contiguous(), up.contiguous(), _ids(n, G, 5)
    want = layer.adapter_add(y, x, down, up, ids, scale)
    for _ in range(20):
        assert torch.equal(layer.adapter_add(y, x, d, u, ids, scale), want)


def test_captured_and_differentiated(layer):
    from moe_gen_b200 import adapt_rows
    n, K, N, r, G = 300, 64, 48, 12, 3
    x, y, go = _rows(n, K, 1), _rows(n, N, 2), _rows(n, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    ids = _ids(n, G, 5)
    plan = layer.adapter_plan(ids, G)
    d, u = down.contiguous().requires_grad_(True), up.contiguous().requires_grad_(True)

    def step():
        out = adapt_rows(layer, y, x, d, u, plan, scale)
        return (out.detach(),) + torch.autograd.grad(out, (d, u), go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (6, 7):
        new = _adapters(G, r, K, N, 10 * seed)
        with torch.no_grad():
            d.copy_(new[0])
            u.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        refs = _reference(x, y, d.detach(), u.detach(), scale, ids, go)
        assert _near(got[0], refs[0]) and _near(got[1], refs[2]) and _near(got[2], refs[3])


def test_views_that_lie_off_the_boundaries_are_refused(layer):
    x, y = _rows(4, 64, 1), _rows(4, 32, 2)
    down, up, _ = _adapters(2, 16, 64, 32, 3)
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    for d, u in ((torch.zeros(2, 16, 65, dtype=torch.bfloat16, device=DEV)[:, :, :64], up), (down, torch.zeros(2, 32, 24, dtype=torch.bfloat16, device=DEV)[:, :, 1:17]),
                 (torch.zeros(2 * 16 * 64 + 65, dtype=torch.bfloat16, device=DEV).as_strided((2, 16, 64), (16 * 64 + 1, 64, 1)), up)):
        with pytest.raises(RuntimeError, match="boundaries"):
            layer.adapter_add(y, x, d, u, ids)
    with pytest.raises(RuntimeError, match="at most"):
        layer.adapter_add(y, x, torch.zeros(2, 130, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 32, 130, dtype=torch.bfloat16, device=DEV), ids)
