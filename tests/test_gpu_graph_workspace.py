"""GPU: captured forwards after the layer has moved to larger workspaces."""
import itertools

import pytest
import torch

from tests.test_gpu_int8 import DEV, FORWARD, _ready

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block,option", list(itertools.product((False, True), (False, True))))
def test_a_replayed_graph_after_a_larger_batch(block, option):
    """Whatever takes the place of the layer's workspace, the memory that a graph writes to stays its own."""
    from moe_gen_b200 import lib as L
    layer, _ = _ready(FORWARD[0])
    norm = torch.ones(layer.H, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(24, layer.H, generator=g).to(torch.bfloat16).to(DEV)
    y = torch.empty_like(x)

    def step():
        return layer.block_forward(x, norm, out=y) if block else layer.forward(x, out=y)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step().clone()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    sizes = [layer._ws.numel()] + ([layer._xnorm.numel() * 2] if block else [])
    if option:
        layer.set_option(L.OPT_FP8_MODE, 0)              # gives the workspace up
    big = torch.randn(700, layer.H, generator=g).to(torch.bfloat16).to(DEV)
    layer.block_forward(big, norm) if block else layer.forward(big)
    torch.cuda.synchronize()
    others = [torch.full((n,), 77, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(4)]
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and all(bool((t == 77).all()) for t in others)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and layer.device_status() == (0, 0)
    layer.close()
