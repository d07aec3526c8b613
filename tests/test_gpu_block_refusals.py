"""GPU: a block on hidden + residual that is refused has written to neither of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("place", (0, 1))
def test_a_refused_block_leaves_the_residual_stream(built_lib, place):
    from moe_gen_b200 import MoELayer
    layer = MoELayer(hidden=512, inter=128, n_experts=8, top_k=2, device=DEV)
    g = torch.Generator().manual_seed(1)
    layer.set_router(torch.randn(8, 512, generator=g) * 0.05)
    for e in range(8):
        layer.load_expert(e, *[torch.randn(*s, generator=g).mul(0.05).to(torch.bfloat16).to(DEV) for s in ((128, 512), (128, 512), (512, 128))])
    t = [torch.randn(40, 512, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    w, xn, before = torch.ones(512, dtype=torch.bfloat16, device=DEV), torch.empty(40, 512, dtype=torch.bfloat16, device=DEV), [v.clone() for v in t]
    ws = layer._workspace(40)

    def call(gate=layer.gate_w.data_ptr(), packed=layer.packed.data_ptr(), size=ws.numel(), eps=1e-6):
        return layer.lib.mg_moe_block_forward_add(layer._h, t[0].data_ptr(), t[1].data_ptr(), w.data_ptr(), eps, 40, gate, None, packed, xn.data_ptr(),
                                                  ws.data_ptr(), size, t[place].data_ptr(), layer._stream())

    for kw, code in ((dict(size=256), -4), (dict(gate=None), -1), (dict(packed=None), -1), (dict(eps=-1.0), -3)):
        assert call(**kw) == code
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(t, before))
    want = layer.block_forward(before[0], w, 1e-6, residual=before[1])
    assert call() == 0 and torch.equal(t[place], want) and torch.equal(t[1 - place], before[1 - place])
    layer.close()


def test_more_experts_than_the_router_takes(built_lib):
    from moe_gen_b200 import MoELayer
    layer = MoELayer(hidden=256, inter=128, n_experts=260, top_k=2, device=DEV)
    layer.set_router(torch.zeros(260, 256))
    t = [torch.randn(3, 256, device=DEV).to(torch.bfloat16) for _ in range(2)]
    before = [v.clone() for v in t]
    for out in t:
        with pytest.raises(RuntimeError, match="256 experts"):
            layer.block_forward(t[0], torch.ones(256, dtype=torch.bfloat16, device=DEV), out=out, residual=t[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(t, before))
    layer.close()
