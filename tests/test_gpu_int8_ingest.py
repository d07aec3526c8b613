"""GPU: what an int8 checkpoint may hold its scales in, and layers of other formats that are given int8 tensors."""
import pytest
import torch

from tests.test_gpu_int8 import _checkpoint_weights, _layer, quantise

pytestmark = pytest.mark.gpu


def test_int8_tensors_where_the_layer_keeps_bf16_are_refused(tmp_path):
    """A shared expert or a router stored in int8 is no bf16 matrix: its bytes without their scales mean nothing."""
    from moe_gen_b200 import ingest
    experts, shared, router = _checkpoint_weights(700)
    bf = [[torch.randn(q.shape).to(torch.bfloat16) for q, _ in e] for e in experts]
    q8 = [(q.to(torch.int8), s) for q, s in map(quantise, shared)]
    for name, kw in (("shared", dict(gate_w=router, shared=q8)), ("router", dict(gate_w=router.to(torch.int8), shared=shared))):
        d = tmp_path / name
        d.mkdir()
        ingest.export_moe_layer(str(d / "model.safetensors"), 0, kw["gate_w"], None, bf, shared=kw["shared"])
        layer = _layer(Is=128, int8=False)
        with pytest.raises(ValueError, match="int8"):
            ingest.load_moe_layer(layer, ingest.Checkpoint(str(d)), 0, n_threads=2)
        layer.close()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_scales_in_any_floating_type(tmp_path, dtype):
    """Scales stored in the model's own type are converted, for the routed experts as for the shared one."""
    from moe_gen_b200 import ingest
    experts, shared, router = _checkpoint_weights(710)
    experts = [[(q, s.to(dtype)) for q, s in e] for e in experts]
    q8 = [(q.to(torch.int8), s.to(dtype)[:, None]) for q, s in map(quantise, shared)]
    ingest.export_moe_layer(str(tmp_path / "model.safetensors"), 0, router, None, experts, shared=q8)
    got, want = _layer(Is=128, norm=True), _layer(Is=128, norm=True)
    ingest.load_moe_layer(got, ingest.Checkpoint(str(tmp_path)), 0, n_threads=2)
    want.set_router(router)
    for e, m in enumerate(experts):
        want.load_expert(e, *[q for q, _ in m], scales=tuple(s.float() for _, s in m))
    want.load_shared(*[q for q, _ in q8], tuple(s.float() for _, s in q8))
    assert torch.equal(got.packed, want.packed)
    got.close()
    want.close()


def test_scales_that_are_no_numbers_are_refused(tmp_path):
    from moe_gen_b200 import ingest
    experts, shared, router = _checkpoint_weights(720)
    experts[3][1] = (experts[3][1][0], experts[3][1][1].to(torch.int32))
    ingest.export_moe_layer(str(tmp_path / "model.safetensors"), 0, router, None, experts, shared=shared)
    layer = _layer(Is=128, norm=True)
    with pytest.raises(ValueError, match="weight_scale"):
        ingest.load_moe_layer(layer, ingest.Checkpoint(str(tmp_path)), 0, n_threads=2)
    layer.close()
