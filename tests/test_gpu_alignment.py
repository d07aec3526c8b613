"""GPU: contiguous views that begin off a 16-byte boundary.  Weights are copied, rows are refused before anything is launched."""
import itertools

import pytest
import torch

from tests.test_gpu_grad import DEV, _setup
from tests.test_gpu_int8 import _layer, _load, _weights

pytestmark = pytest.mark.gpu


def _off(t):
    v = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
    assert v.is_contiguous() and v.data_ptr() % 16
    return v.copy_(t)


@pytest.mark.parametrize("int8,shared", list(itertools.product((False, True), (False, True))))
def test_weights_that_begin_anywhere(int8, shared):
    a, b = (_layer(E=4, Is=128 if shared else 0, int8=int8) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    for e in list(range(4)) + ([-1] if shared else []):
        shapes = ((128, 256), (128, 256), (256, 128))
        m = [_weights(*s, 7 * e + i) if int8 else (torch.randn(s, generator=g).to(torch.bfloat16), None) for i, s in enumerate(shapes)]
        sc = tuple(s for _, s in m) if int8 else None
        a.load_expert(e, *[w for w, _ in m], scales=sc)
        b.load_expert(e, *[_off(w) for w, _ in m], scales=tuple(_off(s) for s in sc) if int8 else None)
    router = torch.randn(4, 256, generator=g).to(torch.bfloat16)
    a.set_router(router)
    b.set_router(_off(router))
    assert torch.equal(a.packed, b.packed) and torch.equal(a.gate_w, b.gate_w) and b.gate_w.data_ptr() % 16 == 0
    x = torch.randn(9, 256, generator=g).to(torch.bfloat16).to(DEV)
    assert torch.equal(a.forward(x), b.forward(x))
    a.close()
    b.close()


def test_fp8_matrices_that_begin_anywhere():
    layer = _layer(int8=False)
    q = torch.randn(128, 256).to(torch.float8_e4m3fn).to(DEV)
    s = torch.rand(1, 2, device=DEV) + 0.5
    off = torch.empty(q.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(q.shape).copy_(q.view(torch.uint8)).view(q.dtype)
    assert off.data_ptr() % 16 and torch.equal(layer.dequant_fp8(off, s), layer.dequant_fp8(q, s))
    layer.close()


def test_rows_that_begin_anywhere_are_refused():
    from moe_gen_b200 import MoeGenError
    layer, idx, counts, pad, dst, rows, live = _setup(10, 8, 2, 256)
    layer.set_router(torch.zeros(8, 256))
    x = torch.zeros(10, 256, dtype=torch.bfloat16, device=DEV)
    norm = torch.ones(256, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: layer.rmsnorm(_off(x), norm), lambda: layer.rmsnorm(x, _off(norm)), lambda: layer.rmsnorm(x, norm, out=_off(x)),
                lambda: layer.permute_rows(_off(x), dst, rows), lambda: layer.block_forward(_off(x), norm),
                lambda: layer.block_forward(x, norm, out=_off(x)), lambda: layer.forward(_off(x)), lambda: layer.forward(x, out=_off(x))):
        with pytest.raises(MoeGenError, match="16-byte"):
            bad()
    assert torch.equal(layer.permute_rows(x, dst, rows), torch.zeros(rows, 256, dtype=torch.bfloat16, device=DEV))
    layer.close()
