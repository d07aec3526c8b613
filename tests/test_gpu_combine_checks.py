"""GPU: the return of the experts' rows takes what torch computed, so it checks what it is given."""
import pytest
import torch

from tests.test_gpu_grad import DEV, _setup

pytestmark = pytest.mark.gpu


def _inputs():
    layer, idx, counts, pad, dst, rows, live = _setup(10, 8, 2, 256)
    out = torch.randn(rows, 256, device=DEV).to(torch.bfloat16)
    w = torch.rand(10, 2, device=DEV)
    sh = torch.randn(10, 256, device=DEV).to(torch.bfloat16)
    return layer, idx, counts, pad, dst, rows, out, w, sh


WRONG = {                                   # name -> what is handed over in place of (out_rows, dst_row, topk_idx, topk_w, shared_out)
    "rows in fp32": lambda o, d, i, w, s: (o.float(), d, i, w, s),
    "rows of half the width": lambda o, d, i, w, s: (o[:, :128], d, i, w, s),
    "picks in int64": lambda o, d, i, w, s: (o, d, i.long(), w, s),
    "destinations in int64": lambda o, d, i, w, s: (o, d.long(), i, w, s),
    "a shared row in fp32": lambda o, d, i, w, s: (o, d, i, w, s.float()),
    "weights in fp64": lambda o, d, i, w, s: (o, d, i, w.double(), s),
    "weights in bf16": lambda o, d, i, w, s: (o, d, i, w.to(torch.bfloat16), s),
    "weights of a view": lambda o, d, i, w, s: (o, d, i, torch.cat([w, w], dim=1)[:, ::2], s),
    "weights of fewer tokens": lambda o, d, i, w, s: (o, d, i, w[:4], s),
    "shared rows of fewer tokens": lambda o, d, i, w, s: (o, d, i, w, s[:4]),
    "destinations of fewer tokens": lambda o, d, i, w, s: (o, d[:4], i, w, s),
    "rows on the host": lambda o, d, i, w, s: (o.cpu(), d, i, w, s),
    "weights on the host": lambda o, d, i, w, s: (o, d, i, w.cpu(), s),
}


@pytest.mark.parametrize("wrong", list(WRONG))
def test_what_combine_refuses(wrong):
    from moe_gen_b200 import combine_rows
    layer, idx, counts, pad, dst, rows, out, w, sh = _inputs()
    o, d, i, w, s = WRONG[wrong](out, dst, idx, w, sh)
    with pytest.raises(ValueError):
        combine_rows(layer, o, d, i, w, counts, pad, s)
    with pytest.raises(ValueError):
        layer.combine(o, d, i, w, s)
    layer.close()


def test_rows_off_a_boundary_are_refused():
    from moe_gen_b200 import MoeGenError, combine_rows
    layer, idx, counts, pad, dst, rows, out, w, sh = _inputs()
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)      # noqa: E731
    for o, s in ((off(out), sh), (out, off(sh)), (off(out), None)):
        with pytest.raises(MoeGenError, match="16-byte"):
            combine_rows(layer, o, dst, idx, w, counts, pad, s)
    # weights are read one by one
    ref = combine_rows(layer, out, dst, idx, w, counts, pad, sh)
    assert torch.equal(combine_rows(layer, out, dst, idx, off(w).copy_(w), counts, pad, sh), ref)
    layer.close()


def test_an_adapter_in_fp32_is_refused_before_anything_is_computed():
    """The case that is met in earnest: rows of an adapter that was left in fp32, with and without gradients."""
    from moe_gen_b200 import combine_rows
    layer, idx, counts, pad, dst, rows, out, w, sh = _inputs()
    adapter = torch.randn(256, 256, device=DEV, requires_grad=True)
    y = out.float() @ adapter
    with pytest.raises(ValueError, match="out_rows"):
        combine_rows(layer, y, dst, idx, w, counts, pad)
    with torch.no_grad(), pytest.raises(ValueError, match="out_rows"):
        combine_rows(layer, y, dst, idx, w, counts, pad)
    assert combine_rows(layer, y.to(torch.bfloat16), dst, idx, w, counts, pad).requires_grad
    layer.close()
