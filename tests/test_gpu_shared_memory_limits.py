"""GPU: launches whose dynamic shared memory lies about what a block has without asking, each in a process of its own, where no larger
call has asked before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, env={**os.environ, "PYTHONPATH": ROOT},
                       timeout=300)
    assert r.returncode == 0 and "SAME" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]


PLAN = r"""
import torch
from oracle import moe_oracle as O
from tests.test_gpu_grad import DEV, _layer
E = EXPERTS
layer = _layer(E=E, k=4)
for T in TOKENS:
    idx = torch.rand(T, E, generator=torch.Generator().manual_seed(T)).topk(4, dim=1)[1].int()
    counts, off, pad, dst = [t.cpu() for t in layer.permute_plan(idx.to(DEV))]
    c, o, order, _ = O.permute_plan(idx.long(), E)
    assert torch.equal(counts.long(), c.long()) and torch.equal(off.long(), o.long())
    size = (c.long() + 127) // 128 * 128
    first = torch.cumsum(size, 0) - size
    want = torch.empty(T * 4, dtype=torch.long)
    e = idx.long().reshape(-1)[order]
    want[order] = first[e] + torch.arange(T * 4) - o.long()[e]
    assert torch.equal(dst.reshape(-1).long(), want)
print("SAME")
"""


@pytest.mark.parametrize("experts,tokens", [(512, [288, 320, 321, 352, 353]), (384, [448, 449, 480, 481])])
def test_plans_whose_bitmaps_fill_the_default(experts, tokens):
    _run(PLAN.replace("EXPERTS", str(experts)).replace("TOKENS", repr(tokens)))


ROUTE = r"""
import torch
from tests.test_gpu_grad import DEV, _layer
for H in (6400, 7168, 8192, 6656):             # a larger row after a smaller one
    layer = _layer(E=64, k=6, H=H)
    g = torch.Generator().manual_seed(H)
    layer.set_router(torch.randn(64, H, generator=g) * 0.1)
    x = torch.randn(40, H, generator=g).to(torch.bfloat16).to(DEV)
    idx, w, logits, fix = layer.gate_route(x)
    torch.cuda.synchronize()
    exact = x.double() @ layer.gate_w.double().t()
    assert ((logits.double() - exact).abs() <= 1e-4 * (x.double().abs() @ layer.gate_w.double().abs().t())).all()
    assert torch.equal(idx.long().sort(dim=1)[0], exact.topk(6, dim=1)[1].sort(dim=1)[0])
    layer.close()
print("SAME")
"""


def test_routing_of_a_larger_hidden_size_after_a_smaller_one():
    _run(ROUTE)
