"""GPU: few bf16 rows through int8_linear, whose bytes lie in shared memory, about the 48 KB that a block may have without asking."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FEW = r"""
import torch
from tests.test_gpu_int8 import DEV, _layer, _strided, _weights, product, quantise, same
layer = _layer()
for m, k in SIZES:                     # from small to large: a larger call raises the kernel's limit for all after it
    wq, ws = _weights(8, k, k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(torch.bfloat16)
    y = layer.int8_linear(x.to(DEV), _strided(wq), ws.to(DEV))
    assert same(y.cpu(), product(*quantise(x), wq, ws)), (m, k)
print("EXACT")
"""


@pytest.mark.parametrize("sizes", [[(1, 49056), (1, 49072), (1, 49073), (1, 49088), (1, 49089), (1, 49152)],
                                   [(2, 24528), (2, 24529), (2, 24544), (2, 24560)],
                                   [(3, 12256), (4, 12257), (3, 12270), (4, 12272), (4, 12288)],
                                   [(8, 6128), (5, 6136), (8, 6144)]])
def test_few_rows_about_the_default_shared_memory(sizes):
    """In a process of its own: the limit raised by an earlier, larger call would hide a launch beyond the default."""
    r = subprocess.run([sys.executable, "-c", FEW.replace("SIZES", repr(sizes))], cwd=ROOT, capture_output=True, text=True,
                       env={**os.environ, "PYTHONPATH": ROOT}, timeout=300)
    assert r.returncode == 0 and "EXACT" in r.stdout, r.stdout[-1000:] + r.stderr[-2000:]
