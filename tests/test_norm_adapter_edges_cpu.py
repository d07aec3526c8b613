"""CPU: more of what the norm and adapter calls refuse, and what they take, before they touch a device.  The handle is the stand-in of
test_norm_adapter_cpu.py, whose marks are all that these checks look at."""
import ctypes as C

import pytest

from moe_gen_b200 import lib as L
from tests.test_norm_adapter_cpu import P, _adapters, handle  # noqa: F401


@pytest.mark.parametrize("kw", [{k: P * a + off} for k, a in (("gdown", 10), ("gup", 11)) for off in (2, 4, 8)])
@pytest.mark.parametrize("rank,cols,n_out", [(16, 64, 32), (4, 64, 32), (8, 72, 33)])
def test_gradients_of_adapters_off_a_boundary_are_refused(handle, kw, rank, cols, n_out):  # noqa: F811
    a = dict(go=3 * P, ldg=64, x=4 * P, ldx=128, n=4, plan=5 * P, s=7 * P, gs=8 * P, gx=9 * P, ldgx=128, gdown=10 * P, gup=11 * P)
    a.update(kw)
    ld_up = (rank + 7) // 8 * 8
    ad = _adapters(rank=rank, cols=cols, n_out=n_out, down_stride=rank * 72, ld_down=72, up_stride=n_out * ld_up, ld_up=ld_up)
    assert L.load().mg_adapter_grad(handle[0], C.byref(ad), a["go"], a["ldg"], a["x"], a["ldx"], a["n"], a["plan"], a["s"], a["gs"], a["gx"],
                                    a["ldgx"], a["gdown"], a["gup"], None) == -2
