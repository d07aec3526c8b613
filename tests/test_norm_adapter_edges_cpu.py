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


@pytest.mark.parametrize("kw,code", [(dict(gate=None), -1), (dict(packed=None), -1), (dict(ws=None), -1), (dict(n=1 << 31), -7), (dict(n=1 << 40), -7), (dict(), -3),
                                     (dict(gate=5 * P + 8), -2), (dict(packed=6 * P + 2), -2), (dict(ws=8 * P + 4), -2)])
def test_blocks_with_a_residual_are_refused_before_anything_is_launched(handle, kw, code):  # noqa: F811
    """The stand-in belongs to no number of ranks, which the block refuses: were the sum launched first, it would be the launch that fails here."""
    a = dict(n=4, gate=5 * P, packed=6 * P, ws=8 * P)
    a.update(kw)
    assert L.load().mg_moe_block_forward_add(handle[0], P, 2 * P, 3 * P, 1e-6, a["n"], a["gate"], None, a["packed"], 7 * P, a["ws"], 1 << 40, P,
                                             None) == code


@pytest.mark.parametrize("n,gx,gw,code", [(0, None, None, 0), (0, 5 * P, None, 0), (3, None, None, -1)])
def test_norm_gradients_of_no_rows(handle, n, gx, gw, code):  # noqa: F811
    """torch's address of an empty tensor is null: a batch without rows is one gradient without an address."""
    assert L.load().mg_add_rmsnorm_grad(handle[0], P, 64, 2 * P, 64, 3 * P, 1e-6, n, 64, 4 * P, 64, gx, 64, gw, None, 0, None) == code


def test_the_longest_rows_of_the_norms_gradient(handle):  # noqa: F811
    n = C.c_size_t()
    assert L.load().mg_add_rmsnorm_grad_ws_bytes(handle[0], 0, L.NORM_GRAD_COLS, C.byref(n)) == 0
    assert L.load().mg_add_rmsnorm_grad_ws_bytes(handle[0], 0, L.NORM_GRAD_COLS + 1, C.byref(n)) == -7
