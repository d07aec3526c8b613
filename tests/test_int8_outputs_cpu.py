"""CPU: which products of few rows run in one launch, whose kernel counts outputs in 32 bits and steps past the last one by a
grid's worth (32 to a block, at most three blocks per SM)."""
import ctypes as C

import pytest

from moe_gen_b200 import lib as L


@pytest.mark.parametrize("rows", (1, 2, 3, 4, 8, 16))
@pytest.mark.parametrize("n_out", ((1 << 30) + 1, (1 << 31) - 14208, (1 << 31) - 520, (1 << 31) - 513))
def test_products_whose_outputs_do_not_count_in_32_bits_take_two_launches(built_lib, rows, n_out):
    n = C.c_size_t()
    assert L.load().mg_int8_linear_ws_bytes(rows, n_out, 16, C.byref(n)) == 0 and n.value >= rows * 128 + rows * 4
