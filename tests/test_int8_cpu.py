"""CPU: what the 8-bit integer and gradient entry points refuse before they touch a device."""
import ctypes as C

import pytest

from moe_gen_b200 import lib as L


def _desc(**kw):
    d = L.LayerDesc(C.sizeof(L.LayerDesc), 256, 128, 0, 64, 6, 1, 1, 0, 0, 1.0, L.WEIGHT_INT8_CHANNEL, 0, 0, 1)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,code", [(dict(ep_size=2), -3), (dict(hidden=131072), -7), (dict(inter=131072), -7),
                                     (dict(inter_shared=131072), -7), (dict(hidden=250), -2), (dict(weight_format=3), -3)])
def test_int8_layers_that_are_refused(built_lib, kw, code):
    lib, h = L.load(), C.c_void_p()
    assert lib.mg_create(C.byref(_desc(**kw)), C.byref(h)) == code and not h.value


def test_scratch_of_the_product(built_lib):
    lib, n = L.load(), C.c_size_t()
    assert lib.mg_int8_linear_ws_bytes(17, 4, 1000, C.byref(n)) == 0 and n.value >= 17 * 1024 + 68
    assert lib.mg_int8_linear_ws_bytes(16, 4096, 2048, C.byref(n)) == 0 and n.value == 0
    assert lib.mg_int8_linear_ws_bytes(16, 4097, 2048, C.byref(n)) == 0 and n.value >= 16 * 2048
    assert lib.mg_int8_linear_ws_bytes(9, 8, 2049, C.byref(n)) == 0 and n.value >= 9 * 2176
    assert lib.mg_int8_linear_ws_bytes(8, 20, 12288, C.byref(n)) == 0 and n.value == 0             # one launch, no scratch
    assert lib.mg_int8_linear_ws_bytes(8, 20, 12289, C.byref(n)) == 0 and n.value >= 8 * 12416
    assert lib.mg_int8_linear_ws_bytes(4, 1 << 30, 4096, C.byref(n)) == 0 and n.value == 0
    assert lib.mg_int8_linear_ws_bytes(5, 4096, 4096, C.byref(n)) == 0 and n.value == 0
    assert lib.mg_int8_linear_ws_bytes(5, 4097, 4096, C.byref(n)) == 0 and n.value >= 5 * 4096
    assert lib.mg_int8_linear_ws_bytes(0, 8, 1000, C.byref(n)) == 0 and n.value == 0
    assert lib.mg_int8_linear_ws_bytes(1 << 30, 8, 131071, C.byref(n)) == 0 and n.value >= (1 << 30) * 131072
    assert lib.mg_int8_linear_ws_bytes(5, 8, 131072, C.byref(n)) == -7
    assert lib.mg_int8_linear_ws_bytes(5, 8, 0, C.byref(n)) == -2 and lib.mg_int8_linear_ws_bytes(-1, 8, 8, C.byref(n)) == -2
    assert lib.mg_int8_linear_ws_bytes(5, 0, 8, C.byref(n)) == -2 and lib.mg_int8_linear_ws_bytes(5, 8, 8, None) == -1


@pytest.mark.parametrize("name", ["mg_quantize_rows_int8", "mg_int8_matmul", "mg_int8_linear", "mg_permute_rows_int8", "mg_expert_ffn_int8",
                                  "mg_shared_ffn_int8", "mg_permute_rows_padded", "mg_permute_rows_grad", "mg_combine_grad",
                                  "mg_route_topk_grad"])
def test_no_handle_is_an_error(built_lib, name):
    lib = L.load()
    args = [None if t in (C.c_void_p,) or not issubclass(t, (C.c_int64, C.c_int32, C.c_size_t)) else 1 for t in L.SIGNATURES[name]]
    assert getattr(lib, name)(*args) == -5 and lib.mg_last_error() != b""
