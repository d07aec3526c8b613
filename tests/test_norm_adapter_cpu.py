"""CPU: what the norm and adapter calls refuse before they touch a device.  The handle is a stand-in: a buffer that begins with a
handle's mark, which is all that the checks look at."""
import ctypes as C

import pytest

from moe_gen_b200 import lib as L

P = 1 << 20                       # an address on every boundary; nothing is read there


@pytest.fixture(scope="module")
def handle(built_lib):
    buf = C.create_string_buffer(1 << 16)
    C.c_uint32.from_buffer(buf).value = 0x4d474232
    yield C.cast(buf, C.c_void_p), buf


@pytest.mark.parametrize("name", [n for n in L.SIGNATURES if n.startswith(("mg_add_rmsnorm", "mg_adapter_", "mg_moe_block_forward_add"))
                                  and L.SIGNATURES[n][0] is C.c_void_p])
def test_no_handle_is_an_error(built_lib, name):
    lib = L.load()
    args = [1 if issubclass(t, (C.c_int64, C.c_int32, C.c_size_t, C.c_float)) else None for t in L.SIGNATURES[name]]
    assert getattr(lib, name)(*args) == -5 and lib.mg_last_error() != b""


NORM = dict(x=P, ldx=64, res=2 * P, ldr=64, w=3 * P, eps=1e-6, n=4, cols=64, sum=4 * P, lds=64, out=5 * P, ldo=64)
BAD_NORM = [(dict(n=-1), -2), (dict(cols=0), -2), (dict(ldx=63), -2), (dict(ldr=63), -2), (dict(lds=63), -2), (dict(ldo=63), -2),
            (dict(cols=(1 << 24) + 1, ldx=1 << 25, ldr=1 << 25, lds=1 << 25, ldo=1 << 25), -7), (dict(n=1 << 31), -7), (dict(eps=-1.0), -3),
            (dict(x=None), -1), (dict(w=None), -1), (dict(out=None), -1), (dict(sum=None), -1), (dict(sum=5 * P), -3),
            (dict(sum=P, lds=72), -3), (dict(sum=2 * P, lds=72), -3)]


@pytest.mark.parametrize("kw,code", BAD_NORM + [(dict(out=P, ldo=72), -3), (dict(out=2 * P, ldo=72), -3)])
def test_norms_that_are_refused(handle, kw, code):
    a = dict(NORM, **kw)
    assert L.load().mg_add_rmsnorm(handle[0], a["x"], a["ldx"], a["res"], a["ldr"], a["w"], a["eps"], a["n"], a["cols"], a["sum"], a["lds"],
                                   a["out"], a["ldo"], None) == code


@pytest.mark.parametrize("kw,code", BAD_NORM + [(dict(scale=None), -1), (dict(out=P), -3), (dict(out=2 * P), -3)])
def test_quantised_norms_that_are_refused(handle, kw, code):
    a = dict(NORM, scale=6 * P)
    a.update(kw)
    assert L.load().mg_add_rmsnorm_int8(handle[0], a["x"], a["ldx"], a["res"], a["ldr"], a["w"], a["eps"], a["n"], a["cols"], a["sum"],
                                        a["lds"], a["out"], a["ldo"], a["scale"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(n=-1), -2), (dict(cols=0), -2), (dict(cols=16385, ldgy=16392, ldh=16392, ldgh=16392, ldgx=16392), -7),
                                     (dict(ldgy=63), -2), (dict(ldh=63), -2), (dict(ldgh=63), -2), (dict(ldgx=63), -2), (dict(eps=-1.0), -3),
                                     (dict(gx=None, gw=None), -1), (dict(gy=None), -1), (dict(h=None), -1), (dict(w=None), -1),
                                     (dict(gx=P, ldgx=72), -3), (dict(gx=4 * P, ldgx=72), -3), (dict(gx=2 * P), -3)])
def test_norm_gradients_that_are_refused(handle, kw, code):
    a = dict(gy=P, ldgy=64, h=2 * P, ldh=64, w=3 * P, eps=1e-6, n=4, cols=64, gh=4 * P, ldgh=64, gx=5 * P, ldgx=64, gw=6 * P, ws=7 * P)
    a.update(kw)
    assert L.load().mg_add_rmsnorm_grad(handle[0], a["gy"], a["ldgy"], a["h"], a["ldh"], a["w"], a["eps"], a["n"], a["cols"], a["gh"],
                                        a["ldgh"], a["gx"], a["ldgx"], a["gw"], a["ws"], 0, None) == code


def _adapters(**kw):
    a = L.Adapters(C.sizeof(L.Adapters), 4, 16, 1.0, 64, 32, P, 16 * 64, 64, 2 * P, 32 * 16, 16, None)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_ADAPTERS = [(dict(struct_bytes=8), -3), (dict(n_adapters=0), -2), (dict(rank=0), -2), (dict(cols=0), -2), (dict(n_out=0), -2),
                (dict(n_adapters=1025), -7), (dict(rank=129), -7), (dict(cols=(1 << 24) + 1), -7), (dict(n_out=(1 << 24) + 1), -7),
                (dict(d_down=None), -1), (dict(d_up=None), -1), (dict(d_down=P + 2), -2), (dict(d_up=2 * P + 8), -2), (dict(ld_down=68), -2),
                (dict(ld_down=56), -2), (dict(ld_up=20), -2), (dict(ld_up=8), -2), (dict(down_stride=16 * 64 + 4), -2),
                (dict(up_stride=32 * 16 + 4), -2), (dict(up_stride=-512), -2)]
BAD_ADD = [(dict(n=-1), -2), (dict(n=1 << 28), -7), (dict(n=257), -7), (dict(x=None), -1), (dict(y=None), -1), (dict(out=None), -1),
           (dict(ids=None), -1), (dict(x=3 * P + 8), -2), (dict(y=4 * P + 8), -2), (dict(out=6 * P + 2), -2), (dict(s=8 * P + 8), -2),
           (dict(plan=7 * P + 8), -2), (dict(ldx=60), -2), (dict(ldx=68), -2), (dict(ldy=36), -2), (dict(ldo=24), -2),
           (dict(out=4 * P, ldo=40), -3), (dict(out=3 * P), -3)]


@pytest.mark.parametrize("which,kw,code", [("ad", k, c) for k, c in BAD_ADAPTERS] + [("add", k, c) for k, c in BAD_ADD])
def test_adapters_that_are_refused(handle, which, kw, code):
    a = dict(x=3 * P, ldx=64, y=4 * P, ldy=32, n=4, ids=5 * P, plan=None, out=6 * P, ldo=32, s=None)
    ad = _adapters(**kw) if which == "ad" else _adapters()
    a.update(kw if which == "add" else {})
    assert L.load().mg_adapter_add(handle[0], C.byref(ad), a["x"], a["ldx"], a["y"], a["ldy"], a["n"], a["ids"], a["plan"], a["out"], a["ldo"],
                                   a["s"], None) == code
    assert L.load().mg_adapter_add(handle[0], None, P, 64, P, 32, 4, P, None, P, 32, None, None) == -1


@pytest.mark.parametrize("which,kw,code", [("ad", k, c) for k, c in BAD_ADAPTERS] +
                         [("grad", k, c) for k, c in [(dict(n=-1), -2), (dict(gx=None, gdown=None, gup=None), -1), (dict(go=None), -1),
                                                      (dict(plan=None), -1), (dict(x=None), -1), (dict(s=None), -1), (dict(gs=None), -1),
                                                      (dict(go=3 * P + 8), -2), (dict(gs=8 * P + 8), -2), (dict(ldg=36), -2),
                                                      (dict(ldx=56), -2), (dict(ldgx=68), -2), (dict(gx=3 * P), -3), (dict(gx=4 * P), -3)]])
def test_adapter_gradients_that_are_refused(handle, which, kw, code):
    a = dict(go=3 * P, ldg=32, x=4 * P, ldx=64, n=4, plan=5 * P, s=7 * P, gs=8 * P, gx=9 * P, ldgx=64, gdown=10 * P, gup=11 * P)
    ad = _adapters(**kw) if which == "ad" else _adapters()
    a.update(kw if which == "grad" else {})
    assert L.load().mg_adapter_grad(handle[0], C.byref(ad), a["go"], a["ldg"], a["x"], a["ldx"], a["n"], a["plan"], a["s"], a["gs"], a["gx"],
                                    a["ldgx"], a["gdown"], a["gup"], None) == code


def test_plans_that_are_refused(handle):
    lib, n, r = L.load(), C.c_size_t(), C.c_int32()
    assert lib.mg_adapter_plan_bytes(-1, 4, C.byref(n)) == -2 and lib.mg_adapter_plan_bytes(4, 0, C.byref(n)) == -2
    assert lib.mg_adapter_plan_bytes(1 << 28, 4, C.byref(n)) == -7 and lib.mg_adapter_plan_bytes(4, 1025, C.byref(n)) == -7
    assert lib.mg_adapter_plan_bytes(4, 4, None) == -1
    assert lib.mg_adapter_plan(handle[0], None, 4, 4, P, None) == -1 and lib.mg_adapter_plan(handle[0], P, 4, 4, None, None) == -1
    assert lib.mg_adapter_plan(handle[0], P, 4, 4, P + 8, None) == -2
    assert lib.mg_adapter_plan_sorted(handle[0], None, P, 4, 4, P, None) == -1
    assert lib.mg_adapter_plan_sorted(handle[0], P, None, 4, 4, P, None) == -1
    assert lib.mg_adapter_plan_sorted(handle[0], P, P, 4, 4, P + 8, None) == -2
    for rank, stride in ((1, 32), (16, 32), (17, 64), (33, 128), (65, 256), (128, 256)):
        assert lib.mg_adapter_rank_stride(rank, C.byref(r)) == 0 and r.value == stride
    assert lib.mg_adapter_rank_stride(0, C.byref(r)) == -7 and lib.mg_adapter_rank_stride(129, C.byref(r)) == -7


@pytest.mark.parametrize("rows,adapters", [(0, 1), (1, 1), (63, 3), (64, 4), (65, 1024), (100000, 7)])
def test_a_plan_holds_its_tiles_segments_and_order(built_lib, rows, adapters):
    """16 bytes to a tile of 128 rows or a part of one, for every adapter and for none, 8 to an adapter, 4 to a row."""
    n = C.c_size_t()
    assert L.load().mg_adapter_plan_bytes(rows, adapters, C.byref(n)) == 0
    assert n.value >= 16 * ((rows + 127) // 128 + adapters + 1) + 8 * adapters + 4 * rows


def test_adapters_struct_matches_the_header():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = open(os.path.join(root, "include", "moegen_b200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct mg_adapters \{(.*?)\} mg_adapters;", src, re.S).group(1), flags=re.S)
    names = [n.strip().lstrip("*").split()[-1].lstrip("*") for part in body.split(";") for n in part.split(",") if n.strip()]
    assert names == [f[0] for f in L.Adapters._fields_]
