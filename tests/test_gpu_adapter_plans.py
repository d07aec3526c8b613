"""GPU: sorted plans whose offsets begin anywhere.  Every row of the results is written, by one tile: the offsets are first made to ascend within
the rows, each no less than the one in front of it, and what then lies in no adapter's segment has none.

Tolerances as in test_gpu_adapters.py, by its formulas in 64 bits."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_adapters import DEV, _adapters, _near, _reference, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


def _ids_of(counts, pad, rows):
    start = torch.tensor(pad).clamp(0, rows).cummax(0)[0]
    at = torch.arange(rows)
    seg = torch.searchsorted(start, at, right=True) - 1              # of segments that begin at one row the last, the others being empty
    inside = (seg >= 0) & (seg < len(counts))
    g = seg.clamp(0, len(counts) - 1)
    live = inside & (at - start[g] < torch.tensor(counts)[g])
    return torch.where(live, g, torch.full_like(g, -1)).int().to(DEV)


def _calls(layer, counts, pad, rows, K, N, r):
    """add and the gradients on buffers that hold NaN before, against the formulas: all rows."""
    from moe_gen_b200 import lib as L
    G = len(counts)
    ids = _ids_of(counts, pad, rows)
    none = ids < 0
    x, y, go = _rows(rows, K, 1), _rows(rows, N, 2), _rows(rows, N, 3)
    x[none] = float("nan")
    go[none] = float("nan")
    down, up, scale = _adapters(G, r, K, N, 4)
    refs = _reference(x, y, down, up, scale, ids, go)
    plan = layer.adapter_plan_sorted(torch.tensor(counts, dtype=torch.int32, device=DEV), torch.tensor(pad, dtype=torch.int32, device=DEV), rows)
    out, gx = (_rows(*t.shape, 9).fill_(float("nan")) for t in (y, x))
    n = C.c_int32()
    L.check(layer.lib.mg_adapter_rank_stride(r, C.byref(n)))
    s, gs = (torch.full((rows, n.value), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    gd, gu = (torch.full(t, float("nan"), dtype=torch.bfloat16, device=DEV) for t in ((G, r, K), (G, N, r)))
    ad = L.ADAPTERS.pack(L.ADAPTERS.size, G, r, 1.0, K, N, down.data_ptr(), down.stride(0), down.stride(1), up.data_ptr(), up.stride(0),
                         up.stride(1), scale.data_ptr())
    ld = [t.stride(0) for t in (x, y, out, go, gx)]
    L.check(layer.lib.mg_adapter_add(layer._h, ad, x.data_ptr(), ld[0], y.data_ptr(), ld[1], rows, None, plan.buf.data_ptr(), out.data_ptr(),
                                     ld[2], s.data_ptr(), layer._stream()))
    L.check(layer.lib.mg_adapter_grad(layer._h, ad, go.data_ptr(), ld[3], x.data_ptr(), ld[0], rows, plan.buf.data_ptr(), s.data_ptr(),
                                      gs.data_ptr(), gx.data_ptr(), ld[4], gd.data_ptr(), gu.data_ptr(), layer._stream()))
    torch.cuda.synchronize()
    assert torch.equal(out[none], y[none]) and not gx[none].any() and not s[none].any()
    assert all(_near(t, ref) for t, ref in zip((out, gx, gd, gu), refs))
    place = y.clone()
    if place.stride(0) % 8 == 0:
        assert torch.equal(layer.adapter_add(place, x, down, up, plan, scale, out=place), out)


@pytest.mark.parametrize("counts,pad,rows", [([5, 5], [130, 258, 300], 400), ([4, 4], [3, 17, 40], 41), ([0, 0], [50, 50, 50], 700),
                                             ([1], [1, 2], 3), ([7], [128, 256], 256), ([200, 128], [384, 640, 768], 900), ([9] * 6, [100000 + 128 * k for k in range(7)], 101000),
                                             ([1] * 1024, [77 + k for k in range(1025)], 1500)])
@pytest.mark.parametrize("K,N,r", [(64, 72, 16), (136, 64, 40)])
def test_rows_in_front_of_the_first_segment(layer, counts, pad, rows, K, N, r):
    _calls(layer, counts, pad, rows, K, N, r)


@pytest.mark.parametrize("counts,pad,rows", [([128, 5], [0, 128, 100], 300), ([200, 200, 9], [0, 200, 100, 300], 320), ([300, 300], [40, 500, 20], 600),
                                             ([128] * 5, [256, 0, 384, 128, 512, 64], 700), ([64] * 300, [(97 * k) % 5000 for k in range(301)], 4000),
                                             ([9, 9], [1 << 30, -5, 12], 64), ([500, 500], [-(1 << 31), (1 << 31) - 1, 0], 300)])
@pytest.mark.parametrize("K,N,r", [(64, 72, 16), (136, 64, 40)])
def test_segments_that_would_reach_into_one_another(layer, counts, pad, rows, K, N, r):
    _calls(layer, counts, pad, rows, K, N, r)


def test_the_experts_of_a_part_of_the_buffer(layer):
    """The offsets of experts 4 to 7 of a plan of eight, as they are in the whole buffer."""
    idx = torch.randint(0, 8, (300, 1), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(1))
    counts, _, pad, _ = layer.permute_plan(torch.cat([idx, (idx + 1) % 8], dim=1))
    _calls(layer, counts[4:].tolist(), pad[4:].tolist(), layer.padded_rows(600), 64, 72, 16)


@pytest.mark.parametrize("counts", [[50, 0, 128, 7], [300, 1, 0, 129, 64], [9] * 40])
def test_either_plan_of_the_same_tiles_gives_the_same_bits(layer, counts):
    """Segments on 128-row boundaries are cut where the ids' rows are: the tiles' rows, their number and so the blocks that share them are the
    same, and the sums' order with them."""
    G, K, N, r = len(counts), 136, 72, 16
    c = torch.tensor(counts, dtype=torch.int32)
    pad = torch.zeros(G + 1, dtype=torch.int32)
    pad[1:] = torch.cumsum((c + 127) // 128 * 128, 0)
    rows = int(pad[-1]) + 128
    ids = _ids_of(counts, pad.tolist(), rows)
    x, y, go = _rows(rows, K, 1), _rows(rows, N, 2), _rows(rows, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    got = []
    for plan in (layer.adapter_plan_sorted(c.to(DEV), pad.to(DEV), rows), layer.adapter_plan(ids, G)):
        out, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
        got.append((out, s) + layer.adapter_grad(go, x, down, up, plan, scale, s))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    refs = _reference(x, y, down, up, scale, ids, go)
    assert _near(got[0][0], refs[0]) and all(_near(t, ref) for t, ref in zip(got[0][2:], refs[1:]))


@pytest.mark.parametrize("counts,extra", [([1] * 100 + [0] * 60, 128), ([3] * 300, 128), ([2] * 160, 40 * 128), ([0] * 300, 128), ([0, 3, 0] * 100, 0), ([9] * 75, 5),
                                          ([0] * 90 + [128] * 70, 128), ([1] * 200, 40 * 128)])
@pytest.mark.parametrize("K,N,r", [(64, 4104, 16), (4100, 72, 13), (72, 4096, 100)])
def test_clusters_that_share_the_tiles_of_long_rows(layer, counts, extra, K, N, r):
    """More tiles than run at once, most of them without an adapter or of few rows, by rows of 4096 columns and more in either direction: up to
    204 tiles of 4096 columns are shared by four blocks, more by two."""
    pad = [0]
    for n in counts:
        pad.append(pad[-1] + (max(n, 1) + 127) // 128 * 128)
    _calls(layer, counts, pad, pad[-1] + extra, K, N, r)
