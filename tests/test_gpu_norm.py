"""GPU: the norm with the residual's addition, in bf16 and 8-bit integers, and its gradient, against the formulas in 64 bits.

Tolerances, u = 2^-24 being half a step of fp32 relative to the value, for V vectors of eight elements to a lane.
rstd: a lane adds 8V squares, a warp 5 times, a block 8 times, all of positive terms: the sum is off by (8V + 13) u relative, its root by half
of that; mean, eps, root and quotient round once each: R = (8V + 13) / 2 + 4 units.
Rows in bf16: w * (h * rstd) is off by R + 2 units, and rounded to bf16 once: (1 + 2^-8) (1 + (R + 2) u) - 1, where that is normal.
Rows in 8 bits: w * (h * rstd) is off by r = R + 2 units.  The maximum by the same, scale and inverse by one more each; a byte before its
rounding by 127 (2r + 2) u, so that it differs from the exact row's by at most half a step and that, and its value by the scale's error too.
Gradients: a lane adds at most 16 products, a warp 5 times, a block 32 times.  The sum over w gy h is off by 54 units of the sum of
magnitudes, rstd by 30 units, thus rstd^3 by 90, and 6 more roundings follow: 150 units of each term's magnitude, and half a step of bf16.
The weight's: n by 31 units, and as many additions as a share has rows, plus shares / 32, plus 5."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
SHAPES = [(1, 256), (1, 7168), (3, 2048), (37, 4096), (2, 8), (5, 1), (7, 1000), (4, 1001), (9, 77), (33, 2056), (2, 16384), (3, 16392), (2, 20001),
          (2048, 512), (2049, 256), (2050, 2048), (3000, 1024), (2048, 2056), (4100, 40)]


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


def _rows(n, cols, seed, ld=None, off=0, scale=1.0):
    """[n, cols] bf16, ld elements apart, beginning off elements behind a 16-byte boundary, NaN around them."""
    ld = cols if ld is None else ld
    g = torch.Generator(device=DEV).manual_seed(seed)
    wide = torch.full((off + n * ld + 8,), float("nan"), dtype=torch.bfloat16, device=DEV)
    v = wide[off:off + n * ld].view(n, ld)[:, :cols]
    v.copy_(torch.randn(n, cols, generator=g, device=DEV) * scale)
    if cols > 8:
        v[:, ::64] *= 8
    return v


def _weight(cols, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.rand(cols, generator=g, device=DEV) * 2 - 0.5).to(torch.bfloat16)


def _units(cols):
    return (8 * ((cols + 2047) // 2048) + 13) / 2 + 4


def _check_rows(y, h, w, eps):
    h, cols = h.double(), h.shape[1]
    want = h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps) * w.double()
    assert ((y.double() - want).abs() <= want.abs() * ((1 + 2.0 ** -8) * (1 + (_units(cols) + 2) * U) - 1) + 2.0 ** -130).all()


@pytest.mark.parametrize("n,cols", SHAPES)
@pytest.mark.parametrize("residual", (True, False))
def test_rows_and_sum(layer, n, cols, residual):
    x, w = _rows(n, cols, 1), _weight(cols, 2)
    r = _rows(n, cols, 3, scale=2.0) if residual else None
    y, h = layer.add_rmsnorm(x, r, w, 1e-6)
    assert (h is x) if not residual else torch.equal(h, x + r)
    _check_rows(y, h, w, 1e-6)
    q, scale, h8 = layer.add_rmsnorm_int8(x, r, w, 1e-6)
    assert torch.equal(h8, h)
    units = _units(cols) + 2
    d = h.double()
    v = d / torch.sqrt(d.square().mean(dim=1, keepdim=True) + 1e-6) * w.double()
    m = v.abs().amax(dim=1).clamp_min(2.0 ** -100)
    assert ((scale.double() - m / 127).abs() <= m / 127 * (units + 2) * U).all()
    assert ((q.double() - v * (127 / m)[:, None]).abs() <= 0.5 + 127 * (2 * units + 2) * U).all()
    assert q.to(torch.int32).abs().max() <= 127


@pytest.mark.parametrize("n,H", [(1, 256), (37, 2048), (2300, 512), (2300, 1024), (2300, 2048), (64, 4096), (16, 7168), (5, 8192), (2, 16384)])
def test_the_same_bits_by_every_kernel(layer, n, H):
    """A row's bits do not depend on the batch, the strides or the alignment."""
    w = _weight(H, 5)
    x, r = _rows(n, H, 6).clone(), _rows(n, H, 7).clone()
    want, want8 = layer.add_rmsnorm(x, r, w, 1e-5), layer.add_rmsnorm_int8(x, r, w, 1e-5)
    for ld, off in ((H + 64, 8), (H + 5, 3)):
        a, b = _rows(n, H, 6, ld, off), _rows(n, H, 7, ld, off)
        a.copy_(x)
        b.copy_(r)
        assert all(torch.equal(p, q) for p, q in zip(layer.add_rmsnorm(a, b, w, 1e-5), want))
        assert all(torch.equal(p, q) for p, q in zip(layer.add_rmsnorm_int8(a, b, w, 1e-5), want8))
    some = slice(n // 2, n // 2 + 1)
    assert all(torch.equal(p, q[some]) for p, q in zip(layer.add_rmsnorm(x[some], r[some], w, 1e-5), want))
    assert all(torch.equal(p, q[some]) for p, q in zip(layer.add_rmsnorm_int8(x[some], r[some], w, 1e-5), want8))


@pytest.mark.parametrize("n,cols,ld,off", [(3, 512, 576, 0), (2100, 512, 576, 0), (5, 512, 576, 8), (5, 512, 577, 1), (2100, 96, 101, 0), (3, 100, 104, 4)])
def test_strided_rows_and_what_lies_around_them(layer, n, cols, ld, off):
    x, r, w = _rows(n, cols, 1, ld, off), _rows(n, cols, 2, ld, off), _weight(cols, 3)
    want = layer.add_rmsnorm(x.contiguous(), r.contiguous(), w)
    want8 = layer.add_rmsnorm_int8(x.contiguous(), r.contiguous(), w)
    hold = [torch.full((n * ld + off + 8,), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    out, total = (t[off:off + n * ld].view(n, ld)[:, :cols] for t in hold)
    y, h = layer.add_rmsnorm(x, r, w, out=out, sum_out=total)
    assert y is out and h is total and torch.equal(y, want[0]) and torch.equal(h, want[1])
    for t, v in zip(hold, (out, total)):
        left = t.clone()
        left[off:off + n * ld].view(n, ld)[:, :cols] = 7.0
        assert (left == 7.0).all()
    assert all(torch.equal(a, b) for a, b in zip(layer.add_rmsnorm_int8(x, r, w), want8))


@pytest.mark.parametrize("n,cols", [(1, 64), (5, 4096), (2100, 512), (3, 77), (3, 16400)])
def test_in_place(layer, n, cols):
    x, r, w = _rows(n, cols, 1), _rows(n, cols, 2), _weight(cols, 3)
    y, h = layer.add_rmsnorm(x, r, w)
    for y_to, h_to in (("x", "r"), ("r", "x"), ("x", None), (None, "x"), (None, "r"), ("r", None)):
        t = {"x": x.clone(), "r": r.clone(), None: None}
        got = layer.add_rmsnorm(t["x"], t["r"], w, out=t[y_to], sum_out=t[h_to])
        assert torch.equal(got[0], y) and torch.equal(got[1], h)
    for h_to in ("x", "r"):
        t = {"x": x.clone(), "r": r.clone()}
        got = layer.add_rmsnorm_int8(t["x"], t["r"], w, sum_out=t[h_to])
        assert all(torch.equal(a, b) for a, b in zip(got, layer.add_rmsnorm_int8(x, r, w)))
    a = x.clone()
    assert torch.equal(layer.add_rmsnorm(a, None, w, out=a)[0], layer.add_rmsnorm(x, None, w)[0])


def test_no_rows_and_what_does_not_fit(layer):
    w = _weight(64, 1)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV)
    y, h = layer.add_rmsnorm(x, x, w)
    assert y.shape == h.shape == (0, 64)
    assert [tuple(t.shape) for t in layer.add_rmsnorm_int8(x, x, w)] == [(0, 64), (0,), (0, 64)]
    gx, gw = layer.add_rmsnorm_grad(x, x, w)
    assert gx.shape == (0, 64) and not gw.any()
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: layer.add_rmsnorm(x, x[:1], w), lambda: layer.add_rmsnorm(x, x, w[:32]), lambda: layer.add_rmsnorm(x.float(), x, w),
                lambda: layer.add_rmsnorm(x, x, w.float()), lambda: layer.add_rmsnorm(x.t(), None, w), lambda: layer.add_rmsnorm(x.cpu(), None, w),
                lambda: layer.add_rmsnorm(x, x, w, out=x[:1]), lambda: layer.add_rmsnorm(x, None, w, sum_out=x),
                lambda: layer.add_rmsnorm(x[0], None, w), lambda: layer.add_rmsnorm_grad(x, x[:1], w), lambda: layer.add_rmsnorm_grad(x, x, w[1:]),
                lambda: layer.add_rmsnorm_grad(x, x, w, grad_h=x[:1])):
        with pytest.raises(ValueError):
            bad()
    y = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: layer.add_rmsnorm(x, x, w, out=y, sum_out=y), lambda: layer.add_rmsnorm(x, x, w, eps=-1.0),
                lambda: layer.add_rmsnorm(x.expand(2, 64)[:1].expand(2, 64), None, w),
                lambda: layer.add_rmsnorm_grad(*[torch.zeros(1, 16392, dtype=torch.bfloat16, device=DEV)] * 2, _weight(16392, 1))):
        with pytest.raises(RuntimeError):
            bad()


def test_rows_of_zeros_and_rows_that_are_not_finite(layer):
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    for n in (6, 2100):
        x = _rows(n, 512, 1)
        x[1] = 0
        x[2, 5] = float("inf")
        x[3, 7] = float("nan")
        x[4] = 1e-38
        y, _ = layer.add_rmsnorm(x, None, w)
        q, scale, _ = layer.add_rmsnorm_int8(x, None, w)
        assert not y[1].any() and not q[1].any() and scale[1] == torch.tensor(2.0 ** -100) / 127
        assert y[2, 5].isnan() and not y[2, :5].any() and y[3].isnan().all()
        assert scale[2:4].isnan().all() and not q[2:4].any()
        assert scale[0].isfinite() and scale[4].isfinite() and y[4].isfinite().all()


# ------------------------------------------------------------------ gradient
def _grad_ref(gy, h, w, eps, gh):
    gy, h, w = gy.double(), h.double(), w.double()
    inv = 1 / torch.sqrt(h.square().mean(dim=1, keepdim=True) + eps)
    n, p = h * inv, w * gy
    gx = inv * (p - n * (p * n).mean(dim=1, keepdim=True))
    mag = inv * (p.abs() + n.abs() * (p * n).abs().mean(dim=1, keepdim=True))
    if gh is not None:
        gx, mag = gx + gh.double(), mag + gh.double().abs()
    return gx, mag, (gy * n).sum(dim=0), (gy * n).abs().sum(dim=0)


@pytest.mark.parametrize("n,cols", [(1, 256), (1, 1), (37, 2048), (5, 7168), (64, 8200), (65, 77), (64, 16384), (63, 40), (300, 4096), (1000, 512), (777, 1000), (50, 1001), (601, 8192), (9, 8200),
                                    (301, 16384), (3, 16383), (3000, 40), (2500, 256)])
@pytest.mark.parametrize("with_h", (True, False))
def test_gradients(layer, n, cols, with_h):
    gy, h, w = _rows(n, cols, 1), _rows(n, cols, 2), _weight(cols, 3)
    gh = _rows(n, cols, 4) if with_h else None
    gx, gw = layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh)
    want, mag, want_w, mag_w = _grad_ref(gy, h, w, 1e-6, gh)
    assert ((gx.double() - want).abs() <= mag * 150 * U + want.abs() * 2.0 ** -8 + 2.0 ** -130).all()
    shares = min(n, 148 * 32)                        # at most: a row each; a share then has ever fewer rows than there are
    assert gw.dtype == torch.float32
    assert ((gw.double() - want_w).abs() <= mag_w * (31 + n / 148 + 1 + shares / 32 + 5) * U).all()
    assert torch.equal(layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh, need_w=False)[0], gx)
    assert torch.equal(layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh, need_x=False)[1], gw)
    again = layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


@pytest.mark.parametrize("n,cols", [(37, 2048), (300, 4096), (601, 8192), (70, 77), (2500, 256), (40, 16384)])
def test_a_gradient_in_the_place_of_another(layer, n, cols):
    """From C: grad_x over grad_y, or over grad_h."""
    gy, h, w, gh = _rows(n, cols, 1), _rows(n, cols, 2), _weight(cols, 3), _rows(n, cols, 4)
    want, _ = layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh, need_w=False)
    for which in (0, 1):
        a, b = gy.clone(), gh.clone()
        to = (a, b)[which]
        assert layer.lib.mg_add_rmsnorm_grad(layer._h, a.data_ptr(), cols, h.data_ptr(), cols, w.data_ptr(), 1e-6, n, cols, b.data_ptr(), cols,
                                             to.data_ptr(), cols, None, None, 0, layer._stream()) == 0
        assert torch.equal(to, want)


@pytest.mark.parametrize("n", (64, 65))
def test_scratch_of_the_gradient(layer, n):
    """None up to 64 rows, refused where it is missing or too small beyond."""
    import ctypes as C
    from moe_gen_b200 import lib as L
    assert L.NORM_GRAD_FEW == 64
    x, w, gw, need = _rows(n, 512, 1), _weight(512, 2), torch.zeros(512, device=DEV), C.c_size_t()
    assert layer.lib.mg_add_rmsnorm_grad_ws_bytes(layer._h, n, 512, C.byref(need)) == 0 and (need.value > 0) == (n > 64)
    ws = torch.empty(max(need.value, 4), dtype=torch.uint8, device=DEV)

    def call(ptr, size):
        return layer.lib.mg_add_rmsnorm_grad(layer._h, x.data_ptr(), 512, x.data_ptr(), 512, w.data_ptr(), 1e-6, n, 512, None, 0, None, 0,
                                             gw.data_ptr(), ptr, size, layer._stream())
    if n > 64:
        assert call(None, 0) == -1 and call(ws.data_ptr(), need.value - 1) == -4 and call(ws.data_ptr() + 2, need.value) == -2
        assert call(ws.data_ptr(), need.value) == 0
    else:
        assert call(None, 0) == 0
    assert torch.equal(gw, layer.add_rmsnorm_grad(x, x, w)[1])


@pytest.mark.parametrize("ld,off", [(600, 0), (600, 8), (513, 0), (512, 1)])
def test_gradients_of_strided_rows(layer, ld, off):
    gy, h, gh, w = _rows(70, 512, 1, ld, off), _rows(70, 512, 2, ld, off), _rows(70, 512, 3, ld, off), _weight(512, 4)
    want = layer.add_rmsnorm_grad(gy.contiguous(), h.contiguous(), w, 1e-6, gh.contiguous())
    got = layer.add_rmsnorm_grad(gy, h, w, 1e-6, gh)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradient_against_differences(layer):
    """sum(gy * y) + sum(gh * h) of the 64-bit formula, moved along random directions of x and of w: central differences, whose third-order
    term at a step of 1e-4 is below 1e-6 of the value here."""
    from moe_gen_b200 import add_norm
    x, r, w = _rows(20, 320, 1), _rows(20, 320, 2), _weight(320, 3)
    gy, gh = _rows(20, 320, 4), _rows(20, 320, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    h, y = add_norm(layer, *leaves, 1e-6)
    gx, gr, gw = torch.autograd.grad((h, y), leaves, (gh, gy))
    assert torch.equal(gx, gr) and gw.dtype == w.dtype
    base, ww = h.detach().double(), w.double()

    def value(hh, wv):
        return (gy.double() * (hh / torch.sqrt(hh.square().mean(dim=1, keepdim=True) + 1e-6) * wv)).sum() + (gh.double() * hh).sum()

    g = torch.Generator(device=DEV).manual_seed(6)
    d = torch.randn(base.shape, generator=g, device=DEV, dtype=torch.float64)
    got, diff = (gx.double() * d).sum(), (value(base + 1e-4 * d, ww) - value(base - 1e-4 * d, ww)) / 2e-4
    assert (got - diff).abs() <= (gx.double() * d).abs().sum() * 2.0 ** -8 + 1e-5 * diff.abs()
    d = torch.randn(ww.shape, generator=g, device=DEV, dtype=torch.float64)
    got, diff = (gw.double() * d).sum(), (value(base, ww + 1e-4 * d) - value(base, ww - 1e-4 * d)) / 2e-4
    assert (got - diff).abs() <= (gw.double() * d).abs().sum() * 2.0 ** -8 + 1e-5 * diff.abs()


def test_autograd_of_parts(layer):
    """One of the two outputs alone, no residual, frozen inputs, a gradient cut out of a flat tensor."""
    from moe_gen_b200 import add_norm
    x, r, w = (_rows(9, 64, 1).clone().requires_grad_(True), _rows(9, 64, 2).clone(), _weight(64, 3).requires_grad_(True))
    g = _rows(9, 64, 4)
    h, y = add_norm(layer, x, r, w)
    assert torch.equal(torch.autograd.grad(y, x, g)[0], layer.add_rmsnorm_grad(g, h.detach(), w.detach())[0])
    h, y = add_norm(layer, x, r, w)
    assert torch.equal(torch.autograd.grad(h, x, g)[0], g)
    h, y = add_norm(layer, x, None, w)
    assert torch.equal(h, x) and h.data_ptr() != x.data_ptr()
    want = layer.add_rmsnorm_grad(g, x.detach(), w.detach(), grad_h=g)
    got = torch.autograd.grad((h, y), (x, w), (g, g))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1].to(torch.bfloat16))
    one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
    h, y = add_norm(layer, x, r, w)
    want = layer.add_rmsnorm_grad(g, h.detach(), w.detach())
    got = torch.autograd.grad(torch.cat([one, y.reshape(-1)]), (x, w), torch.cat([one, g.reshape(-1)]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1].to(torch.bfloat16))


# ------------------------------------------------------------------ beside what the framework had
@pytest.mark.parametrize("fmt", (0, 2))
@pytest.mark.parametrize("T,H", [(1, 512), (37, 512), (2300, 512), (3, 7168), (20, 16384)])
def test_the_block_with_a_residual(built_lib, fmt, T, H):
    """Bit for bit the block on the sum: the norm in it is mg_rmsnorm's."""
    from moe_gen_b200 import MoELayer
    layer = MoELayer(hidden=H, inter=256, n_experts=8, top_k=2, weight_format=fmt, device=DEV)
    g = torch.Generator().manual_seed(T)
    layer.set_router(torch.randn(8, H, generator=g) * 0.05)
    for e in range(8):
        mats = [torch.randn(*s, generator=g).mul(0.05).to(torch.bfloat16).to(DEV) for s in ((256, H), (256, H), (H, 256))]
        if fmt == 2:
            qs = [layer.quantize_rows(m) for m in mats]
            layer.load_expert(e, *[q.contiguous() for q, _ in qs], scales=tuple(s for _, s in qs))
        else:
            layer.load_expert(e, *mats)
    a, r, w = _rows(T, H, 8).clone(), _rows(T, H, 9).clone(), _weight(H, 10)
    want = layer.block_forward(a + r, w, 1e-6)
    assert torch.equal(layer.block_forward(a, w, 1e-6, residual=r), want)
    for at in (0, 1):
        t = [a.clone(), r.clone()]
        assert torch.equal(layer.block_forward(t[0], w, 1e-6, out=t[at], residual=t[1]), want) and torch.equal(t[at], want)
        assert torch.equal(t[1 - at], (a, r)[1 - at])
    with pytest.raises(ValueError):
        layer.block_forward(a, w, residual=r[:, :256])
    layer.close()


@pytest.mark.parametrize("n", (1, 100, 2200))
def test_quantised_rows_go_into_the_products(layer, n):
    """add_rmsnorm_int8 -> int8_matmul: the product of the row's bytes, exact in 64 bits."""
    x, r, w = _rows(n, 1024, 1), _rows(n, 1024, 2), _weight(1024, 3)
    wq, ws = layer.quantize_rows(_rows(200, 1024, 4))
    q, s, h = layer.add_rmsnorm_int8(x, r, w)
    y = layer.int8_matmul(q, s, wq, ws)
    want = (q.double() @ wq.double().t()).float() * s[:, None] * ws
    assert torch.equal(y, want.to(torch.bfloat16))


def test_a_captured_call_and_two_streams(layer):
    x, r, w = _rows(600, 2048, 1).clone(), _rows(600, 2048, 2).clone(), _weight(2048, 3)
    gy = _rows(600, 2048, 4).clone()
    want = layer.add_rmsnorm(x, r, w) + layer.add_rmsnorm_grad(gy, x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.add_rmsnorm(x, r, w) + layer.add_rmsnorm_grad(gy, x, w)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    runs = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                runs.append(layer.add_rmsnorm(x, r, w) + layer.add_rmsnorm_grad(gy, x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for run in runs for a, b in zip(run, want))


def test_rows_beyond_32_bits(layer):
    """Elements at offsets above 2^32: the last rows of 600000 of 7680."""
    n, cols = 600000, 7680
    x, w = torch.zeros(n, cols, dtype=torch.bfloat16, device=DEV), _weight(cols, 1)
    last = _rows(3, cols, 2)
    x[-3:] = last
    y, h = layer.add_rmsnorm(x, x, w)
    want, want_h = layer.add_rmsnorm(last, last, w)
    assert torch.equal(y[-3:], want) and torch.equal(h[-3:], want_h) and not y[:3].any()
    del y, h
    q, s, _ = layer.add_rmsnorm_int8(x, None, w)
    assert torch.equal(q[-3:], layer.add_rmsnorm_int8(last, None, w)[0])
    del q, s
    gx, _ = layer.add_rmsnorm_grad(x, x, w)
    assert torch.equal(gx[-3:], layer.add_rmsnorm_grad(last, last, w)[0])


@pytest.mark.parametrize("shape", [(1, 1), (2, 19), (1, 2100)])
def test_the_patched_decoder_layer_adds_in_the_norms_launch(built_lib, shape):
    """What a patched decoder layer returns is the block on the rounded sum, bit for bit, also where attention hands over rows that
    are not contiguous, begin off a boundary, or have another type (which the addition promotes, and the block refuses)."""
    import types

    import torch.nn as nn
    from moe_gen_b200 import patch_decoder_layer
    g = torch.Generator().manual_seed(3)

    class DeepseekV3MoE(nn.Module):
        pass

    class Layer(nn.Module):
        pass

    class Norm(nn.Module):
        def __init__(self):
            super().__init__()
            self.weight, self.variance_epsilon = nn.Parameter((1 + 0.1 * torch.randn(256, generator=g)).to(torch.bfloat16).to(DEV)), 1e-6

        def forward(self, h):
            return h

    def lin(rows, cols):
        m = nn.Linear(cols, rows, bias=False)
        m.weight = nn.Parameter((torch.randn(rows, cols, generator=g) * 0.05).to(torch.bfloat16).to(DEV), requires_grad=False)
        return m

    def mlp():
        m = nn.Module()
        m.gate_proj, m.up_proj, m.down_proj = lin(128, 256), lin(128, 256), lin(256, 128)
        return m

    moe = DeepseekV3MoE().eval()
    moe.config = types.SimpleNamespace(hidden_size=256, moe_intermediate_size=128, n_routed_experts=8, num_experts_per_tok=2, n_shared_experts=1,
                                       n_group=2, topk_group=1, topk_method="noaux_tc", scoring_func="sigmoid", norm_topk_prob=True,
                                       routed_scaling_factor=2.5)
    moe.gate = nn.Module()
    moe.gate.weight = nn.Parameter(torch.randn(8, 256, generator=g) * 0.05)
    moe.gate.e_score_correction_bias = nn.Parameter(torch.zeros(8))
    moe.experts, moe.shared_experts = nn.ModuleList([mlp() for _ in range(8)]), mlp()
    dl = Layer().eval()
    dl.input_layernorm, dl.post_attention_layernorm, dl.mlp = Norm(), Norm(), moe
    B, S = shape
    kinds = {"plain": lambda t: t * 0.5, "turned": lambda t: (t * 0.5).transpose(0, 1).contiguous().transpose(0, 1),
             "off": lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t * 0.5), "float": lambda t: t.float() * 0.5}
    dl.self_attn = nn.Module()
    layer = patch_decoder_layer(dl, device=DEV)
    x = _rows(B * S, 256, 4).clone().view(B, S, 256)
    want = layer.block_forward(x + x * 0.5, dl.post_attention_layernorm.weight.detach(), 1e-6)
    for name, make in kinds.items():
        dl.self_attn.forward = lambda hidden_states, make=make, **kw: (make(hidden_states), None, None)
        before = x.clone()
        if name == "float":
            with pytest.raises(ValueError):
                dl(x)
        else:
            assert torch.equal(dl(x)[0], want), name
        assert torch.equal(x, before)


@pytest.mark.parametrize("with_h", (True, False))
def test_gradients_of_no_rows(layer, with_h):
    """Of each of the two alone, and through autograd with a frozen weight."""
    from moe_gen_b200 import add_norm
    w = _weight(64, 1)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV)
    gh = x if with_h else None
    gx, gw = layer.add_rmsnorm_grad(x, x, w, 1e-6, gh, need_w=False)
    assert gx.shape == (0, 64) and gw is None
    gx, gw = layer.add_rmsnorm_grad(x, x, w, 1e-6, gh, need_x=False)
    assert gx is None and not gw.any()
    for frozen in (True, False):
        leaves = [x.clone().requires_grad_(True), x.clone().requires_grad_(True), w.clone().requires_grad_(not frozen)]
        h, y = add_norm(layer, *leaves)
        got = torch.autograd.grad((h, y) if with_h else y, leaves[:2 if frozen else 3], (x, x) if with_h else x)
        assert got[0].shape == got[1].shape == (0, 64) and (frozen or not got[2].any())
