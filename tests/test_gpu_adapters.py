"""GPU: low-rank adapters of requests and of experts, and their gradients, against the formulas in 64 bits.

Tolerances.  A sum over n products on the matrix units adds 16 at a time in fp32, in chains that end in sums over 8 warps and 8 blocks: at
most n / 16 + 16 additions, each off by at most 2^-22 (the units align and cut products) of the sum of magnitudes.  s and gs are taken
in two parts of bf16 (2^-8 of 2^-8 of the value), what leaves the call is rounded to one.  With e(s) = (K / 16 + 16) 2^-22 |x| . |down|^T +
2^-16 |s|, where each product of two parts is a sum twice as long:
  out    2^-8 |out| + |f| (e(s) . |up|^T + (rank / 8 + 2) 2^-22 (1 + 2^-8) |s| . |up|^T) + 2^-23 |y|
and likewise for the gradients, whose s and gs enter as the formula has them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = 2.0 ** -8
STEP = 2.0 ** -22


@pytest.fixture(scope="module")
def layer(built_lib):
    from moe_gen_b200 import MoELayer
    made = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, device=DEV)
    yield made
    made.close()


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(n, cols, seed, extra=0, fill=float("nan")):
    """[n, cols] bf16 with rows on 16-byte boundaries, `fill` behind each."""
    ld = (cols + 7) // 8 * 8 + extra
    wide = torch.full((n, ld), fill, dtype=torch.bfloat16, device=DEV)
    wide[:, :cols] = torch.randn(n, cols, generator=_gen(seed), device=DEV)
    return wide[:, :cols]


def _adapters(G, r, K, N, seed):
    down = _rows(G * r, K, seed).as_strided((G, r, K), (r * ((K + 7) // 8 * 8), (K + 7) // 8 * 8, 1))
    up = _rows(G * N, r, seed + 1).as_strided((G, N, r), (N * ((r + 7) // 8 * 8), (r + 7) // 8 * 8, 1))
    down.mul_(K ** -0.5)
    up.mul_(r ** -0.5)
    return down, up, torch.rand(G, generator=_gen(seed + 2), device=DEV) + 0.5


def _ids(n, G, seed, runs=1):
    """Ids from -1 to G, both ends meaning none, in runs."""
    pick = (torch.rand(n, generator=_gen(seed), device=DEV) ** 2 * (G + 2)).long().clamp_(max=G + 1) - 1
    return pick[torch.arange(n, device=DEV) // runs].int()


def _reference(x, y, down, up, scale, ids, go=None):
    """out, grad_x, grad_down, grad_up in 64 bits and the tolerances of each."""
    G, r, K = down.shape
    N = up.shape[1]
    x, y = x.double(), y.double()
    out, tol = y.clone(), torch.zeros_like(y)
    gx, tx = torch.zeros_like(x), torch.zeros_like(x)
    gd, td = (torch.zeros(G, r, K, dtype=torch.float64, device=DEV) for _ in range(2))
    gu, tu = (torch.zeros(G, N, r, dtype=torch.float64, device=DEV) for _ in range(2))
    for g in range(G):
        t = (ids == g).nonzero()[:, 0]
        if t.numel() == 0:
            continue
        A, B, f, xs = down[g].double(), up[g].double(), float(scale[g]), x[t]
        s = xs @ A.t()
        es = (K / 16 + 16) * STEP * (xs.abs() @ A.abs().t()) + HALF ** 2 * s.abs()
        out[t] += f * (s @ B.t())
        tol[t] = abs(f) * (es + (r / 8 + 2) * STEP * s.abs()) @ B.abs().t() * (1 + HALF) + y[t].abs() * 2.0 ** -23
        if go is not None:
            o = go[t].double()
            gs = f * (o @ B)
            eg = (N / 16 + 16) * STEP * abs(f) * (o.abs() @ B.abs()) + HALF ** 2 * gs.abs()
            gx[t] = gs @ A
            tx[t] = (eg + (r / 8 + 2) * STEP * gs.abs()) @ A.abs() * (1 + HALF)
            n = len(t) / 8 + 16
            gd[g], td[g] = gs.t() @ xs, (eg + n * STEP * gs.abs()).t() @ xs.abs() * (1 + HALF)
            gu[g] = f * (o.t() @ s)
            tu[g] = abs(f) * (o.abs().t() @ (es + n * STEP * s.abs())) * (1 + HALF)
    return [(v, e + HALF * v.abs() + 2.0 ** -130) for v, e in ((out, tol), (gx, tx), (gd, td), (gu, tu))]


def _near(got, ref):
    want, tol = ref
    return bool(((got.double() - want).abs() <= tol).all())


CASES = [  # rows, cols, n_out, rank, adapters, run
    (1, 256, 256, 16, 1, 1), (1, 4096, 4096, 16, 8, 1), (1, 8, 8, 1, 1, 1), (2, 33, 17, 3, 2, 1), (15, 100, 1000, 8, 4, 1), (16, 1001, 77, 12, 3, 1),
    (17, 2048, 512, 16, 64, 1), (64, 512, 2048, 32, 5, 7), (200, 777, 333, 64, 3, 50), (201, 640, 1000, 12, 64, 1), (255, 1, 1, 1, 2, 3),
    (256, 96, 4000, 128, 2, 256), (257, 1000, 97, 100, 9, 1), (300, 264, 40, 65, 300, 1), (513, 512, 512, 33, 4, 64), (1000, 130, 2050, 4, 1, 1),
    (2000, 2048, 1024, 64, 16, 100), (3001, 320, 288, 16, 1024, 3), (4096, 31, 63, 128, 7, 1000)]


@pytest.mark.parametrize("n,K,N,r,G,run", CASES)
def test_adapters_by_ids_and_by_plan(layer, n, K, N, r, G, run):
    x, y, go = _rows(n, K, 1), _rows(n, N, 2), _rows(n, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    ids = _ids(n, G, 5, run)
    refs = _reference(x, y, down, up, scale, ids, go)
    plan = layer.adapter_plan(ids, G)
    none = (ids < 0) | (ids >= G)
    out, s = layer.adapter_add(y, x, down, up, ids, scale, keep=True)
    by_plan, s_plan = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
    for got, kept in ((out, s), (by_plan, s_plan)):
        assert _near(got, refs[0]) and torch.equal(got[none], y[none])
        assert not kept[none].any() and not kept.view(n, 2, -1)[:, :, r:].any()
    grads = layer.adapter_grad(go, x, down, up, plan, scale, s_plan)
    assert all(_near(g, ref) for g, ref in zip(grads, refs[1:]))
    assert not grads[0][none].any()
    # always the same bits, whatever is asked for and whoever makes the plan
    assert torch.equal(layer.adapter_add(y, x, down, up, plan, scale), by_plan)
    assert all(torch.equal(a, b) for a, b in zip(layer.adapter_grad(go, x, down, up, ids, scale, s_plan), grads))
    for k in range(3):
        need = [i == k for i in range(3)]
        part = layer.adapter_grad(go, x, down, up, plan, scale, s_plan, *need)
        assert [p is not None for p in part] == need and torch.equal(part[k], grads[k])


def _segments(counts, extra_tiles=1):
    counts = torch.tensor(counts, dtype=torch.int32)
    pad = torch.zeros(len(counts) + 1, dtype=torch.int32)
    pad[1:] = torch.cumsum((counts + 127) // 128 * 128, 0)
    return counts.to(DEV), pad.to(DEV), int(pad[-1]) + 128 * extra_tiles


@pytest.mark.parametrize("counts", [[0], [1], [128], [0, 0, 5], [3, 0, 64, 129, 0, 1000, 1], [7] * 64, [2000, 0, 0, 1], [0] * 8])
@pytest.mark.parametrize("K,N,r", [(256, 512, 8), (1000, 264, 16), (520, 96, 64)])
def test_adapters_of_sorted_rows(layer, counts, K, N, r):
    G = len(counts)
    c, pad, rows = _segments(counts)
    x, y, go = _rows(rows, K, 1), _rows(rows, N, 2), _rows(rows, N, 3)
    ids = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    for g, n in enumerate(counts):
        ids[int(pad[g]):int(pad[g]) + n] = g
    none = ids < 0
    x[none] = float("nan")                             # not read
    go[none] = float("nan")
    down, up, scale = _adapters(G, r, K, N, 4)
    refs = _reference(x, y, down, up, scale, ids, go)
    plan = layer.adapter_plan_sorted(c, pad, rows)
    out, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
    assert _near(out, refs[0]) and torch.equal(out[none], y[none])
    grads = layer.adapter_grad(go, x, down, up, plan, scale, s)
    assert all(_near(g, ref) for g, ref in zip(grads, refs[1:]))
    assert not grads[0][none].any() and not any(grads[k][g].any() for g, n in enumerate(counts) if n == 0 for k in (1, 2))


@pytest.mark.parametrize("counts,extra", [([1] * 100 + [0] * 60, 1), ([3] * 300, 1), ([5, 0, 2], 300), ([2] * 160, 100), ([0] * 20 + [130] * 5, 7),
                                          ([1, 200] * 40, 0), ([9] * 75, 75), ([0] * 300, 1), ([0] * 200 + [4], 2), ([0, 3, 0] * 100, 1)])
def test_tiles_that_share_blocks_and_tiles_that_do_not(layer, counts, extra):
    """More and fewer tiles than run at once, by rounds, by clusters, and by halves of clusters; rows without an adapter behind them."""
    c, pad, rows = _segments(counts, extra)
    ids = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    for g, n in enumerate(counts):
        ids[int(pad[g]):int(pad[g]) + n] = g
    K, N, r = 328, 203, 16 if extra % 2 else 13
    x, y, go = _rows(rows, K, 1), _rows(rows, N, 2), _rows(rows, N, 3)
    down, up, scale = _adapters(len(counts), r, K, N, 4)
    refs = _reference(x, y, down, up, scale, ids, go)
    plan = layer.adapter_plan_sorted(c, pad, rows)
    none = ids < 0
    out, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
    assert _near(out, refs[0]) and torch.equal(out[none], y[none]) and not s[none].any()
    grads = layer.adapter_grad(go, x, down, up, plan, scale, s)
    assert all(_near(g, ref) for g, ref in zip(grads, refs[1:]))
    assert not grads[0][none].any() and not any(grads[k][g].any() for g, n in enumerate(counts) if n == 0 for k in (1, 2))
    place = _rows(rows, N, 2)
    assert torch.equal(layer.adapter_add(place, x, down, up, plan, scale, out=place), out)
    part = layer.adapter_grad(go, x, down, up, plan, scale, s, False, True, True)
    assert torch.equal(part[1], grads[1]) and torch.equal(part[2], grads[2])


def test_plans_from_permute_plan(layer):
    idx = torch.randint(0, 8, (50, 2), generator=_gen(1), device=DEV, dtype=torch.int32)
    idx[:, 1] = (idx[:, 0] + 1) % 8
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = layer.padded_rows(100)
    x = torch.randn(50, 256, generator=_gen(2), device=DEV).to(torch.bfloat16)
    perm = layer.permute_rows(x, dst, rows, counts, pad)
    down, up, scale = _adapters(8, 16, 256, 256, 3)
    ids = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    ids[dst.reshape(-1).long()] = idx.reshape(-1)
    y = _rows(rows, 256, 5)
    plan = layer.adapter_plan_sorted(counts, pad, rows)
    out = layer.adapter_add(y, perm, down, up, plan, scale)
    assert _near(out, _reference(perm, y, down, up, scale, ids)[0])
    assert torch.equal(out, layer.adapter_add(y, perm, down, up, layer.adapter_plan(ids, 8), scale)) or \
        _near(layer.adapter_add(y, perm, down, up, layer.adapter_plan(ids, 8), scale), _reference(perm, y, down, up, scale, ids)[0])


@pytest.mark.parametrize("counts,pad,rows", [([5, 5], [0, 128, 100], 300), ([5, 500], [0, 128, 256], 200), ([-3, 4], [0, 128, 256], 256),
                                             ([9, 9], [-128, 0, 128], 200), ([9, 9], [1 << 30, 1 << 30, 1 << 30], 64), ([4, 4], [3, 17, 40], 41)])
def test_offsets_that_are_none(layer, counts, pad, rows):
    """Segments that descend, leave the rows or begin anywhere are cut off: what is left of adapter g is worked on."""
    c, p = torch.tensor(counts, dtype=torch.int32, device=DEV), torch.tensor(pad, dtype=torch.int32, device=DEV)
    x, y = _rows(rows, 64, 1), _rows(rows, 64, 2)
    down, up, scale = _adapters(2, 16, 64, 64, 3)
    ids = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    for g in range(2):
        lo = min(max(pad[g], 0), rows)
        hi = min(max(pad[g + 1], lo), rows)
        ids[lo:min(hi, lo + max(counts[g], 0))] = g
    before = y.clone()
    out = torch.zeros(rows, 64, dtype=torch.bfloat16, device=DEV)
    layer.adapter_add(y, x, down, up, layer.adapter_plan_sorted(c, p, rows), scale, out=out)
    torch.cuda.synchronize()
    assert torch.equal(y, before)
    seen = ids >= 0
    want, tol = _reference(x, y, down, up, scale, ids)[0]
    assert ((out.double() - want).abs() <= tol)[seen].all()


@pytest.mark.parametrize("n", (5, 256, 700))
def test_in_place_strides_and_rows_left_alone(layer, n):
    K, N, r, G = 200, 136, 24, 6
    x, y = _rows(n, K, 1, extra=16), _rows(n, N, 2, extra=64, fill=7.0)
    down, up, scale = _adapters(G, r, K, N, 3)
    ids = _ids(n, G, 4)
    want = layer.adapter_add(y, x, down, up, ids, scale)
    hold = torch.full((n + 2, N + 40), 9.0, dtype=torch.bfloat16, device=DEV)
    out = hold[1:-1, 8:8 + N]
    assert layer.adapter_add(y, x, down, up, ids, scale, out=out) is out and torch.equal(out, want)
    hold[1:-1, 8:8 + N] = 9.0
    assert (hold == 9.0).all()
    wide = y.as_strided((n, N + 64), (y.stride(0), 1)) if y.stride(0) >= N + 64 else None
    same = layer.adapter_add(y, x, down, up, ids, scale, out=y)
    assert same is y and torch.equal(y, want)
    assert wide is None or (wide[:, N:] == 7.0).all()


def test_scales_and_one_adapter_for_all(layer):
    n, K, N, r = 40, 128, 64, 16
    x, y = _rows(n, K, 1), _rows(n, N, 2)
    down, up, scale = _adapters(3, r, K, N, 3)
    ids = _ids(n, 3, 4)
    a = layer.adapter_add(y, x, down, up, ids, 0.75)
    assert torch.equal(a, layer.adapter_add(y, x, down, up, ids, torch.full((3,), 0.75, device=DEV)))
    assert torch.equal(layer.adapter_add(y, x, down, up, ids), layer.adapter_add(y, x, down, up, ids, 1.0))
    shared = layer.adapter_add(y, x, down[:1].expand(3, r, K), up[:1].expand(3, N, r), ids, 0.75)       # stride 0 between adapters
    first = torch.where((ids >= 0) & (ids < 3), 0, -1).int()
    assert _near(shared, _reference(x, y, down[:1], up[:1], torch.tensor([0.75]), first)[0])


def test_adapters_whose_rows_lie_between_one_anothers(layer):
    """down [rank, adapters, cols] and up [n_out, adapters, rank] seen as adapters: their gradients come as adapters one behind another."""
    x, y, go = _rows(70, 64, 1), _rows(70, 96, 2), _rows(70, 96, 3)
    down, up, scale = _adapters(3, 16, 64, 96, 4)
    ids = _ids(70, 3, 5)
    out, s = layer.adapter_add(y, x, down, up, ids, scale, keep=True)
    want = layer.adapter_grad(go, x, down, up, ids, scale, s)
    d2, u2 = down.transpose(0, 1).contiguous().transpose(0, 1), up.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(layer.adapter_add(y, x, d2, u2, ids, scale), out)
    got = layer.adapter_grad(go, x, d2, u2, ids, scale, s)
    assert all(torch.equal(a, b) and b.is_contiguous() for a, b in zip(want, got))


def test_what_is_not_finite_stays_in_its_row(layer):
    n, K, N, r, G = 90, 160, 96, 12, 4
    x, y = _rows(n, K, 1), _rows(n, N, 2)
    down, up, scale = _adapters(G, r, K, N, 3)
    ids = (torch.arange(n, device=DEV) % (G - 1)).int()
    for who in (ids, layer.adapter_plan(ids, G)):
        clean, s0 = layer.adapter_add(y, x, down, up, who, scale, keep=True)
        bad, bad_down, bad_up = x.clone(), down.clone(), up.clone()
        bad[3] = float("inf")
        bad[10, 5] = float("nan")
        bad_down[3], bad_up[3] = float("nan"), float("inf")            # an adapter without rows
        got, s = layer.adapter_add(y, _realign(bad), bad_down, _realign3(bad_up), who, scale, keep=True)
        keep = torch.ones(n, dtype=torch.bool, device=DEV)
        keep[[3, 10]] = False
        assert torch.equal(got[keep], clean[keep]) and torch.equal(s[keep], s0[keep])
        assert got[10].isnan().all() and not got[3].isfinite().any()
    none = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    y2 = y.clone()
    y2[4] = float("nan")
    y2[5] = -0.0
    y2 = _realign(y2)
    assert torch.equal(layer.adapter_add(y2, x, bad_down, _realign3(bad_up), none, scale).view(torch.int16), y2.contiguous().view(torch.int16))


def _realign(t):
    v = torch.zeros(t.shape[0], (t.shape[1] + 7) // 8 * 8, dtype=t.dtype, device=DEV)[:, :t.shape[1]]
    return v.copy_(t)


def _realign3(t):
    v = torch.zeros(*t.shape[:2], (t.shape[2] + 7) // 8 * 8, dtype=t.dtype, device=DEV)[:, :, :t.shape[2]]
    return v.copy_(t)


def test_refusals(layer):
    x, y = _rows(4, 64, 1), _rows(4, 32, 2)
    down, up, scale = _adapters(2, 16, 64, 32, 3)
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    add = layer.adapter_add
    for bad in (lambda: add(y, x, down, up, ids.long()), lambda: add(y, x, down, up, ids[:3]), lambda: add(y[:3], x, down, up, ids),
                lambda: add(y, x[:, :56], down, up, ids), lambda: add(y.float(), x, down, up, ids), lambda: add(y, x, down[:1], up, ids),
                lambda: add(y, x, down, up[:, :, :8], ids), lambda: add(y, x, down[0], up[0], ids), lambda: add(y, x, down, up, ids, scale[:1]),
                lambda: add(y, x, down, up, ids, scale.double()), lambda: add(y, x, down, up, layer.adapter_plan(ids[:3], 2)),
                lambda: add(y, x, down, up, layer.adapter_plan(ids, 3)), lambda: add(y, x, down, up, ids, out=y[:2]),
                lambda: add(y, x, down.transpose(1, 2), up, ids), lambda: add(y, x.cpu(), down, up, ids),
                lambda: layer.adapter_grad(y, x, down, up, ids, 1.0, torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV)),
                lambda: layer.adapter_plan(ids.long(), 2), lambda: layer.adapter_plan_sorted(ids, ids, 4)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: add(y, x[:, 1:], down[:, :, 1:].clone(), up, ids), lambda: add(y, x, torch.zeros(2, 130, 64, dtype=torch.bfloat16, device=DEV),
                                                                                  torch.zeros(2, 32, 130, dtype=torch.bfloat16, device=DEV), ids),
                lambda: add(y, x, down, torch.zeros(2, 32, 17, dtype=torch.bfloat16, device=DEV)[:, :, :16], ids),
                lambda: layer.adapter_plan(ids, 0), lambda: layer.adapter_plan(ids, 1025)):
        with pytest.raises(RuntimeError):
            bad()
    empty = add(y[:0], x[:0], down, up, ids[:0], keep=True)
    assert empty[0].shape == (0, 32) and empty[1].shape == (0, 32)
    gx, gd, gu = layer.adapter_grad(y[:0], x[:0], down, up, ids[:0], scale, empty[1])
    assert gx.shape == (0, 64) and not gd.any() and not gu.any()


# ------------------------------------------------------------------ differentiable, and beside what the framework had
def test_autograd(layer):
    from moe_gen_b200 import adapt_rows
    c, pad, rows = _segments([5, 0, 200])
    plan = layer.adapter_plan_sorted(c, pad, rows)
    for N in (64, 77):
        x, y, go = _rows(rows, 96, 1, fill=0.0), _rows(rows, N, 2, fill=0.0), _rows(rows, N, 3, fill=0.0)
        down, up, scale = _adapters(3, 16, 96, N, 4)
        leaves = [t.detach().requires_grad_(True) for t in (y, x, down, up)]
        out = adapt_rows(layer, *leaves, plan, scale)
        _, s = layer.adapter_add(y, x, down, up, plan, scale, keep=True)
        want = layer.adapter_grad(go, x, down, up, plan, scale, s)
        got = torch.autograd.grad(out, leaves, go)
        assert torch.equal(got[0], go) and all(torch.equal(a, b) for a, b in zip(got[1:], want))
        out = adapt_rows(layer, y, x, leaves[2], up, plan, scale)
        one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
        got = torch.autograd.grad(torch.cat([one, out.reshape(-1)]), leaves[2], torch.cat([one, go.reshape(-1)]))
        assert torch.equal(got[0], want[1])


def test_scales_stay_what_they_were(layer):
    from moe_gen_b200 import adapt_rows
    x, y = _rows(20, 64, 1), _rows(20, 64, 2)
    down, up, scale = _adapters(3, 8, 64, 64, 4)
    plan = layer.adapter_plan(_ids(20, 3, 5), 3)
    with pytest.raises(ValueError, match="detach"):
        adapt_rows(layer, y, x, down, up, plan, scale.clone().requires_grad_(True))
    leaf = x.clone().requires_grad_(True)
    out = adapt_rows(layer, y, leaf, down, up, plan, scale)
    scale.mul_(2.0)                         # the gradient would be another product's
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, leaf, y)


@pytest.mark.parametrize("n", (1, 100, 900))
def test_a_replayed_call_takes_the_ids_that_are_there(layer, n):
    x, y, go = _rows(n, 512, 1).clone(), _rows(n, 384, 2).clone(), _rows(n, 384, 6).clone()
    down, up, scale = _adapters(6, 32, 512, 384, 3)
    ids = _ids(n, 6, 4).clone()

    def step():
        out, s = layer.adapter_add(y, x, down, up, ids, scale, keep=True)
        return (out, s) + layer.adapter_grad(go, x, down, up, ids, scale, s)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6, 7):
        ids.copy_(_ids(n, 6, seed) if seed < 7 else torch.full_like(ids, -1))
        x.copy_(_rows(n, 512, 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
        assert seed < 7 or (torch.equal(kept[0], y) and not any(t.any() for t in kept[1:]))


def test_gradient_against_differences(layer):
    """L = sum(go * out) is linear in down and in up by themselves: its difference along a direction is the gradient's product with it, up to
    the gradients' roundings."""
    n, K, N, r, G = 150, 72, 56, 16, 3
    x, y, go = _rows(n, K, 1), _rows(n, N, 2), _rows(n, N, 3)
    down, up, scale = _adapters(G, r, K, N, 4)
    ids = _ids(n, G, 7)
    _, s = layer.adapter_add(y, x, down, up, ids, scale, keep=True)
    gx, gd, gu = layer.adapter_grad(go, x, down, up, ids, scale, s)
    refs = _reference(x, y, down, up, scale, ids, go)

    def value(xx, dd, uu):
        return (go.double() * _exact(xx, dd, uu)).sum()

    def _exact(xx, dd, uu):
        out = y.double()
        for g in range(G):
            t = (ids == g).nonzero()[:, 0]
            out[t] = out[t] + float(scale[g]) * (xx[t] @ dd[g].t() @ uu[g].t())
        return out

    base = [x.double(), down.double(), up.double()]
    for k, got in enumerate((gx, gd, gu)):
        d = torch.randn(base[k].shape, generator=_gen(9 + k), device=DEV, dtype=torch.float64)
        plus, minus = list(base), list(base)
        plus[k], minus[k] = base[k] + d, base[k] - d
        diff = (value(*plus) - value(*minus)) / 2
        assert (diff - (got.double() * d).sum()).abs() <= (refs[k + 1][1] * d.abs()).sum() + 1e-9 * diff.abs()


def test_a_run_of_them_together(layer):
    """A decoder step of several requests: add and norm to 8 bits, an int8 projection, adapters on the normalised rows; then a
    training step around frozen experts whose rows carry adapters, captured and replayed."""
    from moe_gen_b200 import MoELayer, adapt_rows, add_norm, combine_rows, route, sort_rows
    T, H, N, G = 70, 512, 320, 5
    x, r, w = (_rows(T, H, 1), _rows(T, H, 2), torch.rand(H, generator=_gen(3), device=DEV).to(torch.bfloat16) + 0.5)
    wq, ws = layer.quantize_rows(_rows(N, H, 4))
    down, up, scale = _adapters(G, 16, H, N, 5)
    ids = _ids(T, G, 6)
    q, qs, h = layer.add_rmsnorm_int8(x, r, w)
    n, h2 = layer.add_rmsnorm(x, r, w)
    assert torch.equal(h, h2)
    base = layer.int8_matmul(q, qs, wq, ws)
    out = layer.adapter_add(base, n, down, up, ids, scale, out=base.clone())
    assert _near(out, _reference(n, base, down, up, scale, ids)[0])

    moe = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2, gating=3, norm_topk_prob=True, device=DEV)
    g = torch.Generator().manual_seed(7)
    for e in range(8):
        moe.load_expert(e, *[torch.randn(*s, generator=g).mul(0.1).to(torch.bfloat16).to(DEV) for s in ((128, 256), (128, 256), (256, 128))])
    gate = (torch.randn(8, 256, generator=g) * 0.1).to(DEV)
    leaves = [_rows(60, 256, 8).clone(), _rows(60, 256, 9).clone(), w[:256].clone(), *(t.clone() for t in _adapters(8, 8, 256, 256, 10)[:2])]
    leaves = [t.requires_grad_(True) for t in leaves]
    goal = _rows(60, 256, 13)

    def step():
        a, res, nw, dn, u = leaves
        hh, yy = add_norm(moe, a, res, nw)
        idx, wt = route(moe, yy.detach().float() @ gate.t())
        counts, _, pad, dst = moe.permute_plan(idx)
        rows = sort_rows(moe, yy, dst, moe.padded_rows(idx.numel()), counts, pad)
        frozen = moe.expert_ffn(rows.detach(), pad, counts)[1]
        out_rows = adapt_rows(moe, frozen, rows, dn, u, moe.adapter_plan_sorted(counts, pad, rows.shape[0]), 0.5)
        moved = hh + combine_rows(moe, out_rows, dst, idx, wt, counts, pad)
        return torch.autograd.grad(moved, leaves, goal)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        with torch.no_grad():
            leaves[0].copy_(_rows(60, 256, 20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))
    assert all(t.isfinite().all() and t.any() for t in kept)
    moe.close()


@pytest.mark.parametrize("n", (100, 900))
def test_two_streams(layer, n):
    x, y = _rows(n, 512, 1), _rows(n, 384, 2)
    down, up, scale = _adapters(6, 32, 512, 384, 3)
    ids = [_ids(n, 6, 4), _ids(n, 6, 5)]
    want = [layer.adapter_add(y, x, down, up, i, scale, keep=True) for i in ids]
    want = [w + layer.adapter_grad(y, x, down, up, i, scale, w[1]) for w, i in zip(want, ids)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                o = layer.adapter_add(y, x, down, up, ids[k], scale, keep=True)
                got[k].append(o + layer.adapter_grad(y, x, down, up, ids[k], scale, o[1]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for run in got[k] for a, b in zip(run, want[k]))


def test_rows_beyond_32_bits(layer):
    """Offsets above 2^32 elements in x, y and the results: the last rows of 600000 of 7680."""
    n, K = 600000, 7680
    x = torch.zeros(n, K, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _rows(3, K, 1)
    down, up, scale = _adapters(2, 16, K, K, 2)
    ids = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    ids[-3:] = torch.tensor([1, 0, 1], dtype=torch.int32, device=DEV)
    out, s = layer.adapter_add(x, x, down, up, ids, scale, keep=True)
    want = layer.adapter_add(x[-3:], x[-3:], down, up, layer.adapter_plan(ids[-3:].clone(), 2), scale)
    ref = _reference(x[-3:], x[-3:], down, up, scale, ids[-3:], x[-3:])
    assert _near(out[-3:], ref[0]) and _near(want, ref[0]) and not out[:3].any()
    del out
    gx, gd, gu = layer.adapter_grad(x, x, down, up, ids, scale, s)
    assert _near(gx[-3:], ref[1]) and _near(gd, ref[2]) and _near(gu, ref[3]) and not gx[:3].any()
