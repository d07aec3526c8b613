"""GPU: gradients around the experts, against the formulas in 64 bits and against differences of the forward.

Tolerances.  Rows: one product of 8 and 24 bits rounded to fp32 and bf16, restated bit for bit.  Sums over k rows: fp32 steps of
2^-24 of the sum of magnitudes, and half a bf16 step.  Sums over H: exact products added in fp32 by chains of at most 8 * 7 per
thread, 5 steps of a warp and 32 of a block: 96 * 2^-24 of the sum of magnitudes.  Scores: exp of l - m, whose argument is off by
2^-24 of itself (|l - m| <= 32: 2^-19), plus a few units: 2^-18 relative, of every term of the formula."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _layer(E=8, k=2, H=256, gating=0, n_group=1, topk_group=1, norm=False, scale=1.0, combine=0, I=128):
    from moe_gen_b200 import MoELayer
    return MoELayer(hidden=H, inter=I, n_experts=E, top_k=k, n_group=n_group, topk_group=topk_group, gating=gating,
                    norm_topk_prob=norm, routed_scale=scale, combine_mode=combine, device=DEV)


def _picks(T, E, k, seed):
    """Distinct experts per token, skewed so that some experts are empty."""
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(T, E, generator=g) + torch.linspace(0.8, 0.0, E)).topk(k, dim=1)[1].int().to(DEV)


CASES = [(1, 8, 1, 256), (1, 64, 6, 2048), (3, 8, 2, 4096), (37, 64, 6, 512), (128, 16, 16, 256), (300, 256, 8, 7168), (129, 4, 4, 768),
         (1030, 160, 6, 1280)]


def _setup(T, E, k, H, **kw):
    layer = _layer(E=E, k=k, H=H, **kw)
    idx = _picks(T, E, k, T + E)
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = layer.padded_rows(T * k)
    live = torch.zeros(rows, dtype=torch.bool, device=DEV)
    live[dst.reshape(-1).long()] = True
    return layer, idx, counts, pad, dst, rows, live


@pytest.mark.parametrize("T,E,k,H", CASES)
def test_sort_and_its_gradient(T, E, k, H):
    layer, idx, counts, pad, dst, rows, live = _setup(T, E, k, H)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    poison = torch.full((rows + 4, H), float("nan"), dtype=torch.bfloat16, device=DEV)
    del poison                                                       # what torch.empty is given next
    perm = layer.permute_rows(x, dst, rows, counts, pad)
    assert torch.equal(perm, layer.permute_rows(x, dst, rows)) and not perm[~live].any()
    gr = torch.randn(rows, H, generator=g).to(torch.bfloat16).to(DEV)
    gr[~live] = float("nan")                                         # rows without a pick are not read
    gx = layer.permute_rows_grad(gr, dst)
    terms = gr[dst.long()].double()                                  # [T, k, H]
    want, mag = terms.sum(dim=1), terms.abs().sum(dim=1)
    assert ((gx.double() - want).abs() <= mag * k * 2.0 ** -24 + want.abs() * 2.0 ** -8 * 1.001).all()
    layer.close()


@pytest.mark.parametrize("T,E,k,H", CASES)
@pytest.mark.parametrize("combine", (0, 1, 2))
def test_combine_gradient(T, E, k, H, combine):
    layer, idx, counts, pad, dst, rows, live = _setup(T, E, k, H, combine=combine)
    g = torch.Generator().manual_seed(2)
    out = torch.randn(rows, H, generator=g).to(torch.bfloat16).to(DEV)
    out[~live] = float("nan")
    w = torch.rand(T, k, generator=g).to(DEV)
    gy = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    gr, gw = layer.combine_grad(gy, out, dst, w, counts, pad)
    wr = w.to(torch.bfloat16).float() if combine else w
    want = torch.zeros(rows, H, dtype=torch.bfloat16, device=DEV)
    want[dst.long()] = (gy.float()[:, None, :] * wr[:, :, None]).to(torch.bfloat16)
    assert torch.equal(gr, want)
    terms = gy.double()[:, None, :] * out[dst.long()].double()
    assert ((gw.double() - terms.sum(dim=2)).abs() <= terms.abs().sum(dim=2) * 96 * 2.0 ** -24).all()
    only_r, none = layer.combine_grad(gy, out, dst, w, counts, pad, need_w=False)
    assert none is None and torch.equal(only_r, gr)
    none, only_w = layer.combine_grad(gy, out, dst, w, counts, pad, need_rows=False)
    assert none is None and torch.equal(only_w, gw)
    again = layer.combine_grad(gy, out, dst, w, counts, pad)
    assert torch.equal(again[0], gr) and torch.equal(again[1], gw)
    layer.close()


def test_left_out_picks_partial_plans_and_no_tokens():
    layer = _layer(E=8, k=2)
    idx = torch.tensor([[0, 5], [6, 7], [1, 2], [5, 0]], dtype=torch.int32, device=DEV)
    counts, _, pad, dst = layer.permute_plan(idx, expert_lo=4, n_plan=4)      # experts 0-3 are another's
    rows = layer.padded_rows(8)
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    perm = layer.permute_rows(x, dst, rows, counts, pad)
    assert torch.equal(perm, layer.permute_rows(x, dst, rows))
    gr, gw = layer.combine_grad(x, perm, dst, torch.ones(4, 2, device=DEV), counts, pad)
    assert gw[2].abs().max() == 0 and float(gw[0, 0]) == 0 and float(gw[0, 1]) > 0 and torch.equal(gr, perm)
    assert layer.permute_rows_grad(perm, dst)[2].abs().max() == 0
    # a table whose entries lie beyond the rows that were handed over: left out
    far = dst.clone()
    far[1, 0] = rows + 5
    gr, gw = layer.combine_grad(x, perm, far, torch.ones(4, 2, device=DEV), counts, pad)
    assert float(gw[1, 0]) == 0
    assert layer.permute_rows(x, far, rows, counts, pad).shape == (rows, 256)
    none = torch.zeros(0, 2, dtype=torch.int32, device=DEV)
    c0, p0, d0 = torch.zeros(8, dtype=torch.int32, device=DEV), torch.zeros(9, dtype=torch.int32, device=DEV), none
    assert not layer.permute_rows(x[:0], d0, 256, c0, p0).any()
    gr, gw = layer.combine_grad(x[:0], perm, d0, torch.zeros(0, 2, device=DEV), c0, p0)
    assert not gr.any() and gw.shape == (0, 2) and layer.permute_rows_grad(perm, d0).shape == (0, 256)
    layer.close()


def test_an_expert_named_twice():
    """Two picks of one row: its gradient is that of both weights, and it counts once in the token's."""
    layer = _layer(E=8, k=3)
    idx = torch.tensor([[1, 4, 1], [2, 2, 2]], dtype=torch.int32, device=DEV)
    counts, _, pad, dst = layer.permute_plan(idx)
    assert dst[0, 0] == dst[0, 2] and dst[1, 0] == dst[1, 1] == dst[1, 2]
    rows = layer.padded_rows(6)
    g = torch.Generator().manual_seed(4)
    out, gy = (torch.randn(n, 256, generator=g).to(torch.bfloat16).to(DEV) for n in (rows, 2))
    w = torch.tensor([[0.5, 1.0, 0.25], [1.0, 2.0, 4.0]], device=DEV)
    gr, gw = layer.combine_grad(gy, out, dst, w, counts, pad)
    assert torch.equal(gr[dst[0, 0].long()], (gy[0].float() * 0.75).to(torch.bfloat16))
    assert torch.equal(gr[dst[1, 0].long()], (gy[1].float() * 7.0).to(torch.bfloat16))
    assert gw[0, 0] == gw[0, 2] and gw[1, 0] == gw[1, 1]
    gx = layer.permute_rows_grad(out, dst)
    assert torch.equal(gx[1], out[dst[1, 0].long()])
    assert torch.equal(gx[0], (out[dst[0, 0].long()].float() + out[dst[0, 1].long()].float()).to(torch.bfloat16))
    layer.close()


# ------------------------------------------------------------------ routing weights
GATES = [dict(E=64, k=6, gating=0), dict(E=64, k=6, gating=0, norm=True), dict(E=64, k=1, gating=0, norm=True, scale=2.0),
         dict(E=160, k=6, gating=1, n_group=8, topk_group=3, scale=16.0), dict(E=16, k=6, gating=1, n_group=8, topk_group=2, norm=True),
         dict(E=256, k=8, gating=2, n_group=8, topk_group=4, norm=True, scale=2.5), dict(E=32, k=4, gating=2, n_group=4, topk_group=2, scale=1.5),
         dict(E=8, k=2, gating=3, norm=True), dict(E=512, k=16, gating=0), dict(E=512, k=12, gating=2, n_group=1, topk_group=1, scale=0.5), dict(E=4, k=4, gating=3, norm=True)]


def _weights64(logits, idx, live, cfg):
    """Routing weights of given picks in 64 bits, differentiable."""
    sig, norm = cfg["gating"] == 2, cfg["gating"] == 3 or (cfg.get("norm", False) and cfg["k"] > 1)
    s = torch.sigmoid(logits) if sig else torch.softmax(logits, dim=1)
    p = s.gather(1, idx) * live
    d = p.sum(dim=1, keepdim=True) + (0.0 if cfg["gating"] == 3 else 1e-20)
    c = cfg.get("scale", 1.0)
    if norm:
        return p / d * (c if sig else 1.0), s, p, d, (c if sig else 1.0)
    return p * c, s, p, None, c


@pytest.mark.parametrize("cfg,T", list(itertools.product(range(len(GATES)), (1, 9, 333))))
def test_routing_weights_gradient(cfg, T):
    cfg = GATES[cfg]
    layer = _layer(**cfg)
    if cfg["gating"] == 2:
        layer.bias = (torch.randn(cfg["E"], generator=torch.Generator().manual_seed(3)) * 0.01).to(DEV)
    g = torch.Generator().manual_seed(T)
    logits = (torch.randn(T, cfg["E"], generator=g) * 3).clamp(-15, 15)
    idx, w = layer.route_topk(logits.to(DEV))
    gw = torch.randn(T, cfg["k"], generator=g)
    got = layer.route_topk_grad(logits.to(DEV), idx, w, gw.to(DEV)).cpu().double()
    i, live = idx.cpu().long(), (w.cpu() != 0).double()
    l64, g64 = logits.double().requires_grad_(True), gw.double()
    w64, s, p, d, c = _weights64(l64, i, live, cfg)
    # the weights themselves: a score's error and, normalised, the sum's
    assert ((w.cpu().double() - w64).abs() <= w64.abs() * 2.0 ** -17).all()
    want = torch.autograd.grad((w64 * g64).sum(), l64)[0]
    s, p = s.detach(), p.detach()
    if d is not None:
        d = d.detach()
        a = c / d * (g64.abs() + (g64.abs() * p).sum(dim=1, keepdim=True) / d) * live
    else:
        a = c * g64.abs() * live
    at = torch.zeros_like(s).scatter_add_(1, i, a)
    total = (a * p).sum(dim=1, keepdim=True)
    mag = at * s * (1 - s) if cfg["gating"] == 2 else s * (at + total)
    assert ((got - want).abs() <= mag * 2.0 ** -17).all()
    # along a direction, against a difference of the weights; its own error is of second order
    v = torch.randn(T, cfg["E"], generator=g).double()
    eps = 1e-4
    with torch.no_grad():
        up, dn = (_weights64(l64 + e * v, i, live, cfg)[0] for e in (eps, -eps))
    diff = ((up - dn) * g64).sum(dim=1) / (2 * eps)
    assert ((got * v).sum(dim=1) - diff).abs().max() <= 1e-5 * (1 + float(mag.sum(dim=1).max()))
    layer.close()


def test_routing_weights_gradient_at_the_ends():
    layer = _layer(E=8, k=2)
    logits = torch.zeros(4, 8)
    logits[1, 1:] = float("-inf")                                    # one expert has all the probability
    logits[2] = torch.tensor([80.0, 79.0, -80.0, 0, 0, 0, 0, 0])
    idx = torch.tensor([[0, 1], [0, 1], [0, 1], [9, -1]], dtype=torch.int32)     # the last token's picks name no expert
    w = torch.ones(4, 2)
    gw = torch.tensor([[1.0, -1.0]] * 4)
    got = layer.route_topk_grad(logits.to(DEV), idx.to(DEV), w.to(DEV), gw.to(DEV)).cpu().double()
    l64 = logits.double().requires_grad_(True)
    want = torch.autograd.grad((torch.softmax(l64, 1)[:3].gather(1, idx[:3].long()) * gw[:3].double()).sum(), l64)[0]
    assert ((got - want)[:3].abs() <= 2.0 ** -17).all() and got[3].abs().max() == 0
    layer.close()
    sig = _layer(E=8, k=2, gating=2, n_group=1, topk_group=1)
    logits = torch.tensor([[30.0, -30.0, 100.0, -100.0, 0, 0, 0, 0]])
    idx = torch.tensor([[0, 1]], dtype=torch.int32)
    got = sig.route_topk_grad(logits.to(DEV), idx.to(DEV), torch.ones(1, 2, device=DEV), torch.ones(1, 2, device=DEV)).cpu().double()[0]
    e = torch.exp(torch.tensor(-30.0, dtype=torch.float64))
    assert abs(got[0] - e / (1 + e) ** 2) <= e * 2.0 ** -17 and abs(got[1] - e / (1 + e) ** 2) <= e * 2.0 ** -17
    assert not got[2:].any()
    # an expert that two picks of a token name has both their gradients
    idx = torch.tensor([[4, 4], [4, 5]], dtype=torch.int32, device=DEV)
    got = sig.route_topk_grad(torch.zeros(2, 8, device=DEV), idx, torch.ones(2, 2, device=DEV), torch.tensor([[1.0, 2.0]] * 2, device=DEV))
    assert got[0, 4] == 0.75 and got[1, 4] == 0.25 and got[1, 5] == 0.5 and got.abs().sum() == 1.5
    sig.close()


# ------------------------------------------------------------------ as they are used: a calibration step around int8 experts
def _calibration(graph):
    from moe_gen_b200 import WEIGHT_INT8_CHANNEL, MoELayer, combine_rows, route, sort_rows
    E, k, H, I, T = 8, 2, 256, 128, 45
    layer = MoELayer(hidden=H, inter=I, n_experts=E, top_k=k, gating=3, norm_topk_prob=True, weight_format=WEIGHT_INT8_CHANNEL,
                     device=DEV)
    g = torch.Generator().manual_seed(11)
    for e in range(E):
        m = [torch.randint(-127, 128, s, generator=g, dtype=torch.int8) for s in ((I, H), (I, H), (H, I))]
        layer.load_expert(e, *m, scales=tuple(torch.full((t.shape[0],), 5e-4) for t in m))
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    gate = (torch.randn(E, H, generator=g) * 0.1).to(DEV)
    adapter = (torch.randn(H, H, generator=g) * 0.02).to(torch.bfloat16).to(DEV)     # on the sorted rows, trained
    target = torch.randn(T, H, generator=g).to(DEV)
    return layer, x, gate, adapter, target, (route, sort_rows, combine_rows)


def _step(layer, x, gate, adapter, target, fns):
    """Loss of a block of frozen int8 experts, an adapter on the sorted rows, and a router."""
    route, sort_rows, combine_rows = fns
    logits = x.float() @ gate.t()
    idx, w = route(layer, logits)
    counts, _, pad, dst = layer.permute_plan(idx)
    n = layer.padded_rows(idx.numel())
    rows = sort_rows(layer, x, dst, n, counts, pad)
    with torch.no_grad():
        xq, xs = layer.quantize_rows(x)
        pq, ps = layer.permute_rows_int8(xq, xs, dst, n)
        _, frozen = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    out = frozen + rows @ adapter
    y = combine_rows(layer, out, dst, idx, w, counts, pad)
    return ((y.float() - target) ** 2).mean(), (idx, dst, frozen)


def _step64(x, gate, adapter, target, idx, dst, frozen):
    p = torch.softmax(x @ gate.t(), dim=1).gather(1, idx.long())
    w = p / p.sum(dim=1, keepdim=True)
    out = frozen[dst.long()] + (x @ adapter)[:, None, :]
    return (((out * w[:, :, None]).sum(dim=1) - target) ** 2).mean()


def test_a_calibration_step_around_int8_experts():
    """Gradients of router, adapter and input of the whole chain, against 64 bits.  The bf16 roundings along it (rows, adapter
    product, sum, output, its gradient, the two products of the backward pass: eight of 2^-8 at most, of random sign) bound the relative norm
    of the difference by 8 * 2^-8."""
    layer, x, gate, adapter, target, fns = _calibration(False)
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, adapter)]
    loss, (idx, dst, frozen) = _step(layer, *leaves, target, fns)
    got = torch.autograd.grad(loss, leaves)
    l64 = [t.double().requires_grad_(True) for t in (x, gate, adapter)]
    loss64 = _step64(*l64, target.double(), idx, dst, frozen.double())
    want = torch.autograd.grad(loss64, l64)
    assert abs(loss.item() - loss64.item()) <= 8 * 2.0 ** -8 * loss64.item()
    for a, b in zip(got, want):
        assert a.shape == b.shape and (a.double() - b).norm() <= 8 * 2.0 ** -8 * b.norm()
    # along the router's gradient, a difference of the 64-bit loss
    v = want[1] / want[1].norm()
    with torch.no_grad():
        f = [_step64(l64[0], l64[1] + e * v, l64[2], target.double(), idx, dst, frozen.double()) for e in (1e-5, -1e-5)]
    assert abs(float((f[0] - f[1]) / 2e-5) - float((got[1].double() * v).sum())) <= 8 * 2.0 ** -8 * float(want[1].norm())
    layer.close()


def test_gradients_only_where_they_are_asked_for():
    from moe_gen_b200 import combine_rows
    layer, idx, counts, pad, dst, rows, live = _setup(20, 8, 2, 256)
    out = torch.randn(rows, 256, device=DEV).to(torch.bfloat16)
    w = torch.rand(20, 2, device=DEV)
    sh = torch.randn(20, 256, device=DEV).to(torch.bfloat16)
    gy = torch.randn(20, 256, device=DEV).to(torch.bfloat16)
    full = [t.clone().requires_grad_(True) for t in (out, w, sh)]
    ref = torch.autograd.grad(combine_rows(layer, full[0], dst, idx, full[1], counts, pad, full[2]), full, gy)
    assert torch.equal(ref[2], gy)
    for need in itertools.product((False, True), repeat=3):
        if not any(need):
            continue
        t = [a.clone().requires_grad_(n) for a, n in zip((out, w, sh), need)]
        y = combine_rows(layer, t[0], dst, idx, t[1], counts, pad, t[2])
        got = torch.autograd.grad(y, [a for a, n in zip(t, need) if n], gy)
        for a, b in zip(got, [r for r, n in zip(ref, need) if n]):
            assert torch.equal(a, b)
    # a gradient that arrives as an expanded view
    y = combine_rows(layer, full[0], dst, idx, full[1], counts, pad)
    a = torch.autograd.grad(y.float().sum(), full[:2])
    b = layer.combine_grad(torch.ones_like(gy), out, dst, w, counts, pad)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    layer.close()


def test_gradient_kernels_in_a_graph_and_on_another_stream():
    layer, idx, counts, pad, dst, rows, live = _setup(50, 64, 6, 512)
    out = torch.randn(rows, 512, device=DEV).to(torch.bfloat16)
    w, gy = torch.rand(50, 6, device=DEV), torch.randn(50, 512, device=DEV).to(torch.bfloat16)
    logits, gw0 = torch.randn(50, 64, device=DEV), torch.randn(50, 6, device=DEV)

    def step():
        return (*layer.combine_grad(gy, out, dst, w, counts, pad), layer.permute_rows_grad(out, dst),
                layer.permute_rows(gy, dst, rows, counts, pad), layer.route_topk_grad(logits, idx, w, gw0))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    layer.close()


def test_refusals():
    layer, idx, counts, pad, dst, rows, live = _setup(10, 8, 2, 256)
    x = torch.zeros(10, 256, dtype=torch.bfloat16, device=DEV)
    out, w = torch.zeros(rows, 256, dtype=torch.bfloat16, device=DEV), torch.ones(10, 2, device=DEV)
    for bad in (lambda: layer.permute_rows(x[:9], dst, rows, counts, pad), lambda: layer.permute_rows(x, dst, rows, counts, pad[:-1]),
                lambda: layer.permute_rows(x, dst.long(), rows, counts, pad), lambda: layer.permute_rows_grad(out.float(), dst),
                lambda: layer.permute_rows_grad(out[:, :128], dst), lambda: layer.permute_rows_grad(out, dst[:, :1]),
                lambda: layer.combine_grad(x, out, dst, w.double(), counts, pad), lambda: layer.combine_grad(x[:5], out, dst, w, counts, pad),
                lambda: layer.combine_grad(x.cpu(), out, dst, w, counts, pad), lambda: layer.combine_grad(x, out, dst, w[:, :1], counts, pad),
                lambda: layer.route_topk_grad(torch.zeros(10, 4, device=DEV), idx, w, w),
                lambda: layer.route_topk_grad(torch.zeros(10, 8, device=DEV), idx.long(), w, w),
                lambda: layer.route_topk_grad(torch.zeros(10, 8, device=DEV), idx, w, w[:4])):
        with pytest.raises(ValueError):
            bad()
    # contiguous views that begin off a 16-byte boundary
    from moe_gen_b200 import MoeGenError
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)      # noqa: E731
    lg = torch.zeros(10, 8, device=DEV)
    for bad in (lambda: layer.permute_rows(off(x), dst, rows, counts, pad), lambda: layer.permute_rows_grad(off(out), dst),
                lambda: layer.combine_grad(off(x), out, dst, w, counts, pad), lambda: layer.combine_grad(x, off(out), dst, w, counts, pad),
                lambda: layer.route_topk_grad(off(lg), idx, w, w)):
        with pytest.raises(MoeGenError, match="16-byte"):
            bad()
    layer.close()


def test_offsets_beyond_32_bits():
    """Buffers of rows of more than 2^31 elements: the last tokens, whose picks fill the last expert's segment."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    E, k, H, T = 8, 8, 7168, 37600                                     # 301824 padded rows of 7168: 2.16e9 elements
    layer = _layer(E=E, k=k, H=H)
    idx = torch.arange(8, dtype=torch.int32, device=DEV).repeat(T, 1)
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = layer.padded_rows(T * k)
    assert rows * H > 1 << 31 and int(dst.max()) * H > 1 << 31
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    x[-5:] = torch.randn(5, H, device=DEV).to(torch.bfloat16)
    perm = layer.permute_rows(x, dst, rows, counts, pad)
    assert torch.equal(perm[dst[-5:].long()], x[-5:, None, :].expand(5, k, H)) and not perm[dst[:-5, 7].long()].any()
    assert not perm[int(pad[-1]):].any()
    gx = layer.permute_rows_grad(perm, dst)
    assert torch.equal(gx[-5:], (x[-5:].float() * 8).to(torch.bfloat16)) and not gx[:-5].any()
    w = torch.full((T, k), 0.5, device=DEV)
    gr, gw = layer.combine_grad(x, perm, dst, w, counts, pad)
    assert torch.equal(gr[dst[-5:].long()].float(), perm[dst[-5:].long()].float() * 0.5) and not gr[int(pad[-1]):].any()
    norm = (x[-5:].double() ** 2).sum(dim=1, keepdim=True)
    assert ((gw[-5:].double() - norm).abs() <= norm * 96 * 2.0 ** -24).all() and not gw[:-5].any()
    layer.close()
    del perm, gr, gx, x
    torch.cuda.empty_cache()
