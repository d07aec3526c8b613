"""GPU: 8-bit integer rows and products.  The sums are exact in 32 bits and every rounding behind them is an IEEE one, so most
of what is compared here is compared bit for bit, with a restatement in 64 bits on the CPU that rounds in the same places.  The
one approximate step is silu: exp is __expf, whose error is 2 + 1.2 |x| units of 2^-23 (|x| <= 64 here: under 2^-16), and the
quotient adds 2 units."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _layer(E=8, k=2, H=256, I=128, Is=0, gating=None, n_group=1, topk_group=1, norm=False, scale=1.0, combine=0, int8=True):
    from moe_gen_b200 import MoELayer, WEIGHT_BF16, WEIGHT_INT8_CHANNEL
    return MoELayer(hidden=H, inter=I, n_experts=E, top_k=k, inter_shared=Is, n_group=n_group, topk_group=topk_group,
                    gating=0 if gating is None else gating, norm_topk_prob=norm, routed_scale=scale, combine_mode=combine,
                    weight_format=WEIGHT_INT8_CHANNEL if int8 else WEIGHT_BF16, device=DEV)


@pytest.fixture(scope="module")
def any_layer():
    return _layer()


def quantise(x):
    """q (int64) and fp32 scales by the definition: both quotients in fp32, the product of 8 and 24 bits exact in 64."""
    m = x.float().abs().amax(dim=1).clamp_min(2.0 ** -100)
    top = torch.full_like(m, 127.0)                  # a number divided by a tensor is a product with its reciprocal in torch
    q = torch.round(x.double() * (top / m).double()[:, None]).long()
    bad = ~torch.isfinite(x.float()).all(dim=1)
    q[bad] = 0
    return q, torch.where(bad, torch.full_like(m, float("nan")), m / top)


def product(xq, xs, wq, ws):
    """bf16(fp32(acc) * scale * w_scale), every step rounded as the kernel's; the sums are whole numbers below 2^53."""
    acc = (xq.double() @ wq.double().t()).float()
    return (acc * xs[:, None] * ws[None, :]).to(torch.bfloat16)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30)) and a.shape == b.shape


def _weights(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (n, (k + 15) // 16 * 16), generator=g, dtype=torch.int8)[:, :k]     # what lies between rows counts for nothing
    return q, torch.rand(n, generator=g) * 0.01 + 1e-4


def _strided(t):
    """The same values on the device, rows as far apart as on the host."""
    n, k = t.shape
    return torch.full((n, t.stride(0) if n > 1 else (k + 15) // 16 * 16), 77, dtype=t.dtype, device=DEV)[:, :k].copy_(t)


ROWS = [(1, 1), (1, 8), (3, 7), (2, 256), (5, 1408), (4, 5120), (3, 7168), (2, 14336), (2, 16384), (2, 16392), (3, 16411), (129, 33),
        (1000, 264)]


@pytest.mark.parametrize("n,k", ROWS)
def test_rows_are_quantised_by_the_definition(any_layer, n, k):
    g = torch.Generator().manual_seed(n * 7 + k)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 4)).to(torch.bfloat16)
    q, s = any_layer.quantize_rows(x.to(DEV))
    want_q, want_s = quantise(x)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().long(), want_q)
    assert q.stride(0) % 128 == 0 and int(q.abs().max()) == 127


def test_ties_zeros_and_the_ends_of_the_range(any_layer):
    x = torch.zeros(9, 64, dtype=torch.bfloat16)
    x[0, :5] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5])          # inv = 1: ties to even
    x[1, :2] = torch.tensor([3.38e38, -1.69e38])
    x[2, :2] = torch.tensor([1e-38, -5e-39])                       # below 2^-100: zeros
    x[3, 3] = 2.0 ** -100
    x[4, 3] = float("inf")
    x[5, 3] = float("nan")
    x[6, 3], x[6, 4] = float("nan"), float("-inf")
    x[8] = -1.0
    q, s = any_layer.quantize_rows(x.to(DEV))
    want_q, want_s = quantise(x)
    assert torch.equal(q.cpu().long(), want_q) and same(s.cpu(), want_s)
    assert q[0, :5].tolist() == [127, 0, 2, 2, 0] and q[2].abs().max() == 0 and q[3, 3] == 127
    assert torch.isnan(s[4:7]).all() and q[4:7].abs().max() == 0 and torch.isfinite(s[[0, 1, 2, 3, 7, 8]]).all()


def test_rows_of_any_stride_and_alignment(any_layer):
    g = torch.Generator().manual_seed(3)
    base = torch.randn(40, 301, generator=g).to(torch.bfloat16)
    dev = base.to(DEV)
    for a, b, step in ((0, 256, 1), (1, 257, 1), (8, 264, 2), (3, 300, 3), (0, 0 + 1, 1)):
        v = base[::step, a:b]
        q, s = any_layer.quantize_rows(dev[::step, a:b])
        want_q, want_s = quantise(v)
        assert torch.equal(q.cpu().long(), want_q) and torch.equal(s.cpu(), want_s), (a, b, step)


# tokens either side of the tile steps (32, 256, 288, 320, 384), outputs either side of 256 and odd, inputs either side of a step
MATMUL = [(1, 1, 1), (1, 16, 64), (2, 8, 128), (7, 255, 127), (8, 256, 128), (9, 257, 129), (17, 300, 384), (31, 512, 640), (32, 40, 1000),
          (33, 777, 1000), (64, 128, 1024), (65, 1000, 80), (97, 777, 1000), (128, 512, 2048), (160, 513, 256), (256, 256, 896),
          (257, 264, 272), (288, 256, 512), (289, 100, 144), (320, 384, 1408), (352, 256, 256), (383, 31, 300), (384, 512, 128),
          (385, 512, 128), (700, 1030, 520), (1153, 96, 192),
          # few rows: one launch, as long as their quantised form fits in a block's shared memory
          (1, 4096, 4096), (1, 33, 98304), (1, 8, 98305), (3, 19, 5001), (4, 50, 24576), (4, 3, 24577), (6, 130, 2049), (8, 20, 12288), (8, 21, 12289),
          (1, 20000, 64), (2, 19001, 72), (7, 4097, 4096), (8, 4096, 1024), (9, 700, 567), (11, 4096, 2048), (16, 33, 2047),
          (16, 4097, 2048), (13, 16, 2049), (15, 1030, 72)]


@pytest.mark.parametrize("m,n,k", MATMUL)
def test_product_is_exact(any_layer, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    wq, ws = _weights(n, k, m * 3 + k)
    xq = torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.int8)[:, :k].copy_(torch.randint(-128, 128, (m, k), generator=g))
    xs = torch.rand(m, generator=g) + 0.1
    y = any_layer.int8_matmul(_strided(xq), xs.to(DEV), _strided(wq), ws.to(DEV))
    assert same(y.cpu(), product(xq, xs, wq, ws))
    x = (torch.randn(m, k, generator=g) * 3).to(torch.bfloat16)
    q, s = quantise(x)
    y = any_layer.int8_linear(x.to(DEV), _strided(wq), ws.to(DEV))
    assert same(y.cpu(), product(q, s, wq, ws))
    assert any_layer.device_status() == (0, 0)


def test_sums_fill_32_bits(any_layer):
    k = 131071
    wq = torch.full((3, 131072), -128, dtype=torch.int8)[:, :k]
    xq = torch.full((2, 131072), -128, dtype=torch.int8)[:, :k]
    xq[1] = 127
    one = torch.ones(3)
    y = any_layer.int8_matmul(_strided(xq), one[:2].to(DEV), _strided(wq), one.to(DEV))
    assert same(y.cpu(), product(xq, one[:2], wq, one)) and float(y[0, 0]) == 2.0 ** 31


@pytest.mark.parametrize("n", (90, 88, 81, 95, 1, 289))
def test_rows_of_nan_stay_to_themselves_and_out_is_written_within_its_bounds(any_layer, n):
    m, k = 70, 200
    wq, ws = _weights(n, k, 5)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[11, 3], x[42, 0] = float("nan"), float("inf")
    big = torch.full((m + 2, (n + 31) // 8 * 8), 7.0, dtype=torch.bfloat16, device=DEV)
    out = any_layer.int8_linear(x.to(DEV), _strided(wq), ws.to(DEV), out=big[1:m + 1, 8:8 + n])
    q, s = quantise(x)
    assert same(out.cpu(), product(q, s, wq, ws))
    rest = big.clone()
    rest[1:m + 1, 8:8 + n] = 7.0
    assert bool((rest == 7.0).all())


def test_a_row_does_not_depend_on_its_batch(any_layer):
    wq, ws = _weights(300, 512, 9)
    w, s = _strided(wq), ws.to(DEV)
    x = torch.randn(500, 512, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    y = any_layer.int8_linear(x, w, s)
    for a, b in ((0, 1), (3, 5), (100, 133), (77, 500)):
        assert torch.equal(any_layer.int8_linear(x[a:b], w, s), y[a:b])
    assert any_layer.int8_linear(x[:0], w, s).shape == (0, 300)


def test_products_on_two_streams_and_in_graphs(any_layer):
    """Two products at once, each on its own stream, and two captured graphs of one layer replayed one beside the other."""
    other = _layer(E=4)
    probs = []
    for i, layer in enumerate((any_layer, other)):
        wq, ws = _weights(1024, 1024, 20 + i)
        x = torch.randn(40 + i, 1024, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
        q, s = quantise(x)
        probs.append((layer, x.to(DEV), _strided(wq), ws.to(DEV), product(q, s, wq, ws)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (layer, x, w, s, _) in enumerate(probs):
            with torch.cuda.stream(streams[i]):
                got[i].append(layer.int8_linear(x, w, s))
    torch.cuda.synchronize()
    for i, p in enumerate(probs):
        assert all(same(y.cpu(), p[4]) for y in got[i])
    graphs, outs = [], []
    for i, (layer, x, w, s, _) in enumerate(probs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.int8_linear(x, w, s))
        graphs.append(g)
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(same(o.cpu(), p[4]) for o, p in zip(outs, probs))


# ------------------------------------------------------------------ experts
SHAPES = [dict(E=8, k=2, H=256, I=128), dict(E=64, k=6, H=512, I=256, Is=256), dict(E=16, k=1, H=256, I=384),
          dict(E=4, k=4, H=768, I=128, Is=128)]


def _load(layer, seed):
    mats = {}
    for e in list(range(layer.E)) + ([-1] if layer.Is else []):
        n = layer.Is if e < 0 else layer.I
        m = [_weights(a, b, seed + 10 * e + i) for i, (a, b) in enumerate(((n, layer.H), (n, layer.H), (layer.H, n)))]
        layer.load_expert(e, *[q for q, _ in m], scales=tuple(s for _, s in m))
        mats[e] = m
    return mats


def _h64(xq, xs, mats):
    (gq, gs), (uq, us), _ = mats
    g = (xq.double() @ gq.double().t()) * xs.double()[:, None] * gs.double()
    u = (xq.double() @ uq.double().t()) * xs.double()[:, None] * us.double()
    return g, u, g / (1 + torch.exp(-g)) * u


def _check_mlp(xq, xs, mats, h, out):
    """h within half a bf16 step (2^-8) and silu's and the scales' error (2^-15) of the 64-bit value; out exact from h."""
    _, _, want = _h64(xq, xs, mats)
    assert ((h.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -15) + 1e-30).all()
    hq, hs = quantise(h)
    assert same(out, product(hq, hs, *mats[2]))


@pytest.mark.parametrize("shape,T", list(itertools.product(range(len(SHAPES)), (1, 5, 128, 129, 517))))
def test_experts_stage_by_stage(shape, T):
    layer = _layer(**SHAPES[shape])
    mats = _load(layer, 100 * shape)
    g = torch.Generator().manual_seed(T)
    x = (torch.randn(T, layer.H, generator=g) * 0.05).to(torch.bfloat16)
    # most tokens on the first experts, some experts empty
    score = torch.rand(T, layer.E, generator=g) + torch.linspace(1.0, 0.0, layer.E)
    idx = score.topk(layer.k, dim=1)[1].int().to(DEV)
    counts, _, pad, dst = layer.permute_plan(idx)
    rows = layer.padded_rows(T * layer.k)
    xq, xs = layer.quantize_rows(x.to(DEV))
    want_q, want_s = quantise(x)
    pq, ps = layer.permute_rows_int8(xq.contiguous(), xs, dst, rows)
    flat = dst.reshape(-1).long()
    src = torch.arange(T, device=DEV).repeat_interleave(layer.k)
    assert torch.equal(pq[flat].cpu().long(), want_q[src.cpu()]) and torch.equal(ps[flat].cpu(), want_s[src.cpu()])
    h, out = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    c, p = counts.cpu().tolist(), pad.cpu().tolist()
    assert sum(c) == T * layer.k
    for e in range(layer.E):
        if c[e]:
            r = slice(p[e], p[e] + c[e])
            _check_mlp(pq[r].cpu().long(), ps[r].cpu(), mats[e], h[r].cpu(), out[r].cpu())
    if layer.Is:
        y = layer.shared_ffn_int8(xq.contiguous(), xs)
        (gq, gs), (uq, us), (dq, ds) = mats[-1]
        gg, uu, _ = _h64(want_q, want_s, mats[-1])
        # the shared expert's intermediate rows are not handed out: within what their roundings can change
        hh = (gg / (1 + torch.exp(-gg)) * uu)
        m = hh.abs().amax(dim=1)
        # a quantised element is off by half a step of m / 127, and that and bf16's half step by what the kernel's h differs
        slack = (m / 127 * 0.5 + m * 2.0 ** -7)[:, None] * (dq.double().abs().sum(dim=1) * ds.double())[None, :]
        want = (hh @ dq.double().t()) * ds.double()
        assert ((y.cpu().double() - want).abs() <= slack + want.abs() * 2.0 ** -7).all()
    assert layer.device_status() == (0, 0)
    layer.close()


@pytest.mark.parametrize("counters", (False, True))
def test_experts_with_and_without_job_counters(counters):
    from moe_gen_b200 import lib as L
    layer = _layer(E=16, k=2, H=512, I=512)
    mats = _load(layer, 7)
    T = 900
    x = torch.randn(T, 512, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    idx = torch.rand(T, 16, generator=torch.Generator().manual_seed(9)).topk(2, dim=1)[1].int().to(DEV)
    counts, _, pad, dst = layer.permute_plan(idx)
    xq, xs = layer.quantize_rows(x)
    pq, ps = layer.permute_rows_int8(xq, xs, dst, layer.padded_rows(T * 2))
    if counters:
        with layer.job_counters(torch.zeros(L.JOB_COUNTERS, dtype=torch.int32, device=DEV)):
            h, out = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    else:
        h, out = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    c, p = counts.cpu().tolist(), pad.cpu().tolist()
    for e in range(16):
        r = slice(p[e], p[e] + c[e])
        _check_mlp(pq[r].cpu().long(), ps[r].cpu(), mats[e], h[r].cpu(), out[r].cpu())
    layer.close()


# ------------------------------------------------------------------ whole layer
FORWARD = [dict(E=64, k=6, H=512, I=256, Is=256, combine=1), dict(E=8, k=2, H=256, I=256, gating=3, norm=True, combine=2),
           dict(E=32, k=4, H=256, I=128, Is=128, gating=2, n_group=8, topk_group=4, norm=True, scale=2.5),
           dict(E=32, k=3, H=512, I=128, gating=1, n_group=4, topk_group=2, scale=16.0, combine=1)]


def _staged(layer, x, logits):
    idx, w = layer.route_topk(logits)
    counts, _, pad, dst = layer.permute_plan(idx)
    xq, xs = layer.quantize_rows(x)
    pq, ps = layer.permute_rows_int8(xq, xs, dst, layer.padded_rows(idx.numel()))
    _, out = layer.expert_ffn_int8(pq, ps, pad, counts, dst)
    return layer.combine(out, dst, idx, w, layer.shared_ffn_int8(xq, xs) if layer.Is else None)


def _ready(cfg, seed=50):
    layer = _layer(**cfg)
    mats = _load(layer, seed)
    g = torch.Generator().manual_seed(seed)
    layer.set_router(torch.randn(layer.E, layer.H, generator=g) * 0.1,
                     torch.randn(layer.E, generator=g) * 0.01 if cfg.get("gating") == 2 else None)
    return layer, mats


@pytest.mark.parametrize("cfg,T", list(itertools.product(range(len(FORWARD)), (0, 1, 16, 65, 128, 129, 1100))))
def test_forward_is_its_stages(cfg, T):
    layer, _ = _ready(FORWARD[cfg])
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, layer.H, generator=g).to(torch.bfloat16).to(DEV)
    if T == 0:
        assert layer.forward(x).shape == (0, layer.H)
        return
    logits = torch.randn(T, layer.E, generator=g).to(DEV)
    want = _staged(layer, x, logits)
    assert torch.equal(layer.forward_from_logits(x, logits), want)
    lg = layer.gate_route(x)[2]
    assert torch.equal(layer.forward(x), _staged(layer, x, lg))
    norm = torch.ones(layer.H, dtype=torch.bfloat16, device=DEV)
    xn = layer.rmsnorm(x, norm)
    ref = (layer.forward(xn).float() + x.float()).to(torch.bfloat16)
    assert torch.equal(layer.block_forward(x, norm), ref)
    host = x.cpu().pin_memory()
    assert torch.equal(layer.forward_host(host, chunk_tokens=64), torch.cat(
        [layer.forward(c.contiguous()) for c in torch.split(x, layer.host_chunks(T, 64))]).cpu())
    assert layer.device_status() == (0, 0)
    layer.close()


def test_forward_against_the_definition_in_64_bits():
    """Each output is off by at most half a step of the result and, per pick, by half a step of the row (2^-8 both) and by what
    the rows between the products may be off: half a bf16 step each, which moves a quantised element by at most one step
    of m / 127 (m the row's largest); the down product's weights carry it.  Bounded with the sum of |w| |weights|."""
    layer, mats = _ready(FORWARD[0], 70)
    T = 37
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, layer.H, generator=g).to(torch.bfloat16)
    logits = torch.randn(T, layer.E, generator=g)
    p = torch.softmax(logits.double(), dim=1)
    w, idx = p.topk(layer.k, dim=1)
    q, s = quantise(x)
    y, slack = torch.zeros(T, layer.H, dtype=torch.float64), torch.zeros(T, layer.H, dtype=torch.float64)
    for e in list(range(layer.E)) + [-1]:
        t, j = (torch.arange(T), None) if e < 0 else (idx == e).nonzero(as_tuple=True)
        if t.numel() == 0:
            continue
        _, _, h = _h64(q[t], s[t], mats[e])
        h = h.to(torch.bfloat16)
        hq, hs = quantise(h)
        dq, ds = mats[e][2]
        o = (hq.double() @ dq.double().t()) * hs.double()[:, None] * ds.double()
        c = torch.ones(t.numel(), dtype=torch.float64) if e < 0 else w[t, j]
        y[t] += o * c[:, None]
        # one step of every element at most, and the roundings of weight (bf16 mode), row and product
        one = hs.double()[:, None] * (dq.double().abs().sum(dim=1) * ds.double())[None, :]
        slack[t] += (one + o.abs() * 3 * 2.0 ** -8) * c[:, None]
    got = layer.forward_from_logits(x.to(DEV), logits.to(DEV)).cpu().double()
    assert ((got - y).abs() <= slack + y.abs() * 2.0 ** -7 + 1e-12).all()
    # and on the whole no more than the 8 bits of the steps that are rounded to bf16 (four of them)
    assert (got - y).norm() <= 4 * 2.0 ** -8 * y.norm()
    layer.close()


def test_forward_in_a_graph_and_with_a_workspace_that_held_anything():
    layer, _ = _ready(FORWARD[0])
    x = torch.randn(24, layer.H, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    want = layer.forward(x)
    layer._ws.random_(0, 256)
    assert torch.equal(layer.forward(x), want)
    y = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer.forward(x, out=y)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        layer.forward(x, out=y)
    x2 = torch.randn(24, layer.H, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    want2 = layer.forward(x2)
    for src, ref in ((x.clone(), want), (x2, want2)):
        x.copy_(src)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
    layer.set_stage_timing(True)
    assert torch.equal(layer.forward(x2), want2)
    torch.cuda.synchronize()
    assert layer.stage_times()["expert_gemm1"] > 0
    layer.close()


def test_refusals(any_layer):
    from moe_gen_b200 import MoeGenError
    layer = _layer(Is=128)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(16, 256, dtype=torch.int8, device=DEV)
    s = torch.ones(16, device=DEV)
    with pytest.raises(ValueError):
        layer.load_expert(0, w, w, w)
    with pytest.raises(ValueError):
        layer.load_expert(0, *[torch.zeros(a, b, dtype=torch.int8) for a, b in ((128, 256), (128, 256), (256, 128))])
    with pytest.raises(ValueError):
        layer.load_expert(0, *[torch.zeros(a, b, dtype=torch.int8) for a, b in ((128, 256), (128, 256), (256, 128))],
                          scales=(torch.ones(128), torch.ones(128), torch.ones(128)))
    with pytest.raises(ValueError):
        layer.int8_linear(x.float(), w, s)
    with pytest.raises(ValueError):
        layer.int8_linear(x, w[:, :128], s)
    with pytest.raises(ValueError):
        layer.int8_linear(x, w, s[:8])
    with pytest.raises(ValueError):
        layer.int8_linear(x, w, s, out=torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError):
        layer.quantize_rows(x.t())
    with pytest.raises(MoeGenError):                                   # weight rows off 16-byte strides, and off a boundary
        layer.int8_linear(x[:, :250], torch.zeros(16, 250, dtype=torch.int8, device=DEV), s)
    with pytest.raises(MoeGenError):
        layer.int8_linear(x[:, :240], w[:, 1:241], s)
    with pytest.raises(MoeGenError):                                   # output rows off 8-element strides
        layer.int8_linear(x, w, s, out=torch.zeros(4, 17, dtype=torch.bfloat16, device=DEV)[:, :16])
    with pytest.raises(MoeGenError):
        layer.int8_matmul(torch.zeros(4, 250, dtype=torch.int8, device=DEV), s[:4].contiguous(), w[:, :250], s)
    with pytest.raises(MoeGenError):                                   # more than 32 bits of sums
        layer.quantize_rows(torch.zeros(1, 131072, dtype=torch.bfloat16, device=DEV))
    counts, _, pad, dst = layer.permute_plan(torch.zeros(4, 2, dtype=torch.int32, device=DEV))
    with pytest.raises(MoeGenError, match="int8"):
        layer.expert_ffn(torch.zeros(256, 256, dtype=torch.bfloat16, device=DEV), pad, counts)
    with pytest.raises(MoeGenError, match="int8"):
        layer.shared_ffn(x)
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)      # noqa: E731
    q, sc = layer.quantize_rows(x)
    pq, ps = layer.permute_rows_int8(q, sc, dst, 256)
    for bad in (lambda: layer.permute_rows_int8(off(q), sc, dst, 256), lambda: layer.expert_ffn_int8(off(pq), ps, pad, counts, dst),
                lambda: layer.shared_ffn_int8(off(q), sc), lambda: layer.int8_matmul(off(q), sc, w, s)):
        with pytest.raises(MoeGenError, match="16-byte"):
            bad()
    lg = torch.zeros(4, 8, device=DEV)
    for bad in (lambda: layer.forward_from_logits(off(x), lg), lambda: layer.forward_from_logits(x, lg, out=off(x))):
        with pytest.raises(MoeGenError, match="16-byte"):
            bad()
    bf = _layer(int8=False)
    q, sc = bf.quantize_rows(x)
    with pytest.raises(MoeGenError, match="not int8"):
        bf.expert_ffn_int8(torch.zeros(256, 256, dtype=torch.int8, device=DEV), torch.zeros(256, device=DEV), pad, counts, dst)
    with pytest.raises(MoeGenError):
        bf.shared_ffn_int8(q, sc)
    layer.close()
    bf.close()


# ------------------------------------------------------------------ checkpoints and modules
def _checkpoint_weights(seed, E=8, H=256, I=128, Is=128):
    """Per expert ((q, scale), ...) with scales as a column, as such checkpoints store them; the shared expert in bf16."""
    def mats(n, s):
        return [(q.contiguous(), sc[:, None]) for q, sc in (_weights(a, b, s + i) for i, (a, b) in enumerate(((n, H), (n, H), (H, n))))]
    g = torch.Generator().manual_seed(seed)
    shared = [torch.randn(a, b, generator=g).mul(0.05).to(torch.bfloat16) for a, b in ((Is, H), (Is, H), (H, Is))]
    return [mats(I, seed + 10 * e) for e in range(E)], shared, torch.randn(E, H, generator=g).to(torch.bfloat16)


def _direct(experts, shared, router):
    layer = _layer(Is=128, norm=True)
    layer.set_router(router)
    for e, m in enumerate(experts):
        layer.load_expert(e, *[q for q, _ in m], scales=tuple(s for _, s in m))
    q = [quantise(w) for w in shared]
    layer.load_shared(*[a.to(torch.int8) for a, _ in q], tuple(s for _, s in q))
    return layer


@pytest.mark.parametrize("shared_int8", (False, True))
def test_int8_checkpoint(tmp_path, shared_int8):
    from moe_gen_b200 import ingest
    experts, shared, router = _checkpoint_weights(300)
    want = _direct(experts, shared, router)
    stored = [(q.to(torch.int8), s[:, None]) for q, s in map(quantise, shared)] if shared_int8 else shared
    ingest.export_moe_layer(str(tmp_path / "model.safetensors"), 2, router, None, experts, shared=stored)
    got = _layer(Is=128, norm=True)
    ingest.load_moe_layer(got, ingest.Checkpoint(str(tmp_path)), 2, n_threads=2)
    assert torch.equal(got.packed, want.packed) and torch.equal(got.gate_w, want.gate_w)
    bf = _layer(Is=128, int8=False)
    with pytest.raises(ValueError, match="int8"):
        ingest.load_moe_layer(bf, ingest.Checkpoint(str(tmp_path)), 2)
    for layer in (want, got, bf):
        layer.close()


def test_patched_modules_of_int8_experts():
    from types import SimpleNamespace as NS
    from moe_gen_b200 import patch_moe_module

    class Lin(torch.nn.Module):
        def __init__(self, w, s=None):
            super().__init__()
            self.weight = torch.nn.Parameter(w.to(DEV), requires_grad=False)
            if s is not None:
                self.weight_scale = torch.nn.Parameter(s.to(DEV), requires_grad=False)

    experts, shared, router = _checkpoint_weights(400)
    x = torch.randn(2, 33, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    want = _direct(experts, shared, router)
    DeepseekV2MoE = type("DeepseekV2MoE", (torch.nn.Module,), {})
    mod = DeepseekV2MoE()
    mod.config = NS(hidden_size=256, moe_intermediate_size=128, n_routed_experts=8, num_experts_per_tok=2, n_shared_experts=1,
                    norm_topk_prob=True, routed_scaling_factor=1.0, scoring_func="softmax", topk_method="greedy")
    names = ("gate_proj", "up_proj", "down_proj")
    mod.gate = Lin(router)
    mod.experts = [NS(**{n: Lin(*m) for n, m in zip(names, e)}) for e in experts]
    mod.shared_experts = NS(**{n: Lin(w) for n, w in zip(names, shared)})
    mod.eval()
    layer = patch_moe_module(mod)
    assert torch.equal(layer.packed, want.packed)
    # the module's combine mode rounds products to bf16, which the directly built layer does not: compared through the patched one
    assert torch.equal(mod.forward(x), layer.forward(x)) and layer.desc.weight_format == 2
    MixtralSparseMoeBlock = type("MixtralSparseMoeBlock", (torch.nn.Module,), {})
    mix = MixtralSparseMoeBlock()
    mix.gate, mix.top_k = Lin(router), 2
    mix.experts = [NS(w1=Lin(*e[0]), w3=Lin(*e[1]), w2=Lin(*e[2])) for e in experts]
    y, logits = (patch_moe_module(mix), mix.forward(x))[1]
    assert y.shape == x.shape and logits.shape == (66, 8) and bool(torch.isfinite(y.float()).all())
    lay = mix._moegen_b200_layer
    assert torch.equal(y.view(-1, 256), _staged(lay, x.view(-1, 256), lay.gate_logits(x.view(-1, 256))))


def test_layers_that_stream_or_shard_refuse_int8_experts():
    from moe_gen_b200 import WEIGHT_INT8_CHANNEL
    from moe_gen_b200.ep import EPMoELayer
    from moe_gen_b200.stream import StreamedMoELayer
    with pytest.raises(ValueError, match="int8"):
        StreamedMoELayer(group_experts=4, hidden=256, inter=128, n_experts=8, top_k=2, weight_format=WEIGHT_INT8_CHANNEL)
    layer = _layer()
    with pytest.raises(ValueError, match="int8"):
        EPMoELayer(layer)
    layer.close()


def test_offsets_beyond_32_bits(any_layer):
    """Rows, products and outputs of more than 2^31 elements: the last rows against the first rows' own call."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    m, k, n = 262160, 8200, 16
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)              # 2.15e9 elements
    tail = torch.randn(33, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[-33:] = tail.to(DEV)
    q, s = any_layer.quantize_rows(x)
    want_q, want_s = quantise(tail)
    assert torch.equal(q[-33:].cpu().long(), want_q) and torch.equal(s[-33:].cpu(), want_s) and not q[:40].any()
    wq, ws = _weights(n, k, 2)
    y = any_layer.int8_matmul(q, s, _strided(wq), ws.to(DEV))
    assert same(y[-33:].cpu(), product(want_q, want_s, wq, ws)) and not y[:-33].any()
    del x, q, y
    torch.cuda.empty_cache()
    m, k, n = 300000, 64, 7400                                          # 2.2e9 outputs
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    x[-33:] = tail[:, :k].to(DEV)
    wq, ws = _weights(n, k, 3)
    y = any_layer.int8_linear(x, _strided(wq), ws.to(DEV))
    assert same(y[-33:].cpu(), product(*quantise(tail[:, :k]), wq, ws)) and not y[:64].any()
    assert any_layer.device_status() == (0, 0)
    del x, y
    torch.cuda.empty_cache()
