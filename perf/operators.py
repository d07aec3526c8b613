"""Cases that time the 8-bit integer products of the MoE block and the gradients of its routing and row
movements through the public entry points, beside plain forms in elementary torch operations.

Kinds of case ("op"):
  linear  y = x . W^T with int8 weights (fp32 scale per output channel) and activations quantised to int8 per
          token: MoELayer.int8_linear.  "m", "n", "k": tokens, outputs, inputs
  layer   the MoE layer of an int8 checkpoint on given router logits: MoELayer.forward_from_logits.  "shape",
          "tokens", "zipf" (exponent of the router's load skew, 0 for a balanced load)
  sort    tokens sorted by expert, and the gradient of their rows brought back to the tokens:
          MoELayer.permute_rows and .permute_rows_grad.  "shape", "tokens"
  back    the experts' rows brought back with their routing weights, and the gradients of rows and weights:
          MoELayer.combine and .combine_grad.  "shape", "tokens"
  gates   the gradient of the routing weights with respect to the router logits: MoELayer.route_topk_grad.
          "shape", "tokens"

Quantisation of a row x (int8, symmetric): m = max(max|x|, 2^-100), scale = m / 127 and inv = 127 / m in fp32,
q = x * inv rounded to the nearest integer, ties to even; the row's values are q * scale.
"""
import math

import torch

own = False

SOFTMAX_GREEDY, SOFTMAX_GROUP_MAX, SIGMOID_NOAUX_TC, SOFTMAX_TOPK_RENORM = 0, 1, 2, 3     # MoELayer(gating=...)

# hidden, inter, experts, top_k, inter_shared, n_group, topk_group, gating, norm_topk_prob, routed_scale
SHAPES = {
    "v2lite": (2048, 1408, 64, 6, 2816, 1, 1, SOFTMAX_GREEDY, False, 1.0),
    "mixtral8x7b": (4096, 14336, 8, 2, 0, 1, 1, SOFTMAX_TOPK_RENORM, True, 1.0),
    "v2_236b": (5120, 1536, 160, 6, 3072, 8, 3, SOFTMAX_GROUP_MAX, False, 16.0),
    "v3": (7168, 2048, 256, 8, 2048, 8, 4, SIGMOID_NOAUX_TC, True, 2.5),
}
# most tokens of one call of the layer; v3's 256 experts (11 GB) are left to the row movements and the router
LAYER_TOKENS = {"v2lite": 8192, "mixtral8x7b": 8192, "v2_236b": 4096}
ROW_TOKENS = 8192
GATE_TOKENS = 65536
LINEAR_WORK = 8192 * 7168 * 4096


def listed():
    return [
        # one sequence decoding through a projection beside the MoE block: the weights' bytes and latency
        {"name": "linear_1", "op": "linear", "m": 1, "n": 4096, "k": 4096},
        # a ragged batch and a layer whose sizes no tile divides
        {"name": "linear_97_ragged", "op": "linear", "m": 97, "n": 777, "k": 1000},
        # a prefill micro-batch through a wide projection
        {"name": "linear_8192", "op": "linear", "m": 8192, "n": 4096, "k": 7168},
        # a handful of sequences decoding on the small model: launches and latency
        {"name": "layer_v2lite_8", "op": "layer", "shape": "v2lite", "tokens": 8, "zipf": 0.0},
        # an odd decode batch on 160 experts under the skewed load of real routers
        {"name": "layer_v2_236b_201", "op": "layer", "shape": "v2_236b", "tokens": 201, "zipf": 1.2},
        # a prefill batch on few, large experts
        {"name": "layer_mixtral_8192", "op": "layer", "shape": "mixtral8x7b", "tokens": 8192, "zipf": 0.0},
        # rows of a small calibration batch, forward and backward
        {"name": "sort_v2lite_37", "op": "sort", "shape": "v2lite", "tokens": 37},
        # rows of a training micro-batch of the largest model
        {"name": "sort_v3_8192", "op": "sort", "shape": "v3", "tokens": 8192},
        # a single token's rows brought back, and their gradients
        {"name": "back_mixtral_1", "op": "back", "shape": "mixtral8x7b", "tokens": 1},
        # the same for the training micro-batch
        {"name": "back_v3_8192", "op": "back", "shape": "v3", "tokens": 8192},
        # router of a small batch, softmax over 64 experts
        {"name": "gates_v2lite_37", "op": "gates", "shape": "v2lite", "tokens": 37},
        # router of a large batch, sigmoid scores normalised over the picks
        {"name": "gates_v3_65536", "op": "gates", "shape": "v3", "tokens": 65536},
    ]


def _log_size(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "layer", "sort", "back", "gates"])
    if op == "linear":
        n, k = _log_size(rng, 16, 8192), _log_size(rng, 64, 8192)
        return {"op": op, "m": _log_size(rng, 1, min(8192, LINEAR_WORK // (n * k))), "n": n, "k": k}
    if op == "layer":
        shape = rng.choice(sorted(LAYER_TOKENS))
        return {"op": op, "shape": shape, "tokens": _log_size(rng, 1, LAYER_TOKENS[shape]),
                "zipf": rng.choice([0.0, 1.2, round(rng.uniform(0.3, 1.2), 2)])}
    shape = rng.choice(sorted(SHAPES))
    return {"op": op, "shape": shape, "tokens": _log_size(rng, 1, GATE_TOKENS if op == "gates" else ROW_TOKENS)}


# ------------------------------------------------------------------ inputs, from the seed alone
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) % (1 << 62))
    return g


def _hidden(rows, cols, g):
    """Hidden states: unit variance, one channel in 64 eight times as wide (the outliers of real activations)."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x[:, ::64] *= 8.0
    return x.to(torch.bfloat16)


def _int8_weight(n, k, g):
    """[n, k] int8 with rows on 16-byte boundaries, and fp32 scales [n]: N(0, 0.02) quantised per row."""
    q = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
    q.copy_((torch.randn(n, k, generator=g, device="cuda", dtype=torch.bfloat16) * 32.0).round_().clamp_(-127, 127))
    s = (0.02 / 32.0) * (0.5 + torch.rand(n, generator=g, device="cuda"))
    return q, s


def _logits(case, seed):
    """Router logits on the grid of bf16, so that equal ones are exactly equal; skewed by a Zipf law if asked."""
    E = SHAPES[case["shape"]][2]
    g = _gen(seed, 1)
    lg = torch.randn(case["tokens"], E, generator=g, device="cuda") * 1.5
    if case.get("zipf", 0.0) > 0:
        order = torch.randperm(E, generator=g, device="cuda")
        law = (torch.arange(1, E + 1, dtype=torch.float64, device="cuda") ** -case["zipf"]).log()
        col = torch.empty(E, device="cuda")
        col[order] = (law - law.mean()).float()
        lg = lg + col
    return lg.to(torch.bfloat16).float()


def _top(c, k):
    """Indices of the k largest of every row, the lower index first among equals."""
    return torch.sort(c, dim=1, descending=True, stable=True)[1][:, :k]


def _scores(shape, logits):
    if SHAPES[shape][7] == SIGMOID_NOAUX_TC:
        return 1.0 / (1.0 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(dim=1, keepdim=True))
    return e / e.sum(dim=1, keepdim=True)


def _route(shape, logits):
    """Picks [T, k] (int64) and routing weights [T, k] in the type of the logits."""
    _, _, E, k, _, G, tg, gating, norm, scale = SHAPES[shape]
    s = _scores(shape, logits)
    c = s
    if gating in (SOFTMAX_GROUP_MAX, SIGMOID_NOAUX_TC):
        v = s.view(-1, G, E // G)
        gs = v.amax(dim=2) if gating == SOFTMAX_GROUP_MAX else v.topk(2, dim=2)[0].sum(dim=2)
        keep = torch.zeros_like(gs, dtype=torch.bool).scatter_(1, _top(gs, tg), True)
        c = torch.where(keep.unsqueeze(2), v, torch.zeros_like(v)).view(-1, E)
    idx = _top(c, k)
    p = (s if gating == SIGMOID_NOAUX_TC else c).gather(1, idx)
    if gating == SOFTMAX_TOPK_RENORM:
        return idx, p / p.sum(dim=1, keepdim=True)
    if norm and k > 1:
        w = p / (p.sum(dim=1, keepdim=True) + 1e-20)
        return idx, w * scale if gating == SIGMOID_NOAUX_TC else w
    return idx, p * scale


def _padded_rows(R, E):
    """Rows of a buffer that holds R rows sorted by expert whatever the routing (MoELayer.padded_rows)."""
    return ((R + 127) // 128 + E) * 128


def _plan(idx, E):
    """Rows sorted by expert, every expert's on a 128-row boundary: counts, first rows, row of (token, slot)."""
    T, k = idx.shape
    flat = idx.reshape(-1)
    counts = torch.bincount(flat, minlength=E)
    pad = torch.zeros(E + 1, dtype=torch.int64, device=idx.device)
    pad[1:] = torch.cumsum((counts + 127) // 128 * 128, 0)
    order = torch.sort(flat, stable=True)[1]
    first = torch.cumsum(counts, 0) - counts
    dst = torch.empty_like(flat)
    dst[order] = torch.arange(T * k, device=idx.device) - first[flat[order]] + pad[flat[order]]
    return counts.int(), pad.int(), dst.view(T, k).int(), _padded_rows(T * k, E)


def _layer(shape, int8=False):
    from moe_gen_b200 import WEIGHT_BF16, WEIGHT_INT8_CHANNEL, MoELayer
    H, I, E, k, Is, G, tg, gating, norm, scale = SHAPES[shape]
    if not int8:                                  # row movements and routing: a layer without weights to speak of
        I, Is = 128, 0
    return MoELayer(hidden=H, inter=I, n_experts=E, top_k=k, inter_shared=Is, n_group=G, topk_group=tg, gating=gating,
                    norm_topk_prob=norm, routed_scale=scale,
                    weight_format=WEIGHT_INT8_CHANNEL if int8 else WEIGHT_BF16)


def prepare(case, seed):
    op, st = case["op"], {"op": case["op"]}
    if op == "linear":
        st["x"] = _hidden(case["m"], case["k"], _gen(seed, 2))
        st["w"], st["s"] = _int8_weight(case["n"], case["k"], _gen(seed, 3))
        if own:
            st["layer"] = _layer("v2lite")
        return st
    shape, T = case["shape"], case["tokens"]
    H, I, E, k, Is = SHAPES[shape][:5]
    st["shape"], st["logits"] = shape, _logits(case, seed)
    if own:
        st["layer"] = _layer(shape, int8=op == "layer")
    if op == "layer":
        st["x"] = _hidden(T, H, _gen(seed, 2))
        experts = []
        for e in list(range(E)) + ([-1] if Is else []):
            g, n = _gen(seed, 1000 + e), Is if e < 0 else I
            mats = [_int8_weight(a, b, g) for a, b in ((n, H), (n, H), (H, n))]
            if own:
                st["layer"].load_expert(e, *[q for q, _ in mats], scales=tuple(s for _, s in mats))
            else:
                experts.append(mats)
        st["experts"] = experts
        return st
    idx, w = _route(shape, st["logits"].double())
    st["idx"], st["w"] = idx.int(), w.float()
    if op == "gates":
        st["gw"] = torch.randn(T, k, generator=_gen(seed, 4), device="cuda")
        return st
    st["counts"], st["pad"], st["dst"], st["rows"] = _plan(idx, E)
    live = torch.zeros(st["rows"], dtype=torch.bool, device="cuda")
    live[st["dst"].reshape(-1).long()] = True
    rows = torch.randn(st["rows"], H, generator=_gen(seed, 5), device="cuda").to(torch.bfloat16) * live.unsqueeze(1)
    if op == "sort":
        st["x"], st["grad"] = _hidden(T, H, _gen(seed, 2)), rows
    else:
        st["out"], st["gy"] = rows, torch.randn(T, H, generator=_gen(seed, 6), device="cuda").to(torch.bfloat16)
    return st


# ------------------------------------------------------------------ plain forms
def _quantise(x, dt):
    """int8 values of x's rows (in type dt) and the fp32 scales."""
    m = x.float().abs().amax(dim=1, keepdim=True).clamp_min(2.0 ** -100)
    inv = 127.0 / m
    return torch.round(x.double() * inv.double()).to(dt), m / 127.0      # the product has 32 bits: exact in 64


def _linear(x, q, s):
    xq, sx = _quantise(x, torch.float32)
    return (xq @ q.float().t()) * sx * s


def _mlp(x, mats):
    (gq, gs), (uq, us), (dq, ds) = mats
    g, u = _linear(x, gq, gs), _linear(x, uq, us)
    h = (g / (1.0 + torch.exp(-g)) * u).to(torch.bfloat16)               # what lies between the products is bf16
    return _linear(h, dq, ds)


def _layer_plain(st):
    x, shape = st["x"], st["shape"]
    E, Is = SHAPES[shape][2], SHAPES[shape][4]
    idx, w = _route(shape, st["logits"])
    y = torch.zeros(x.shape, device=x.device)
    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel():
            y.index_add_(0, t, _mlp(x[t], st["experts"][e]) * w[t, j].unsqueeze(1))
    if Is:
        y += _mlp(x, st["experts"][E])
    return y.to(torch.bfloat16)


def _gates_plain(shape, logits, idx, w, gw):
    _, _, E, k, _, _, _, gating, norm, scale = SHAPES[shape]
    s = _scores(shape, logits)
    i = idx.long()
    live = w != 0                                  # a pick out of a masked group has weight 0 and passes nothing on
    p = torch.where(live, s.gather(1, i), torch.zeros_like(w))
    if gating == SOFTMAX_TOPK_RENORM or (norm and k > 1):
        d = p.sum(dim=1, keepdim=True) + (0.0 if gating == SOFTMAX_TOPK_RENORM else 1e-20)
        gp = (gw - (gw * p).sum(dim=1, keepdim=True) / d) / d
        if gating == SIGMOID_NOAUX_TC:
            gp = gp * scale
    else:
        gp = gw * scale
    gs = torch.zeros_like(s).scatter_add_(1, i, torch.where(live, gp, torch.zeros_like(gp)))
    if gating == SIGMOID_NOAUX_TC:
        return gs * s * (1.0 - s)
    return s * (gs - (gs * s).sum(dim=1, keepdim=True))


def run(st):
    op = st["op"]
    if own:
        layer = st["layer"]
        if op == "linear":
            return layer.int8_linear(st["x"], st["w"], st["s"])
        if op == "layer":
            return layer.forward_from_logits(st["x"], st["logits"])
        if op == "sort":
            rows = layer.permute_rows(st["x"], st["dst"], st["rows"], st["counts"], st["pad"])
            return rows, layer.permute_rows_grad(st["grad"], st["dst"])
        if op == "back":
            y = layer.combine(st["out"], st["dst"], st["idx"], st["w"])
            return (y,) + tuple(layer.combine_grad(st["gy"], st["out"], st["dst"], st["w"], st["counts"], st["pad"]))
        return layer.route_topk_grad(st["logits"], st["idx"], st["w"], st["gw"])
    if op == "linear":
        return _linear(st["x"], st["w"], st["s"]).to(torch.bfloat16)
    if op == "layer":
        return _layer_plain(st)
    if op == "gates":
        return _gates_plain(st["shape"], st["logits"], st["idx"], st["w"], st["gw"])
    dst = st["dst"].long()
    T, k = dst.shape
    if op == "sort":
        x, g = st["x"], st["grad"]
        rows = torch.zeros(st["rows"], x.shape[1], dtype=x.dtype, device=x.device)
        rows[dst.reshape(-1)] = x.repeat_interleave(k, dim=0)
        gx = torch.zeros(x.shape, device=x.device)
        for j in range(k):
            gx += g[dst[:, j]].float()
        return rows, gx.to(x.dtype)
    out, gy, w = st["out"], st["gy"].float(), st["w"]
    y = torch.zeros(gy.shape, device=gy.device)
    grows, gw = torch.zeros_like(out), torch.empty_like(w)
    for j in range(k):
        r = out[dst[:, j]].float()
        y += r * w[:, j:j + 1]
        gw[:, j] = (gy * r).sum(dim=1)
        grows[dst[:, j]] = (gy * w[:, j:j + 1]).to(out.dtype)
    return y.to(out.dtype), grows, gw


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    H, I, E, k, Is, _, _, gating = SHAPES[case["shape"]][:8]
    T = case["tokens"]
    R = T * k
    if op == "layer":
        hit = E * (1.0 - (1.0 - k / E) ** T) if case["zipf"] == 0 else min(E, R) * 0.5
        weights = int(hit) * 3 * H * I + 3 * H * Is
        return {"bytes": weights + 4 * T * E + 4 * T * H, "flops": 6 * H * (R * I + T * Is)}
    P = _padded_rows(R, E)                          # rows no pick points at are written as zeros
    if op == "sort":
        return {"bytes": 2 * H * (T + P) + 2 * H * (R + T) + 4 * R, "flops": R * H}
    if op == "back":
        return {"bytes": 2 * H * (R + T) + 2 * H * (T + P) + 12 * R, "flops": 5 * R * H}
    scores = R if gating == SIGMOID_NOAUX_TC else T * E         # sigmoids of the picks alone, or a softmax over all
    return {"bytes": 4 * scores + 4 * T * E + 12 * R, "flops": 4 * scores}


# ------------------------------------------------------------------ the definitions in 64 bits
def _x_quant(x):
    x = x.double()
    m = torch.clamp(x.abs().max(dim=1)[0], min=2.0 ** -100).float()
    inv, scale = (127.0 / m).double(), (m / 127.0).double()
    return torch.round(x * inv[:, None]), scale[:, None]


def _x_linear(x, q, s):
    v, scale = _x_quant(x)
    return torch.mm(v, q.double().t()) * scale * s.double()


def _x_layer(case, seed):
    H, I, E, k, Is, G, tg, gating, norm, scale = SHAPES[case["shape"]]
    x, lg = _hidden(case["tokens"], H, _gen(seed, 2)), _logits(case, seed).double()
    T = case["tokens"]
    p = torch.softmax(lg, dim=1)
    c = p.clone()
    if gating == SOFTMAX_GROUP_MAX:
        best = p.view(T, G, -1).max(dim=2)[0]
        rank = torch.sort(torch.sort(best, dim=1, descending=True, stable=True)[1], dim=1)[1]
        c.view(T, G, -1)[rank >= tg] = 0.0
    picks = torch.sort(c, dim=1, descending=True, stable=True)[1][:, :k]
    w = torch.gather(c, 1, picks)
    w = w / w.sum(dim=1, keepdim=True) if gating == SOFTMAX_TOPK_RENORM or norm else w * scale
    dense = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, picks, w)
    hit = torch.zeros(T, E, dtype=torch.bool, device="cuda").scatter_(1, picks, True)
    y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in list(range(E)) + ([-1] if Is else []):
        rows = torch.arange(T, device="cuda") if e < 0 else hit[:, e].nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        g, n = _gen(seed, 1000 + e), Is if e < 0 else I
        (wg, sg), (wu, su), (wd, sd) = [_int8_weight(a, b, g) for a, b in ((n, H), (n, H), (H, n))]
        a, b = _x_linear(x[rows], wg, sg), _x_linear(x[rows], wu, su)
        h = (a * torch.sigmoid(a) * b).to(torch.bfloat16)
        o = _x_linear(h, wd, sd)
        y[rows] += o if e < 0 else o * dense[rows, e][:, None]
    return y


def _x_gates(shape, lg, idx, w, gw):
    """Derivative of the routing weights' formula, by torch's differentiation in 64 bits; the picks are constants."""
    _, _, E, k, _, _, _, gating, norm, scale = SHAPES[shape]
    lg = lg.double().requires_grad_(True)
    s = torch.sigmoid(lg) if gating == SIGMOID_NOAUX_TC else torch.softmax(lg, dim=1)
    p = torch.gather(s, 1, idx.long()) * (w != 0)
    if gating == SOFTMAX_TOPK_RENORM:
        v = p / p.sum(dim=1, keepdim=True)
    elif norm and k > 1:
        v = p / (p.sum(dim=1, keepdim=True) + 1e-20) * (scale if gating == SIGMOID_NOAUX_TC else 1.0)
    else:
        v = p * scale
    with torch.enable_grad():
        return torch.autograd.grad(v, lg, gw.double())[0]


def exact(case, seed):
    op = case["op"]
    if op == "linear":
        q, s = _int8_weight(case["n"], case["k"], _gen(seed, 3))
        return _x_linear(_hidden(case["m"], case["k"], _gen(seed, 2)), q, s)
    if op == "layer":
        return _x_layer(case, seed)
    keep = globals()["own"]
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = keep
    if op == "gates":
        return _x_gates(st["shape"], st["logits"], st["idx"], st["w"], st["gw"])
    dst = st["dst"].long()
    T, k = dst.shape
    n, H = st["rows"], SHAPES[st["shape"]][0]
    if op == "sort":
        owner = torch.full((n,), -1, dtype=torch.int64, device="cuda")
        owner[dst.reshape(-1)] = torch.arange(T * k, device="cuda") // k
        rows = torch.where((owner >= 0)[:, None], st["x"][owner.clamp(min=0)].double(), 0.0)
        gx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        gx.index_add_(0, owner[owner >= 0], st["grad"][owner >= 0].double())
        return rows, gx
    w = st["w"].double()
    y = torch.empty(T, H, dtype=torch.float64, device="cuda")
    gw = torch.empty(T, k, dtype=torch.float64, device="cuda")
    grows = torch.zeros(n, H, dtype=torch.float64, device="cuda")
    for t0 in range(0, T, 1024):                   # in pieces: [1024, k, H] in 64 bits
        d = dst[t0:t0 + 1024]
        r, g = st["out"][d].double(), st["gy"][t0:t0 + 1024].double()
        y[t0:t0 + 1024] = torch.einsum("tk,tkh->th", w[t0:t0 + 1024], r)
        gw[t0:t0 + 1024] = torch.einsum("th,tkh->tk", g, r)
        grows[d] = g[:, None, :] * w[t0:t0 + 1024, :, None]
    return y, grows, gw
