"""Cases that time the residual's addition with the RMS norm behind it (rows out in bf16 or in 8-bit integers), its gradient,
and low-rank adapters beside a projection, for serving and for training, through the public entry points, beside plain forms
in elementary torch operations.

Kinds of case ("op"):
  norm       h = x + residual, y = weight * h / sqrt(mean(h^2) + eps): MoELayer.add_rmsnorm, or with "out": "int8" the rows
             quantised: MoELayer.add_rmsnorm_int8.  "rows", "cols", "ld" (elements between rows), "residual" (False: h = x)
  norm_grad  gradients of h and of the weight, with the gradient that reaches h itself: MoELayer.add_rmsnorm_grad.
             "rows", "cols"
  adapt      out[t] = y[t] + scale[g] (x[t] . down[g]^T) . up[g]^T, g = ids[t]: MoELayer.adapter_add.  "rows", "cols",
             "n_out", "rank", "adapters", "run" (mean length of a run of rows of one request)
  train      the same over rows sorted by expert, an adapter to an expert, and the gradients of rows and adapters:
             MoELayer.adapter_plan_sorted, .adapter_add and .adapter_grad.  "tokens", "top_k", "adapters", "cols", "n_out",
             "rank"

h is rounded to bf16 before it is normalised, as a residual stream is that is kept in bf16.  Quantisation of a normalised row
(fp32; int8, symmetric): m = max(max|y|, 2^-100), scale = m / 127 and inv = 127 / m in fp32, q = y * inv rounded to the nearest
integer, ties to even; the row's values are q * scale.
"""
import math

import torch

own = False

EPS = 1e-6
# hidden, experts, top_k
SHAPES = {"v2lite": (2048, 64, 6), "mixtral8x7b": (4096, 8, 2), "v2_236b": (5120, 160, 6), "v3": (7168, 256, 8)}
NORM_ELEMENTS = 16384 * 7168
NORM8_ELEMENTS = GRAD_ELEMENTS = 8192 * 7168
ADAPT_ELEMENTS = 8192 * 4096                # rows * the longer of cols and n_out
ADAPTER_ELEMENTS = 1 << 26                  # adapters * rank * (cols + n_out)
TRAIN_ELEMENTS = 8192 * 6 * 2048


def listed():
    return [
        # one sequence decoding, in front of the block: launch and latency
        {"name": "norm_1", "op": "norm", "rows": 1, "cols": 4096, "ld": 4096, "residual": True, "out": "bf16"},
        # the norm over a compressed cache entry, 512 of 576 columns, of an odd decode batch
        {"name": "norm_part_203", "op": "norm", "rows": 203, "cols": 512, "ld": 576, "residual": False, "out": "bf16"},
        # the residual stream of a large prefill batch of the widest model
        {"name": "norm_16384", "op": "norm", "rows": 16384, "cols": 7168, "ld": 7168, "residual": True, "out": "bf16"},
        # a small batch in front of int8 experts
        {"name": "norm8_37", "op": "norm", "rows": 37, "cols": 2048, "ld": 2048, "residual": True, "out": "int8"},
        # a prefill batch in front of int8 experts or projections
        {"name": "norm8_8192", "op": "norm", "rows": 8192, "cols": 7168, "ld": 7168, "residual": True, "out": "int8"},
        # a calibration batch's way back through the norm
        {"name": "norm_grad_37", "op": "norm_grad", "rows": 37, "cols": 2048},
        # the same for a training micro-batch of the widest model
        {"name": "norm_grad_8192", "op": "norm_grad", "rows": 8192, "cols": 7168},
        # one sequence decoding with one of eight adapters
        {"name": "adapt_1", "op": "adapt", "rows": 1, "cols": 4096, "n_out": 4096, "rank": 16, "adapters": 8, "run": 1},
        # an odd decode batch, a request to a row, 64 adapters of a rank and an output that no tile divides
        {"name": "adapt_201_ragged", "op": "adapt", "rows": 201, "cols": 5120, "n_out": 1000, "rank": 12, "adapters": 64, "run": 1},
        # prompts of a few requests through a projection of the widest model
        {"name": "adapt_8192", "op": "adapt", "rows": 8192, "cols": 4096, "n_out": 4096, "rank": 64, "adapters": 8, "run": 700},
        # a calibration batch on 64 experts with an adapter each
        {"name": "train_v2lite_37", "op": "train", "tokens": 37, "top_k": 6, "adapters": 64, "cols": 2048, "n_out": 2048, "rank": 8},
        # a training micro-batch of the same layer
        {"name": "train_v2lite_8192", "op": "train", "tokens": 8192, "top_k": 6, "adapters": 64, "cols": 2048, "n_out": 2048,
         "rank": 16},
    ]


def _log_size(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "adapt", "adapt", "train"])
    if op == "norm":
        out = rng.choice(["bf16", "int8"])
        cols = rng.choice([rng.choice(sorted(SHAPES.values()))[0], _log_size(rng, 64, 8192)])
        rows = _log_size(rng, 1, (NORM8_ELEMENTS if out == "int8" else NORM_ELEMENTS) // 7168)
        return {"op": op, "rows": rows, "cols": cols, "ld": cols + rng.choice([0, 0, 64, 5]), "residual": rng.random() < 0.7,
                "out": out}
    if op == "norm_grad":
        cols = rng.choice([rng.choice(sorted(SHAPES.values()))[0], _log_size(rng, 64, 8192)])
        return {"op": op, "rows": _log_size(rng, 1, GRAD_ELEMENTS // max(cols, 7168)), "cols": cols}
    rank = rng.choice([4, 8, 12, 16, 32, 64, 100, 128])
    cols, n_out = _log_size(rng, 64, 8192), _log_size(rng, 16, 8192)
    if op == "adapt":
        adapters = _log_size(rng, 1, max(1, min(256, ADAPTER_ELEMENTS // (rank * (cols + n_out)))))
        rows = _log_size(rng, 1, min(8192, ADAPT_ELEMENTS // max(cols, n_out)))
        if rows > 1024:
            rank = min(rank, 64)
        return {"op": op, "rows": rows, "cols": cols, "n_out": n_out, "rank": rank, "adapters": adapters,
                "run": rng.choice([1, _log_size(rng, 1, 1000)])}
    hidden, experts, top_k = SHAPES[rng.choice(sorted(SHAPES))]
    rank = min(rank, 16 if experts > 8 else 64)
    return {"op": op, "tokens": _log_size(rng, 1, TRAIN_ELEMENTS // (2 * top_k * hidden)), "top_k": top_k, "adapters": experts,
            "cols": hidden, "n_out": hidden, "rank": rank}


# ------------------------------------------------------------------ inputs, from the seed alone
def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) % (1 << 62))
    return g


def _hidden(rows, cols, g, ld=None):
    """Hidden states [rows, cols], ld elements apart: unit variance, one channel in 64 eight times as wide (the outliers of
    real activations)."""
    x = torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.bfloat16)
    x[:, ::64] *= 8.0
    if ld is None or ld == cols:
        return x
    wide = torch.zeros(rows, ld, device="cuda", dtype=torch.bfloat16)
    wide[:, :cols] = x
    return wide[:, :cols]


def _norm_weight(cols, g):
    return (0.5 + torch.rand(cols, generator=g, device="cuda")).to(torch.bfloat16)


def _adapters(case, seed):
    """down [adapters, rank, cols] and up [adapters, n_out, rank], rows on 16-byte boundaries, and scales [adapters]."""
    A, r, K, N = case["adapters"], case["rank"], case["cols"], case["n_out"]
    g = _gen(seed, 11)
    made = []
    for rows, cols, std in ((r, K, K ** -0.5), (N, r, r ** -0.5)):
        m = torch.zeros(A, rows, (cols + 7) // 8 * 8, device="cuda", dtype=torch.bfloat16)[:, :, :cols]
        m.copy_(torch.randn(A, rows, cols, generator=g, device="cuda", dtype=torch.bfloat16) * std)
        made.append(m)
    return made[0], made[1], 0.5 + torch.rand(A, generator=g, device="cuda")


def _rows16(rows, cols, g):
    """Rows on 16-byte boundaries whatever their length."""
    m = torch.empty(rows, (cols + 7) // 8 * 8, device="cuda", dtype=torch.bfloat16)[:, :cols]
    return m.copy_(_hidden(rows, cols, g))


def _ids(case, seed):
    """An adapter to each row, in runs of one request's rows; adapters differ in popularity; one request in 16 has none."""
    T, A, run = case["rows"], case["adapters"], case["run"]
    g = _gen(seed, 12)
    start = torch.rand(T, generator=g, device="cuda") < 1.0 / run
    request = torch.cumsum(start.long(), 0)
    pick = (torch.rand(T + 1, generator=g, device="cuda") ** 2 * A).long().clamp_(max=A - 1)
    pick[torch.rand(T + 1, generator=g, device="cuda") < 1.0 / 16] = -1
    return pick[request].int()


def _padded_rows(R, E):
    """Rows of a buffer that holds R rows sorted by expert whatever the routing (MoELayer.padded_rows)."""
    return ((R + 127) // 128 + E) * 128


def _segments(case, seed):
    """Rows of every expert for picks of distinct experts per token, the load uneven, every expert's rows on a 128-row
    boundary: counts, first rows, rows of the buffer."""
    T, k, E = case["tokens"], case["top_k"], case["adapters"]
    g = _gen(seed, 13)
    score = torch.rand(T, E, generator=g, device="cuda") + 0.5 * torch.rand(E, generator=g, device="cuda")
    counts = torch.bincount(score.topk(k, dim=1)[1].reshape(-1), minlength=E)
    pad = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    pad[1:] = torch.cumsum((counts + 127) // 128 * 128, 0)
    return counts.int(), pad.int(), _padded_rows(T * k, E)


def _live(counts, pad, rows):
    at = torch.arange(rows, device=counts.device)
    e = torch.searchsorted(pad[1:].long(), at, right=True).clamp_(max=counts.numel() - 1)
    return at - pad[e] < counts[e]


def prepare(case, seed):
    op, st = case["op"], dict(case)
    if own:
        from moe_gen_b200 import MoELayer
        st["layer"] = MoELayer(hidden=256, inter=128, n_experts=8, top_k=2)      # any layer serves
    if op == "norm":
        R, C = case["rows"], case["cols"]
        st["x"], st["w"] = _hidden(R, C, _gen(seed, 1), case["ld"]), _norm_weight(C, _gen(seed, 2))
        st["res"] = _hidden(R, C, _gen(seed, 3), case["ld"]) if case["residual"] else None
    elif op == "norm_grad":
        R, C = case["rows"], case["cols"]
        st["h"], st["w"] = _hidden(R, C, _gen(seed, 1)), _norm_weight(C, _gen(seed, 2))
        st["gy"], st["gh"] = (torch.randn(R, C, generator=_gen(seed, s), device="cuda", dtype=torch.bfloat16) for s in (4, 5))
    else:
        st["down"], st["up"], st["scale"] = _adapters(case, seed)
        if op == "adapt":
            st["ids"], R = _ids(case, seed), case["rows"]
            st["x"], st["y"] = _rows16(R, case["cols"], _gen(seed, 14)), _rows16(R, case["n_out"], _gen(seed, 15))
        else:
            st["counts"], st["pad"], st["n"] = _segments(case, seed)
            live = _live(st["counts"], st["pad"], st["n"]).unsqueeze(1)          # rows that hold no pick are zeros
            for what, cols, s in (("x", case["cols"], 14), ("y", case["n_out"], 15), ("go", case["n_out"], 16)):
                st[what] = _hidden(st["n"], cols, _gen(seed, s)) * live
    return st


# ------------------------------------------------------------------ plain forms
def _sum_and_rows(st):
    """h (bf16) and its normalised rows in fp32."""
    h = st["x"] if st["res"] is None else (st["x"].float() + st["res"].float()).to(torch.bfloat16)
    f = h.float()
    return h, f / torch.sqrt((f * f).mean(dim=1, keepdim=True) + EPS) * st["w"].float()


def _tiles(first, counts, order, n_tiles, size):
    """Rows in tiles of one adapter each: the adapter of a tile, its rows and which of them exist."""
    G = counts.numel()
    ends = torch.cumsum((counts + size - 1) // size, 0)
    tile = torch.arange(n_tiles, device=counts.device)
    g = torch.searchsorted(ends, tile, right=True)
    some = g < G
    g = g.clamp(max=G - 1)
    inside = (tile - (ends[g] - (counts[g] + size - 1) // size)).unsqueeze(1) * size + torch.arange(size, device=counts.device)
    live = some.unsqueeze(1) & (inside < counts[g].unsqueeze(1))
    at = torch.where(live, first[g].unsqueeze(1) + inside, torch.zeros_like(inside))
    return g, order[at] if order is not None else at, live


def _take(rows, at, live):
    return rows[at.reshape(-1)].float().view(*at.shape, -1) * live.unsqueeze(2)


def _bring(out, at, values):
    """out += the tiles' rows; those that do not exist bring zeros to some row."""
    return out.index_add_(0, at.reshape(-1), values.reshape(-1, values.shape[2]))


def _adapter_plain(st, first, counts, order, rows, grad):
    """Adapters over rows that come sorted (order: None) or by an order, tile by tile."""
    G = counts.numel()
    size = 1
    while size < 64 and size * G < rows:
        size *= 2
    g, at, live = _tiles(first, counts, order, (rows + size - 1) // size + G, size)
    down, up, scale = st["down"][g].float(), st["up"][g].float(), st["scale"][g].view(-1, 1, 1)
    x = _take(st["x"], at, live)
    s = torch.bmm(x, down.transpose(1, 2))
    out = _bring(st["y"].float(), at, torch.bmm(s, up.transpose(1, 2)) * scale).to(torch.bfloat16)
    if not grad:
        return out
    go = _take(st["go"], at, live)
    gs = torch.bmm(go, up) * scale
    gx = _bring(torch.zeros(st["x"].shape, device=x.device), at, torch.bmm(gs, down))
    gdown = torch.zeros(st["down"].shape, device=x.device).index_add_(0, g, torch.bmm(gs.transpose(1, 2), x))
    gup = torch.zeros(st["up"].shape, device=x.device).index_add_(0, g, torch.bmm(go.transpose(1, 2), s) * scale)
    return out, gx.to(torch.bfloat16), gdown.to(torch.bfloat16), gup.to(torch.bfloat16)


def run(st):
    op = st["op"]
    if op == "norm":
        if st["out"] == "int8":
            if own:
                q, scale, h = st["layer"].add_rmsnorm_int8(st["x"], st["res"], st["w"], EPS)
            else:
                h, y = _sum_and_rows(st)
                m = y.abs().amax(dim=1).clamp_min(2.0 ** -100)
                scale, q = m / 127.0, torch.round(y.double() * (127.0 / m).double().unsqueeze(1)).to(torch.int8)
            values = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
            torch.mul(q, scale.unsqueeze(1), out=values)
            return (values, scale) if st["res"] is None else (values, scale, h)
        if own:
            y, h = st["layer"].add_rmsnorm(st["x"], st["res"], st["w"], EPS)
        else:
            h, y = _sum_and_rows(st)
            y = y.to(torch.bfloat16)
        return y if st["res"] is None else (y, h)
    if op == "norm_grad":
        if own:
            return st["layer"].add_rmsnorm_grad(st["gy"], st["h"], st["w"], EPS, st["gh"])
        h, gy = st["h"].float(), st["gy"].float()
        inv = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        n, wg = h * inv, st["w"].float() * gy
        gx = (wg - n * (wg * n).mean(dim=1, keepdim=True)) * inv + st["gh"].float()
        return gx.to(torch.bfloat16), (gy.double() * n.double()).sum(dim=0).float()        # long sums in 64 bits
    if op == "adapt":
        if own:
            return st["layer"].adapter_add(st["y"], st["x"], st["down"], st["up"], st["ids"], st["scale"])
        ids, G = st["ids"].long(), st["adapters"]
        some = torch.where(ids < 0, torch.full_like(ids, G), ids)
        counts = torch.bincount(some, minlength=G + 1)[:G]
        order = torch.sort(some, stable=True)[1]
        return _adapter_plain(st, torch.cumsum(counts, 0) - counts, counts, order, st["rows"], False)
    if own:
        layer = st["layer"]
        plan = layer.adapter_plan_sorted(st["counts"], st["pad"], st["n"])
        out, s = layer.adapter_add(st["y"], st["x"], st["down"], st["up"], plan, st["scale"], keep=True)
        return (out,) + tuple(layer.adapter_grad(st["go"], st["x"], st["down"], st["up"], plan, st["scale"], s))
    return _adapter_plain(st, st["pad"][:-1].long(), st["counts"].long(), None, st["tokens"] * st["top_k"], True)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["cols"]
        moved = 2 * n + (4 * n if case["residual"] else 0) + (n + 2 * n if case["out"] == "int8" else 2 * n)
        if case["out"] == "int8":
            moved += n                             # the values that are returned: written above, made of the bytes
        return {"bytes": moved + 2 * case["cols"], "flops": 6 * n}
    if op == "norm_grad":
        n = case["rows"] * case["cols"]
        return {"bytes": 8 * n + 6 * case["cols"], "flops": 12 * n}
    K, N, r, A = case["cols"], case["n_out"], case["rank"], case["adapters"]
    if op == "adapt":
        T = case["rows"]
        requests = max(1.0, T / case["run"])
        hit = min(A * (1.0 - (1.0 - 1.0 / A) ** requests), requests)
        return {"bytes": int(2 * T * (K + 2 * N) + 2 * hit * r * (K + N) + 4 * T), "flops": 2 * T * r * (K + N)}
    R = case["tokens"] * case["top_k"]
    P = _padded_rows(R, A)
    hit = A * (1.0 - (1.0 - case["top_k"] / A) ** case["tokens"])
    # rows in once for either direction, rows out (those without a pick too), adapters in and their gradients out
    return {"bytes": int(2 * R * (K + N) + 2 * P * N + 2 * R * N + 2 * P * K + 2 * hit * r * (K + N) + 2 * A * r * (K + N)),
            "flops": 6 * R * r * (K + N)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _x_norm(h, w):
    h = h.double()
    return torch.rsqrt(h.square().sum(dim=1, keepdim=True) / h.shape[1] + EPS) * h * w.double()


def _x_adapters(st, rows_of, grad):
    out = st["y"].double()
    gx = torch.zeros(st["x"].shape, dtype=torch.float64, device="cuda")
    gdown, gup = (torch.zeros(st[k].shape, dtype=torch.float64, device="cuda") for k in ("down", "up"))
    for e in range(st["adapters"]):
        rows = rows_of(e)
        if rows.numel() == 0:
            continue
        A, B, c = st["down"][e].double(), st["up"][e].double(), st["scale"][e].double()
        x = st["x"][rows].double()
        s = torch.einsum("tk,rk->tr", x, A)
        out[rows] += c * torch.einsum("tr,nr->tn", s, B)
        if grad:
            go = st["go"][rows].double()
            gs = c * torch.einsum("tn,nr->tr", go, B)
            gx[rows] = torch.einsum("tr,rk->tk", gs, A)
            gdown[e] = torch.einsum("tr,tk->rk", gs, x)
            gup[e] = c * torch.einsum("tn,tr->nr", go, s)
    return (out, gx, gdown, gup) if grad else out


def exact(case, seed):
    keep = globals()["own"]
    globals()["own"] = False
    try:
        st = prepare(case, seed)
    finally:
        globals()["own"] = keep
    op = case["op"]
    if op == "norm":
        h = st["x"] if st["res"] is None else (st["x"].double() + st["res"].double()).to(torch.bfloat16)
        y = _x_norm(h, st["w"])
        if case["out"] == "int8":
            m = torch.clamp(y.abs().max(dim=1)[0], min=2.0 ** -100).float()
            y = torch.round(y * (127.0 / m).double()[:, None]) * (m / 127.0).double()[:, None]
            return (y, (m / 127.0).double()) if st["res"] is None else (y, (m / 127.0).double(), h.double())
        return y if st["res"] is None else (y, h.double())
    if op == "norm_grad":
        h, w = st["h"].double().requires_grad_(True), st["w"].double().requires_grad_(True)
        with torch.enable_grad():
            y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * w
            gh, gw = torch.autograd.grad(y, (h, w), st["gy"].double())
        return gh + st["gh"].double(), gw
    if op == "adapt":
        return _x_adapters(st, lambda e: (st["ids"] == e).nonzero()[:, 0], False)
    pad, counts = st["pad"].tolist(), st["counts"].tolist()
    return _x_adapters(st, lambda e: torch.arange(pad[e], pad[e] + counts[e], device="cuda"), True)
