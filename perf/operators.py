"""What the router's training operators and the 8-bit integer products are measured on.

Five operators, each in its plain form (elementary torch operations in 32 bits) and, where `own` is true, as the
calls a user makes of k3moe:

- balance:   the router's load-balance loss with its per-sequence expert counts (k3moe.balance_loss)
- routegrad: the gradient of the router logits, from the balance loss and from the combine weights
             (k3moe.route_backward)
- linear:    y = x . W^T with int8 weights (a scale a channel) and x quantised to int8 (a scale a token):
             k3moe.quant_int8, k3moe.gemm_int8
- gated:     the same product of act(gate) * up, the down projection behind a gated activation:
             k3moe.act_quant_int8, k3moe.gemm_int8
- experts:   the products of routed rows with their experts' int8 weights, over the routing tables
             (k3moe.quant_int8_permute or k3moe.act_quant_int8, then k3moe.grouped_gemm_int8)
"""
import math
import os
import sys

import torch

own = False

TILE = 128       # rows of a routing tile
TINY = 1e-20     # added to a row's sum of scores, as the router's top-k adds it to its K picks' sum
PACKAGE = os.path.join(os.getcwd(), "kern-k3-pp-prefill_b200")


def listed():
    return [
        # a packed prefill chunk: 16 sequences in 8192 rows, 896 experts, top-8
        {"name": "balance_chunk", "op": "balance", "T": 8192, "E": 896, "K": 8, "B": 16, "masked": False},
        # a small batch of one sequence with padding, few experts: launch latency
        {"name": "balance_small", "op": "balance", "T": 64, "E": 61, "K": 4, "B": 1, "masked": True},
        # the same chunk's logits gradient, both terms, in 32 bits
        {"name": "routegrad_chunk", "op": "routegrad", "T": 8192, "E": 896, "K": 8, "B": 16, "masked": False,
         "weights": True, "dtype": "float32"},
        # a ragged padded batch, the balance term alone, rounded to bf16 for the products behind it
        {"name": "routegrad_ragged", "op": "routegrad", "T": 1531, "E": 256, "K": 4, "B": 7, "masked": True,
         "weights": False, "dtype": "bfloat16"},
        # the shared expert's gate-up product of a prefill chunk
        {"name": "linear_chunk", "op": "linear", "T": 8192, "N": 4096, "C": 7168, "dtype": "bfloat16"},
        # the same for one decoded token: the weights are read once
        {"name": "linear_token", "op": "linear", "T": 1, "N": 4096, "C": 7168, "dtype": "bfloat16"},
        # a ragged batch, sizes off every tile, 32-bit results
        {"name": "linear_ragged", "op": "linear", "T": 333, "N": 1003, "C": 2007, "dtype": "float32"},
        # the shared expert's down product of a prefill chunk
        {"name": "gated_chunk", "op": "gated", "T": 8192, "N": 7168, "C": 2048, "act": "swiglu"},
        # the same for a decode batch, with the other gate
        {"name": "gated_decode", "op": "gated", "T": 64, "N": 7168, "C": 2048, "act": "situ"},
        # gate-up products of a prefill chunk on the experts one of eight ranks holds
        {"name": "experts_up", "op": "experts", "T": 1024, "E": 112, "world": 1, "K": 8, "N": 4096, "C": 7168,
         "gated": False},
        # their down products
        {"name": "experts_down", "op": "experts", "T": 1024, "E": 112, "world": 1, "K": 8, "N": 7168, "C": 2048,
         "gated": True},
        # a decode batch: few rows, each on an expert of its own, seven in eight picks on other ranks
        {"name": "experts_decode", "op": "experts", "T": 64, "E": 112, "world": 8, "K": 8, "N": 4096, "C": 7168,
         "gated": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["balance", "routegrad", "linear", "gated", "experts"])
    if op in ("balance", "routegrad"):
        T, E = _log(rng, 1, 8192), _log(rng, 8, 896)
        c = {"op": op, "T": T, "E": E, "K": rng.choice([1, 2, 4, 8]), "B": _log(rng, 1, min(T, 64)),
             "masked": rng.random() < 0.5}
        if op == "routegrad":
            c["weights"] = rng.random() < 0.5
            c["dtype"] = rng.choice(["float32", "bfloat16"])
        return c
    if op == "linear":
        return {"op": op, "T": _log(rng, 1, 8192), "N": _log(rng, 64, 4096), "C": _log(rng, 64, 7168),
                "dtype": rng.choice(["float32", "bfloat16"])}
    if op == "gated":
        return {"op": op, "T": _log(rng, 1, 8192), "N": _log(rng, 64, 7168), "C": _log(rng, 64, 2048),
                "act": rng.choice(["swiglu", "situ"])}
    gated = rng.random() < 0.5
    return {"op": op, "T": _log(rng, 1, 1024), "E": _log(rng, 8, 112), "world": rng.choice([1, 2, 4, 8]),
            "K": rng.choice([1, 2, 4, 8]), "N": _log(rng, 64, 7168 if gated else 4096),
            "C": _log(rng, 64, 2048 if gated else 7168), "gated": gated}


# ------------------------------------------------------------------ what a program has in hand
def _inputs(case, seed):
    """The inputs themselves, from the seed alone."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    op = case["op"]
    if op in ("balance", "routegrad"):
        return _router_inputs(case, g, dev)
    T, N, C = case["T"], case["N"], case["C"]
    s = {}
    width = 2 * C if op == "gated" or case.get("gated") else C
    rows = T
    if op == "experts":
        s.update(_route(case, g, dev))
        rows = s["cap"] if case["gated"] else T
    # hidden states: of order one, a channel in 64 with outliers
    x = torch.randn((rows, width), generator=g, device=dev)
    x *= 1.0 + 7.0 * (torch.rand((1, width), generator=g, device=dev) < 1 / 64)
    s["x"] = x.to(torch.bfloat16)
    # weights as a checkpoint holds them: int8, their rows padded to a multiple of 16 bytes
    experts = case["E"] if op == "experts" else 1
    ld = -(-C // 16) * 16
    s["w"] = torch.zeros((experts * N, ld), dtype=torch.int8, device=dev)
    step = max(1, (1 << 27) // ld)
    for i in range(0, experts * N, step):
        part = s["w"][i:i + step, :C]
        part.copy_((torch.randn(part.shape, generator=g, device=dev) * 36).round_().clamp_(-127, 127))
    s["w"] = s["w"][:, :C]
    s["sw"] = (0.5 + torch.rand(experts * N, generator=g, device=dev)) / (36 * math.sqrt(C))
    return s


def _router_inputs(case, g, dev):
    T, E, K, B = case["T"], case["E"], case["K"], case["B"]
    s = {"S": torch.randn((T, E), generator=g, device=dev) * 1.5}
    bias = torch.rand(E, generator=g, device=dev) * 0.2 - 0.1
    s["idx"] = torch.topk(torch.sigmoid(s["S"]) + bias, K, dim=1).indices.to(torch.int32)
    cuts = torch.sort(torch.randint(0, T + 1, (B - 1,), generator=g, device=dev)).values
    ends = torch.tensor([T], device=dev)
    s["seq"] = torch.cat([torch.zeros_like(ends), cuts, ends]).to(torch.int32)
    s["mask"] = (torch.rand(T, generator=g, device=dev) < 0.85).to(torch.uint8) if case["masked"] else None
    s["alpha"] = 0.001
    if case["op"] == "routegrad":
        ones = _ones(s, B).double()                    # what the forward pass left behind
        hit = torch.zeros((T, E), dtype=torch.float64, device=dev)
        hit.scatter_(1, s["idx"].long(), 1.0)
        s["counts"] = (ones.t() @ hit).round().to(torch.int32)
        s["rows"] = ones.sum(0).to(torch.int32)
        s["dloss"] = 0.5 + torch.rand(1, generator=g, device=dev)
        s["rs"] = torch.tensor([2.5], dtype=torch.bfloat16, device=dev)
        s["dwts"] = torch.randn((T, K), generator=g, device=dev) * 1e-3 if case["weights"] else None
    return s


def _route(case, g, dev):
    """Picks, and the routing tables in the framework's form: an expert's rows in row order, tiles of 128 rows."""
    T, E, K = case["T"], case["E"], case["K"]
    total = E * case["world"]
    idx = torch.topk(torch.randn((T, total), generator=g, device=dev), K, dim=1).indices
    flat = idx.reshape(-1)
    local = flat < E
    key = torch.where(local, flat, total)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=total + 1)[:E]
    tiles = (counts + TILE - 1) // TILE
    first_tile = torch.cumsum(tiles, 0) - tiles
    first_pick = torch.cumsum(counts, 0) - counts
    n = int(counts.sum())
    picks = order[:n]                                   # picks by expert, then by row
    expert = flat[picks]
    place = torch.arange(n, device=dev) - first_pick[expert]
    perm = first_tile[expert] * TILE + place
    exp2perm = torch.full((T * K,), -1, dtype=torch.int32, device=dev)
    exp2perm[picks] = perm.to(torch.int32)
    max_ctas = E + -(-T * K // TILE)
    cap = max_ctas * TILE
    route_map = torch.zeros(cap, dtype=torch.int32, device=dev)
    route_map[perm] = (picks // K).to(torch.int32)
    nne = int(tiles.sum())
    cta_batch = torch.zeros(max_ctas, dtype=torch.int32, device=dev)
    cta_limit = torch.zeros(max_ctas, dtype=torch.int32, device=dev)
    tile = torch.arange(nne, device=dev)
    of = torch.repeat_interleave(torch.arange(E, device=dev), tiles)
    cta_batch[:nne] = of.to(torch.int32)
    cta_limit[:nne] = torch.minimum((tile + 1) * TILE, first_tile[of] * TILE + counts[of]).to(torch.int32)
    meta = torch.tensor([nne, nne * TILE, -1, 0], dtype=torch.int32, device=dev)
    # the plain form's plan: the experts that have rows, and each row's place among them
    touched = torch.nonzero(counts).reshape(-1)
    slot = torch.zeros(E, dtype=torch.int64, device=dev)
    slot[touched] = torch.arange(touched.numel(), device=dev)
    return {"counts": counts.to(torch.int32), "cta_batch": cta_batch, "cta_limit": cta_limit, "meta": meta,
            "route_map": route_map, "exp2perm": exp2perm.reshape(T, K), "max_ctas": max_ctas, "cap": cap,
            "perm": perm, "token": picks // K, "expert": expert, "place": place, "touched": touched,
            "slot": slot[expert], "most": int(counts.max())}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "experts":
        # rows of padding are not written
        s["out"] = torch.zeros((s["cap"], case["N"]), dtype=torch.bfloat16, device=s["x"].device)
    return s


# ------------------------------------------------------------------ the plain forms
def _ones(s, B):
    """[T, B]: whether row t counts in sequence b."""
    t = torch.arange(s["S"].shape[0], device=s["S"].device)[:, None]
    one = (t >= s["seq"][None, :B]) & (t < s["seq"][None, 1:])
    return one if s["mask"] is None else one & (s["mask"][:, None] != 0)


def _scores(s):
    score = torch.sigmoid(s["S"])
    z = score.sum(1, keepdim=True) + TINY
    return score, z


def _balance(s, case):
    E, K, B = case["E"], case["K"], case["B"]
    ones = _ones(s, B)
    score, z = _scores(s)
    p = torch.where(ones.any(1, keepdim=True), score / z, 0.0)
    hit = torch.zeros_like(p).scatter_(1, s["idx"].long(), 1.0)
    of = ones.float().t()
    counts, prob, rows = of @ hit, of @ p, of.sum(1)
    n = rows.clamp(min=1)[:, None]
    each = (E / K * counts / n * prob / n).sum(1)
    full = (rows > 0).sum().clamp(min=1)
    loss = (s["alpha"] * each.sum() / full).reshape(1)
    return {"loss": loss, "counts": counts.to(torch.int32), "prob": prob, "rows": rows.to(torch.int32)}


def _routegrad(s, case):
    E, K, B = case["E"], case["K"], case["B"]
    score, z = _scores(s)
    slope = score * torch.sigmoid(-s["S"])
    ones = _ones(s, B)
    full = (s["rows"] > 0).sum().clamp(min=1)
    n = s["rows"].clamp(min=1).float()[:, None]
    f = s["alpha"] * s["dloss"] / full * E / K * s["counts"].float() / n / n    # [B, E]
    ft = ones.float() @ f
    p = score / z
    dS = torch.where(ones.any(1, keepdim=True), (ft - (ft * p).sum(1, keepdim=True)) * slope / z, 0.0)
    if s["dwts"] is not None:
        idx = s["idx"].long()
        sk = score.gather(1, idx)
        den = sk.sum(1, keepdim=True) + TINY
        mean = (s["dwts"] * sk).sum(1, keepdim=True) / den
        dS = dS.scatter_add(1, idx, s["rs"].float() / den * (s["dwts"] - mean) * slope.gather(1, idx))
    return dS.to(getattr(torch, case["dtype"]))


def _quant(x):
    """int8 codes (as floats) and a scale a row: the largest magnitude becomes 127."""
    amax = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127.0 / amax.clamp(min=torch.finfo(torch.float32).tiny))
    return q, amax / 127.0


def _gate(x, act):
    g, u = x.float().chunk(2, dim=1)
    if act == "swiglu":
        return g * torch.sigmoid(g) * u
    return 4.0 * torch.tanh(g / 4.0) * torch.sigmoid(g) * (25.0 * torch.tanh(u / 25.0))


def _product(s, case):
    x = _gate(s["x"], case["act"]) if case["op"] == "gated" else s["x"].float()
    q, sx = _quant(x)
    y = (q @ s["w"].float().t()) * sx * s["sw"]
    return y.to(getattr(torch, case.get("dtype", "bfloat16")))


def _experts(s, case):
    E, N, C = case["E"], case["N"], case["C"]
    out = torch.zeros((s["cap"], N), dtype=torch.bfloat16, device=s["x"].device)
    if s["perm"].numel() == 0:
        return out
    x = _gate(s["x"][s["perm"]], "swiglu") if case["gated"] else s["x"].float()
    q, sx = _quant(x)
    if not case["gated"]:
        q, sx = q[s["token"]], sx[s["token"]]
    a = torch.zeros((s["touched"].numel(), s["most"], C), device=q.device)
    a[s["slot"], s["place"]] = q
    w = s["w"].reshape(E, N, C) if s["w"].is_contiguous() else s["w"].unflatten(0, (E, N))
    y = torch.bmm(a, w[s["touched"]].float().transpose(1, 2))[s["slot"], s["place"]]
    out[s["perm"]] = (y * sx * s["sw"].reshape(E, N)[s["expert"]]).to(torch.bfloat16)
    return out


# ------------------------------------------------------------------ one pass
def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        return _own(s, case)
    if op == "balance":
        return _balance(s, case)
    if op == "routegrad":
        return _routegrad(s, case)
    return _experts(s, case) if op == "experts" else _product(s, case)


def _own(s, case):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import k3moe

    op = case["op"]
    if op == "balance":
        b = k3moe.balance_loss(s["S"], s["idx"], s["alpha"], seq=s["seq"], mask=s["mask"])
        return {"loss": b.loss, "counts": b.counts, "prob": b.prob, "rows": b.rows}
    if op == "routegrad":
        return k3moe.route_backward(s["S"], s["idx"], s["alpha"], counts=s["counts"], rows=s["rows"], dloss=s["dloss"],
                                    dwts=s["dwts"], rs=s["rs"], seq=s["seq"], mask=s["mask"],
                                    dtype=getattr(torch, case["dtype"]))
    if op in ("linear", "gated"):
        if op == "linear":
            q, sx = k3moe.quant_int8(s["x"])
        else:
            q, sx = k3moe.act_quant_int8(s["x"], k3moe.ACT_SITU if case["act"] == "situ" else k3moe.ACT_SWIGLU)
        return k3moe.gemm_int8(q, sx, s["w"], s["sw"], dtype=getattr(torch, case.get("dtype", "bfloat16")))
    t = k3moe.Tables(counts=s["counts"], cta_batch=s["cta_batch"], cta_limit=s["cta_limit"], meta=s["meta"],
                     route_map=s["route_map"], exp2perm=s["exp2perm"], max_ctas=s["max_ctas"], cap_rows=s["cap"])
    if case["gated"]:
        q, sx = k3moe.act_quant_int8(s["x"], k3moe.ACT_SWIGLU, tables=t)
    else:
        q, sx = k3moe.quant_int8_permute(s["x"], t)
    return k3moe.grouped_gemm_int8(q, sx, s["w"], s["sw"], t, case["E"], out=s["out"])


# ------------------------------------------------------------------ work, and the definition in 64 bits
def work(case):
    op = case["op"]
    if op in ("balance", "routegrad"):
        T, E, K, B = case["T"], case["E"], case["K"], case["B"]
        n = 4 * T * E + 4 * T * K + 4 * (B + 1) + 8 * B * E + (T if case["masked"] else 0)
        if op == "routegrad":
            n += T * E * (4 if case["dtype"] == "float32" else 2) + (4 * T * K if case["weights"] else 0) - 4 * B * E
        return {"bytes": n, "flops": 10 * T * E}
    T, N, C = case["T"], case["N"], case["C"]
    if op in ("linear", "gated"):
        size = 4 if case.get("dtype") == "float32" else 2
        return {"bytes": 2 * T * C * (2 if op == "gated" else 1) + N * C + 4 * N + size * T * N, "flops": 2 * T * N * C}
    # picks on this rank and experts with a row, as uniform routing gives them
    rows = T * case["K"] / case["world"]
    experts = case["E"] * (1 - (1 - 1 / case["E"]) ** rows)
    read = 2 * rows * 2 * C if case["gated"] else 2 * T * C
    return {"bytes": read + experts * N * C + 2 * rows * N, "flops": 2 * rows * N * C}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op in ("balance", "routegrad"):
        return _exact_router(s, case)
    x = s["x"].double()
    if op == "gated" or case.get("gated"):
        half = x.shape[1] // 2
        g, u = x[:, :half], x[:, half:]
        if case.get("act") == "situ":
            x = 100 * torch.tanh(g / 4) * torch.tanh(u / 25) / (1 + torch.exp(-g))
        else:
            x = g * u / (1 + torch.exp(-g))
    amax = x.abs().max(dim=1).values[:, None]
    codes = torch.round(127 * x / torch.where(amax > 0, amax, 1.0))
    scale = amax / 127
    N = case["N"]
    if op != "experts":
        # sums of products of codes below 2^53: exact
        return torch.matmul(codes, s["w"].double().T) * scale * s["sw"].double()[None]
    out = torch.zeros((s["cap"], N), dtype=torch.float64, device=x.device)
    bounds = torch.cumsum(s["counts"], 0).tolist()
    at = 0
    for e, end in enumerate(bounds):
        if end > at:
            rows = s["perm"][at:end]
            src = rows if case["gated"] else s["token"][at:end]
            w = s["w"][e * N:(e + 1) * N].double()
            out[rows] = torch.matmul(codes[src], w.T) * scale[src] * s["sw"][e * N:(e + 1) * N].double()
        at = end
    return out


def _exact_router(s, case):
    E, K, B, T = case["E"], case["K"], case["B"], case["T"]
    sig = 1 / (1 + torch.exp(-s["S"].double()))
    down = 1 / (1 + torch.exp(s["S"].double()))
    z = sig.sum(dim=1, keepdim=True) + 1e-20
    cuts = s["seq"].tolist()
    on = torch.ones(T, dtype=torch.bool, device=sig.device) if s["mask"] is None else s["mask"] != 0
    parts, counts, prob, rows = [], [], [], []
    for b in range(B):
        at = torch.arange(cuts[b], cuts[b + 1], device=sig.device)
        at = at[on[cuts[b]:cuts[b + 1]]]
        parts.append(at)
        rows.append(at.numel())
        counts.append(torch.bincount(s["idx"][at].reshape(-1).long(), minlength=E))
        prob.append((sig[at] / z[at]).sum(dim=0))
    full = max(1, sum(n > 0 for n in rows))
    if case["op"] == "balance":
        each = [(E * c.double() / (K * n) * p / n).sum() for c, p, n in zip(counts, prob, rows) if n]
        loss = s["alpha"] * torch.stack(each).sum() / full if each else torch.zeros((), device=sig.device).double()
        return {"loss": loss.reshape(1), "counts": None, "prob": torch.stack(prob), "rows": None}
    grad = torch.zeros((T, E), dtype=torch.float64, device=sig.device)
    for at, c, n in zip(parts, counts, rows):
        if n:
            f = s["alpha"] * s["dloss"].double() * E * c.double() / (K * n * n * full)
            p = sig[at] / z[at]
            grad[at] = (f[None] - (p @ f)[:, None]) * p * down[at]
    if s["dwts"] is not None:
        at = s["idx"].long()
        sk, dk = torch.take_along_dim(sig, at, 1), torch.take_along_dim(down, at, 1)
        den = sk.sum(dim=1, keepdim=True) + 1e-20
        dw = s["dwts"].double()
        ds = s["rs"].double() * (dw * den - (dw * sk).sum(dim=1, keepdim=True)) / den ** 2
        grad.scatter_add_(1, at, ds * sk * dk)
    return grad
