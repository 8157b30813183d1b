"""The operators of a mixture-of-experts layer: cases, plain forms and calls.

A token's logits choose k of E experts (`route`), its row is copied to its experts' groups (`gather`), each group is
multiplied by its expert's matrix (`grouped`; `gemv_w4` with 4-bit weights, where a group has a few rows) and the
products are added up per token (`combine`).  The training directions are cases of their own: `route_grad`,
`combine_grad`, and `grouped` with respect to the rows (`dgrad`) and to the weights (`wgrad`).

With `own` false `run` computes an operator from elementary torch operations in 32 bits; with `own` true it makes the
calls of this package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence being decoded: nothing but latency
        {"name": "route 1 token", "op": "route", "tokens": 1, "experts": 64, "k": 4, "type": "f32", "renorm": True, "masked": 0.0},
        # a training step's tokens, some of them padding, some experts closed to some tokens
        {"name": "route 16384 tokens", "op": "route", "tokens": 16384, "experts": 128, "k": 8, "type": "bf16", "renorm": True,
         "masked": 0.05},
        # its backward pass, weights from the softmax over all experts
        {"name": "route grad 8192 tokens", "op": "route_grad", "tokens": 8192, "experts": 256, "k": 8, "type": "f32", "renorm": False,
         "masked": 0.02},
        # rows of a prefill or training batch into expert order
        {"name": "gather 8192x4096 k4", "op": "gather", "tokens": 8192, "experts": 64, "k": 4, "width": 4096, "type": "bf16",
         "dropped": 0.05},
        # a small batch being decoded, back into token order
        {"name": "combine 257x2048 k8", "op": "combine", "tokens": 257, "experts": 64, "k": 8, "width": 2048, "type": "f16",
         "dropped": 0.0},
        # the training batch's gradient of both the rows and the weights
        {"name": "combine grad 8192x4096 k4", "op": "combine_grad", "tokens": 8192, "experts": 64, "k": 4, "width": 4096, "type": "bf16",
         "dropped": 0.05},
        # decoding: a few rows for each expert, every expert's matrix read
        {"name": "grouped 64 rows", "op": "grouped", "side": "fwd", "rows": 64, "spare": 0, "experts": 32, "n": 2048, "k": 4096,
         "skew": 0.5, "type": "bf16"},
        # a training batch
        {"name": "grouped 32768 rows", "op": "grouped", "side": "fwd", "rows": 32768, "spare": 1024, "experts": 32, "n": 4096, "k": 4096,
         "skew": 0.5, "type": "bf16"},
        # odd sizes, uneven groups
        {"name": "grouped dgrad 5003 rows", "op": "grouped", "side": "dgrad", "rows": 5003, "spare": 61, "experts": 9, "n": 1000,
         "k": 2056, "skew": 1.0, "type": "bf16"},
        # a training batch's weight gradients, kept in 32 bits
        {"name": "grouped wgrad 16384 rows", "op": "grouped", "side": "wgrad", "rows": 16384, "spare": 0, "experts": 16, "n": 2048,
         "k": 4096, "skew": 0.5, "type": "f32"},
        # one token through one large matrix
        {"name": "gemv w4 1x8192x8192", "op": "gemv_w4", "rows": 1, "experts": 1, "n": 8192, "k": 8192, "group": 128, "zeros": False,
         "skew": 0.0, "type": "bf16"},
        # a decoded batch's rows over the experts' 4-bit matrices
        {"name": "gemv w4 24 rows 16 experts", "op": "gemv_w4", "rows": 24, "experts": 16, "n": 4096, "k": 2048, "group": 32,
         "zeros": True, "skew": 0.5, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["route", "route_grad", "gather", "combine", "combine_grad", "grouped", "grouped", "grouped", "gemv_w4", "gemv_w4"])
    if op in ("route", "route_grad"):
        experts = _log(rng, 4, 512)
        return {"op": op, "tokens": _log(rng, 1, 32768), "experts": experts, "k": rng.randint(1 if op == "route" else 2, min(8, experts)),
                "type": rng.choice(["f32", "bf16", "f16"]), "renorm": rng.random() < 0.5, "masked": rng.choice([0.0, 0.02, 0.2])}
    if op in ("gather", "combine", "combine_grad"):
        experts = _log(rng, 8, 256)
        return {"op": op, "tokens": _log(rng, 1, 16384), "experts": experts, "k": rng.randint(1, 8),
                "width": _log(rng, 64, 8192) if rng.random() < 0.2 else 8 * _log(rng, 8, 1024),
                "type": rng.choice(["f32", "bf16", "f16"]), "dropped": rng.choice([0.0, 0.1])}
    if op == "grouped":
        side = rng.choice(["fwd", "dgrad", "wgrad"])
        return {"op": op, "side": side, "rows": _log(rng, 1, 32768), "spare": rng.choice([0, 0, 17, 300]), "experts": _log(rng, 1, 64),
                "n": 8 * _log(rng, 16, 1024), "k": 8 * _log(rng, 16, 1024), "skew": rng.choice([0.0, 0.5, 1.0]),
                "type": rng.choice(["bf16", "f32"]) if side == "wgrad" else "bf16"}
    group = rng.choice([32, 64, 128])
    return {"op": op, "rows": _log(rng, 1, 64), "experts": rng.choice([1, 1, _log(rng, 2, 64)]), "n": _log(rng, 100, 16384),
            "k": group * _log(rng, max(1, 256 // group), 16384 // group), "group": group, "zeros": rng.random() < 0.5,
            "skew": rng.choice([0.0, 0.5]), "type": rng.choice(["bf16", "f16"])}


def draw(rng):
    most = max((work(c) for c in listed()), key=lambda w: w["flops"])
    bytes_most = max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= most["flops"] and w["bytes"] <= bytes_most:
            return case


def work(case):
    op = case["op"]
    if op in ("route", "route_grad"):
        T, E, k, s = case["tokens"], case["experts"], case["k"], SIZE[case["type"]]
        if op == "route":  # logits; choice, weight, position and order of each; the groups' borders
            return {"bytes": T * E * s + T * k * 16 + (E + 1) * 4, "flops": 3 * T * E}
        return {"bytes": 2 * T * E * s + T * k * 12, "flops": 6 * T * E}
    if op in ("gather", "combine", "combine_grad"):
        T, k, H, s = case["tokens"], case["k"], case["width"], SIZE[case["type"]]
        n = T * k * (1 - case["dropped"])
        if op == "gather":
            return {"bytes": (T + n) * H * s + T * k * 4, "flops": 0}
        if op == "combine":
            return {"bytes": (T + n) * H * s + T * k * 8, "flops": 2 * n * H}
        return {"bytes": (T + 2 * n) * H * s + T * k * 12, "flops": 3 * n * H}
    R, E, N, K = case["rows"], case["experts"], case["n"], case["k"]
    used = E * (1 - (1 - 1 / E) ** R)  # experts with a row at all
    if op == "grouped":
        weights = E * N * K * SIZE[case["type"]] if case["side"] == "wgrad" else used * N * K * 2
        return {"bytes": weights + R * (N + K) * 2, "flops": 2 * R * N * K}
    scales = N * K // case["group"] * (3 if case["zeros"] else 2)
    return {"bytes": used * (N * K // 2 + scales) + R * (N + K) * 2, "flops": 2 * R * N * K}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, g, scale=1.0, dtype=torch.bfloat16):
    """Normal values in `dtype`, drawn in slices so that the 32-bit ones need no large buffer."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat, step = out.view(-1), 1 << 26
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_(torch.randn(part.numel(), device=DEV, generator=g) * scale)
    return out


def _groups(case, seed):
    """Borders of the groups of `rows` rows over the experts, uneven by `skew`: host list and device tensor."""
    r = np.random.RandomState(seed)
    E = case["experts"]
    p = np.exp(case["skew"] * r.randn(E))
    counts = r.multinomial(case["rows"], p / p.sum())
    bounds = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return int(counts.max()), torch.from_numpy(bounds).to(DEV)


def _positions(ids, E):
    """Row of each (token, choice) in expert order (by expert, then by token), -1 for a choice of -1."""
    flat = torch.where(ids < 0, E, ids).reshape(-1)
    order = torch.argsort(flat, stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(flat.numel(), device=ids.device)
    return torch.where(flat < E, pos, -1).to(torch.int32).reshape(ids.shape)


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    s = {"case": case}
    if op in ("route", "route_grad"):
        T, E, k = case["tokens"], case["experts"], case["k"]
        logits = 2 * torch.randn((T, E), device=DEV, generator=g)
        if case["masked"]:
            logits[torch.rand((T, E), device=DEV, generator=g) < case["masked"]] = float("-inf")  # experts closed to a token
            logits[torch.rand((T,), device=DEV, generator=g) < case["masked"]] = float("-inf")    # padding
        s["logits"] = logits.to(DTYPES[case["type"]])
        if op == "route_grad":
            s["ids"], s["weights"] = _choose(s["logits"], k, case["renorm"])
            s["dweights"] = torch.randn((T, k), device=DEV, generator=g)
        else:  # what a decoding loop keeps from step to step: ids, weights, pos, order, offsets
            shapes = ((T, k), torch.int32), ((T, k), torch.float32), ((T, k), torch.int32), ((T * k,), torch.int32), ((E + 1,), torch.int32)
            s["into"] = [torch.empty(shape, dtype=dt, device=DEV) for shape, dt in shapes]
    elif op in ("gather", "combine", "combine_grad"):
        T, E, k, H, dt = case["tokens"], case["experts"], case["k"], case["width"], DTYPES[case["type"]]
        ids = torch.rand((T, E), device=DEV, generator=g).argsort(dim=1)[:, :k]
        if case["dropped"]:
            ids = torch.where(torch.rand((T, k), device=DEV, generator=g) < case["dropped"], -1, ids)
        s["pos"] = _positions(ids, E)
        if op != "combine":
            s["x"] = _randn((T, H), g, dtype=dt)
        if op != "gather":
            s["y"] = _randn((T * k, H), g, dtype=dt)
            s["weights"] = torch.rand((T, k), device=DEV, generator=g)
        if op != "combine":
            s["rows"] = torch.zeros((T * k, H), dtype=dt, device=DEV)  # rows without a token keep what they hold
    elif op == "grouped":
        R, E, N, K, side = case["rows"], case["experts"], case["n"], case["k"], case["side"]
        s["longest"], s["offsets"] = _groups(case, seed)
        if side != "wgrad":
            s["w"] = _randn((E, N, K), g, 1 / math.sqrt(K if side == "fwd" else N))
            s["out"] = torch.zeros((R + case["spare"], N if side == "fwd" else K), dtype=torch.bfloat16, device=DEV)
        if side != "dgrad":
            s["x"] = _randn((R + case["spare"], K), g)
        if side != "fwd":
            s["dy"] = _randn((R + case["spare"], N), g, 1 / math.sqrt(N) if side == "wgrad" else 1.0)
    else:
        R, E, N, K, G, dt = case["rows"], case["experts"], case["n"], case["k"], case["group"], DTYPES[case["type"]]
        s["longest"], s["offsets"] = _groups(case, seed)
        s["x"] = _randn((R, K), g, dtype=dt)
        s["q"] = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device=DEV, generator=g)  # k even: low half
        s["scales"] = ((0.5 + torch.rand((E, N, K // G), device=DEV, generator=g)) / (4 * math.sqrt(K))).to(dt)
        s["zeros"] = torch.randint(4, 12, (E, N, K // G), dtype=torch.uint8, device=DEV, generator=g) if case["zeros"] else None
        s["out"] = torch.zeros((R, N), dtype=dt, device=DEV)
        if E == 1:  # one matrix: no groups
            s["offsets"], s["q"], s["scales"] = None, s["q"][0], s["scales"][0]
            s["zeros"] = None if s["zeros"] is None else s["zeros"][0]
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------
def _choose(logits, k, renorm):
    """The k largest logits of each token, the lowest expert first among equals, and their softmax weights; a logit of
    -inf is never chosen (id -1, weight 0)."""
    value = logits.float()
    top, ids = torch.sort(value, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    open_ = top > float("-inf")
    largest = torch.where(open_[:, :1], top[:, :1], 0.0)
    e = torch.exp(top - largest)
    total = e.sum(1, keepdim=True) if renorm else torch.exp(value - largest).sum(1, keepdim=True)
    weights = torch.where(open_, e / torch.where(total > 0, total, 1.0), 0.0)
    return torch.where(open_, ids, -1).to(torch.int32), weights


def _plain_route(s, c):
    ids, weights = _choose(s["logits"], c["k"], c["renorm"])
    E, n = c["experts"], ids.numel()
    pos = _positions(ids.long(), E)
    flat = pos.reshape(-1).long()
    order = torch.full((n + 1,), -1, dtype=torch.int32, device=ids.device)
    order[torch.where(flat < 0, n, flat)] = torch.arange(n, dtype=torch.int32, device=ids.device)
    counts = (ids.reshape(1, -1) == torch.arange(E, device=ids.device)[:, None]).sum(1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    filled = torch.where(torch.arange(n, device=ids.device) < offsets[-1], order[:n], -1)
    return {"ids": ids, "weights": weights, "pos": pos, "order": filled, "offsets": offsets}


def _plain_route_grad(s, c):
    """p = softmax (over the chosen or over all); dl = p * (g - sum of g * p over the chosen)."""
    value, ids, w = s["logits"].float(), s["ids"].long(), s["weights"]
    chosen = ids >= 0
    at = torch.where(chosen, ids, 0)
    g = torch.where(chosen, s["dweights"], 0.0)
    dense = torch.zeros_like(value).scatter_add_(1, at, g)
    mean = (g * w).sum(1, keepdim=True)
    if c["renorm"]:
        p = torch.zeros_like(value).scatter_add_(1, at, torch.where(chosen, w, 0.0))
    else:
        largest = value.max(1, keepdim=True).values
        e = torch.exp(value - torch.where(largest > float("-inf"), largest, 0.0))
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
    return (p * (dense - mean)).to(s["logits"].dtype)


def _plain_gather(s, c):
    rows, flat = s["rows"].shape[0], s["pos"].reshape(-1).long()
    out = torch.zeros((rows + 1, c["width"]), dtype=s["x"].dtype, device=s["x"].device)
    out[torch.where(flat < 0, rows, flat)] = s["x"].repeat_interleave(c["k"], dim=0)
    return out[:rows]


def _plain_combine(s, c):
    pos = s["pos"].long()
    y = s["y"].float()[pos.clamp(min=0)]
    return torch.where(pos[..., None] < 0, 0.0, y * s["weights"][..., None]).sum(1).to(s["y"].dtype)


def _plain_combine_grad(s, c):
    pos, dout = s["pos"].long(), s["x"].float()
    rows, flat = s["rows"].shape[0], pos.reshape(-1)
    y = s["y"].float()[pos.clamp(min=0)]
    dw = torch.where(pos < 0, 0.0, (y * dout[:, None, :]).sum(2))
    dy = torch.zeros((rows + 1, c["width"]), device=dout.device)
    dy[torch.where(flat < 0, rows, flat)] = (dout[:, None, :] * s["weights"][..., None]).reshape(-1, c["width"])
    return {"dy": dy[:rows].to(s["y"].dtype), "dweights": dw}


def _padded(rows, s):
    """[E, longest, width] in 32 bits: each group's rows, zeros behind them."""
    first, last = s["offsets"][:-1, None].long(), s["offsets"][1:, None].long()
    at = first + torch.arange(s["longest"], device=rows.device)
    return torch.where((at < last)[..., None], rows.float()[at.clamp(max=rows.shape[0] - 1)], 0.0)


def _unpadded(y, rows, s):
    """The rows of [E, longest, width] in group order, zeros behind the last."""
    at = torch.arange(rows, device=y.device)
    e = torch.searchsorted(s["offsets"][1:].long(), at, right=True).clamp(max=y.shape[0] - 1)
    i = (at - s["offsets"].long()[e]).clamp(max=y.shape[1] - 1)
    return torch.where((at < s["offsets"][-1])[:, None], y[e, i], 0.0)


def _plain_grouped(s, c):
    if c["side"] == "fwd":
        return _unpadded(_padded(s["x"], s) @ s["w"].float().transpose(1, 2), s["x"].shape[0], s).to(torch.bfloat16)
    if c["side"] == "dgrad":
        return _unpadded(_padded(s["dy"], s) @ s["w"].float(), s["dy"].shape[0], s).to(torch.bfloat16)
    return (_padded(s["dy"], s).transpose(1, 2) @ _padded(s["x"], s)).to(DTYPES[c["type"]])


def _plain_gemv_w4(s, c):
    q = torch.stack([s["q"] & 15, s["q"] >> 4], dim=-1).float().flatten(-2)
    q = q.unflatten(-1, (-1, c["group"])) - (8.0 if s["zeros"] is None else s["zeros"].float()[..., None])
    w = (q * s["scales"].float()[..., None]).flatten(-2)
    if s["offsets"] is None:
        return (s["x"].float() @ w.t()).to(s["x"].dtype)
    return _unpadded(_padded(s["x"], s) @ w.transpose(1, 2), s["x"].shape[0], s).to(s["x"].dtype)


PLAIN = {"route": _plain_route, "route_grad": _plain_route_grad, "gather": _plain_gather, "combine": _plain_combine,
         "combine_grad": _plain_combine_grad, "grouped": _plain_grouped, "gemv_w4": _plain_gemv_w4}


# ---- the package's calls ------------------------------------------------------------------------------------------
def _own(s, c):
    import prism_b200 as pb
    op = c["op"]
    if op == "route":
        r = pb.route_topk(s["logits"], c["k"], renormalize=c["renorm"], out=s["into"])
        return {"ids": r.ids, "weights": r.weights, "pos": r.pos, "order": r.order, "offsets": r.offsets}
    if op == "route_grad":
        return pb.route_topk_grad(s["logits"], s["ids"], s["weights"], s["dweights"], renormalize=c["renorm"])
    if op == "gather":
        return pb.route_gather(s["x"], s["pos"], out=s["rows"])
    if op == "combine":
        return pb.route_combine(s["y"], s["pos"], s["weights"])
    if op == "combine_grad":
        dy, dweights = pb.route_combine_grad(s["x"], s["y"], s["pos"], s["weights"], dy=s["rows"])
        return {"dy": dy, "dweights": dweights}
    if op == "gemv_w4":
        return pb.gemv_w4(s["x"], s["q"], s["scales"], zeros=s["zeros"], offsets=s["offsets"], out=s["out"])
    if c["side"] == "fwd":
        return pb.grouped_gemm_bf16(s["x"], s["w"], s["offsets"], out=s["out"])
    if c["side"] == "dgrad":
        return pb.grouped_gemm_bf16_dgrad(s["dy"], s["w"], s["offsets"], out=s["out"])
    return pb.grouped_gemm_bf16_wgrad(s["dy"], s["x"], s["offsets"], dtype=DTYPES[c["type"]])


def run(state):
    c = state["case"]
    return _own(state, c) if own else PLAIN[c["op"]](state, c)


# ---- 64 bits ------------------------------------------------------------------------------------------------------
def _exact_route(s, c):
    """k rounds of taking the largest of what is left, and a count of the rows in front of each, in numpy."""
    l, k, E = s["logits"].double().cpu().numpy(), c["k"], c["experts"]
    T = l.shape[0]
    left, ids = l.copy(), np.full((T, k), -1, np.int32)
    for j in range(k):
        best = left.argmax(1)
        some = left[np.arange(T), best] > -np.inf
        ids[some, j] = best[some]
        left[np.arange(T), best] = -np.inf
    m = np.where(ids[:, :1] >= 0, l.max(1, keepdims=True), 0.0)
    chosen = np.where(ids >= 0, np.exp(np.take_along_axis(l, np.maximum(ids, 0), 1) - m), 0.0)
    total = chosen.sum(1, keepdims=True) if c["renorm"] else np.exp(l - m).sum(1, keepdims=True)
    weights = chosen / np.where(total > 0, total, 1.0)
    member = np.zeros((T, E), np.int64)
    member[np.nonzero(ids >= 0)[0], ids[ids >= 0]] = 1
    offsets = np.concatenate([[0], member.sum(0).cumsum()]).astype(np.int32)
    rank = member.cumsum(0) - member
    pos = np.where(ids >= 0, offsets[np.maximum(ids, 0)] + np.take_along_axis(rank, np.maximum(ids, 0).astype(np.int64), 1), -1)
    order = np.full((T * k,), -1, np.int32)
    order[pos[pos >= 0]] = np.nonzero(pos.reshape(-1) >= 0)[0]
    return {"ids": ids, "weights": weights, "pos": pos.astype(np.int32), "order": order, "offsets": offsets}


def _exact_route_grad(s, c):
    """Row by row of the softmax's Jacobian, the weights computed again from the logits."""
    l, ids, g = s["logits"].double().cpu().numpy(), s["ids"].cpu().numpy(), s["dweights"].double().cpu().numpy()
    T, E = l.shape
    G = np.zeros((T, E))
    chosen = np.zeros((T, E), bool)
    t, j = np.nonzero(ids >= 0)
    G[t, ids[t, j]], chosen[t, ids[t, j]] = g[t, j], True
    support = chosen if c["renorm"] else l > -np.inf
    m = np.max(np.where(support, l, -np.inf), axis=1, keepdims=True)
    p = np.where(support, np.exp(np.where(support, l, 0.0) - np.where(m > -np.inf, m, 0.0)), 0.0)
    p /= np.maximum(p.sum(1, keepdims=True), np.finfo(float).tiny)
    return p * G - p * (p * G).sum(1, keepdims=True)


def _exact_rows(s, c):
    T, k, pos = c["tokens"], c["k"], s["pos"].long()
    token = torch.arange(T, device=DEV)[:, None].expand(T, k)[pos >= 0]
    row = pos[pos >= 0]
    if c["op"] == "gather":
        out = torch.zeros(s["rows"].shape, dtype=torch.float64, device=DEV)
        out[row] = s["x"].double()[token]
        return out
    w = s["weights"].double()[pos >= 0]
    if c["op"] == "combine":
        out = torch.zeros((T, c["width"]), dtype=torch.float64, device=DEV)
        for j in range(k):
            live = pos[:, j] >= 0
            out[live] += s["weights"][live, j].double()[:, None] * s["y"][pos[live, j]].double()
        return out
    dy = torch.zeros(s["rows"].shape, dtype=torch.float64, device=DEV)
    dy[row] = w[:, None] * s["x"][token].double()
    dw = torch.zeros((T, k), dtype=torch.float64, device=DEV)
    for j in range(k):
        live = pos[:, j] >= 0
        dw[live, j] = torch.linalg.vecdot(s["x"][live].double(), s["y"][pos[live, j]].double())
    return {"dy": dy, "dweights": dw}


def _exact_grouped(s, c):
    bounds = s["offsets"].tolist()
    groups = list(enumerate(zip(bounds[:-1], bounds[1:])))
    if c["side"] == "wgrad":
        out = torch.zeros((c["experts"], c["n"], c["k"]), dtype=torch.float64, device=DEV)
        for e, (a, b) in groups:
            out[e] = torch.einsum("rn,rk->nk", s["dy"][a:b].double(), s["x"][a:b].double())
        return out
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for e, (a, b) in groups:
        if c["side"] == "fwd":
            out[a:b] = torch.einsum("rk,nk->rn", s["x"][a:b].double(), s["w"][e].double())
        else:
            out[a:b] = torch.einsum("rn,nk->rk", s["dy"][a:b].double(), s["w"][e].double())
    return out


def _exact_gemv_w4(s, c):
    N, K, G = c["n"], c["k"], c["group"]
    bounds = [0, c["rows"]] if s["offsets"] is None else s["offsets"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    for e, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        if a == b:
            continue
        q, scale = s["q"].reshape(-1, N, K // 2)[e], s["scales"].reshape(-1, N, K // G)[e].double()
        zero = torch.full_like(scale, 8.0) if s["zeros"] is None else s["zeros"].reshape(-1, N, K // G)[e].double()
        w = torch.empty((N, K), dtype=torch.float64, device=DEV)
        w[:, 0::2], w[:, 1::2] = (q % 16).double(), torch.div(q, 16, rounding_mode="floor").double()
        w = (w - zero.repeat_interleave(G, 1)) * scale.repeat_interleave(G, 1)
        out[a:b] = torch.einsum("rk,nk->rn", s["x"][a:b].double(), w)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s, case)
    if case["op"] == "route_grad":
        return _exact_route_grad(s, case)
    if case["op"] == "grouped":
        return _exact_grouped(s, case)
    return _exact_gemv_w4(s, case) if case["op"] == "gemv_w4" else _exact_rows(s, case)
