"""Performance cases of the operators that stand beside the attention in a layer: what the rows of a batch are multiplied with
depends on the row.

  route     router logits of every row -> the experts that it goes to and their weights (`hy3_b200.route`)
  experts   each row through its experts' gated feed-forward networks, summed by those weights (`hy3_b200.experts`)
  adapters  each row's low-rank adapter added to what a shared projection gave it (`hy3_b200.adapters`)

Where `own` is false, the operators run in their plain form: elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of one conversation at the router: 192 experts, top 8, sigmoid scores with a bias for balance; latency only
        {"name": "route_1x192", "op": "route", "rows": 1, "experts": 192, "top_k": 8, "score": "sigmoid", "bias": True, "groups": 1, "top_groups": 1, "dtype": "fp32", "closed": 0.0},
        # the largest chunk that the backend takes, through the same router; 2 % of the experts closed for a row
        {"name": "route_2048x192", "op": "route", "rows": 2048, "experts": 192, "top_k": 8, "score": "sigmoid", "bias": True, "groups": 1, "top_groups": 1, "dtype": "fp32", "closed": 0.02},
        # a long prompt's rows, softmax over 256 experts in 8 groups of which a row may use 4, 16-bit logits
        {"name": "route_16384x256_groups", "op": "route", "rows": 16384, "experts": 256, "top_k": 8, "score": "softmax", "bias": False, "groups": 8, "top_groups": 4, "dtype": "bf16", "closed": 0.0},
        # one token of one conversation through a whole layer of 192 experts: 8 of them are read
        {"name": "experts_1_of_192", "op": "experts", "rows": 1, "experts": 192, "first": 0, "held": 192, "top_k": 8, "hidden": 4096, "inter": 1536, "dtype": "bf16", "closed": 0.0},
        # a small server: 8 conversations
        {"name": "experts_8_of_192", "op": "experts", "rows": 8, "experts": 192, "first": 0, "held": 192, "top_k": 8, "hidden": 4096, "inter": 1536, "dtype": "bf16", "closed": 0.0},
        # batched serving: 64 sequences, a token each
        {"name": "experts_64_of_192", "op": "experts", "rows": 64, "experts": 192, "first": 0, "held": 192, "top_k": 8, "hidden": 4096, "inter": 1536, "dtype": "bf16", "closed": 0.0},
        # the largest chunk that the backend takes
        {"name": "experts_2048_of_192", "op": "experts", "rows": 2048, "experts": 192, "first": 0, "held": 192, "top_k": 8, "hidden": 4096, "inter": 1536, "dtype": "bf16", "closed": 0.0},
        # one of 8 GPUs that split the experts: 24 of 192 are held, and the rows of all 8 (1024 each) come by
        {"name": "experts_8192_24_held", "op": "experts", "rows": 8192, "experts": 192, "first": 72, "held": 24, "top_k": 8, "hidden": 4096, "inter": 1536, "dtype": "bf16", "closed": 0.0},
        # odd sizes: a small model's 10 experts, fp16, some slots without an expert
        {"name": "experts_333_fp16_odd", "op": "experts", "rows": 333, "experts": 10, "first": 0, "held": 10, "top_k": 3, "hidden": 1032, "inter": 200, "dtype": "fp16", "closed": 0.03},
        # one conversation with an adapter on the query, key and value projection (4096 -> 64 + 8 + 8 heads of 128)
        {"name": "adapters_1_qkv", "op": "adapters", "rows": 1, "requests": 1, "adapters": 8, "rank": 16, "width": 4096, "out": 10240, "dtype": "bf16", "base": "fp32", "without": 0.0},
        # 64 conversations, up to 40 adapters among them, on the output projection (64 heads of 128 -> 4096)
        {"name": "adapters_64_o", "op": "adapters", "rows": 64, "requests": 64, "adapters": 40, "rank": 64, "width": 8192, "out": 4096, "dtype": "bf16", "base": "bf16", "without": 0.2},
        # chunks of 7 prompts of different lengths, each with its adapter, on the query, key and value projection
        {"name": "adapters_2048_qkv", "op": "adapters", "rows": 2048, "requests": 7, "adapters": 16, "rank": 32, "width": 4096, "out": 10240, "dtype": "bf16", "base": "fp32", "without": 0.15},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, step * int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step))))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "adapters"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "route":
        groups = rng.choice([1, 1, 1, 2, 4, 8])
        experts = _log_int(rng, 8 * groups, 512, groups)
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(12, experts // groups * top_groups))
        return {"op": "route", "rows": _log_int(rng, 1, 32768), "experts": experts, "top_k": top_k, "score": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "closed": rng.choice([0.0, 0.0, 0.1])}
    if kind == "experts":
        experts = _log_int(rng, 4, 192)
        held = rng.choice([experts, experts, max(1, experts // 4)])
        case = {"op": "experts", "rows": _log_int(rng, 1, 8192), "experts": experts, "first": rng.randint(0, experts - held), "held": held,
                "top_k": rng.randint(1, min(8, experts)), "hidden": _log_int(rng, 256, 5120, 8), "inter": _log_int(rng, 64, 2560, 8), "dtype": dtype,
                "closed": rng.choice([0.0, 0.0, 0.05])}
        # no more weights than the largest listed layer's, no more operations than its largest chunk's
        while case["held"] * case["hidden"] * case["inter"] > 192 * 4096 * 1536:
            case["inter"] = max(64, case["inter"] // 16 * 8)
        while case["rows"] * case["top_k"] * case["hidden"] * case["inter"] * 6.0 > 6e14:
            case["rows"] //= 2
        return case
    rows = _log_int(rng, 1, 4096)
    return {"op": "adapters", "rows": rows, "requests": rng.choice([rows, min(rows, _log_int(rng, 1, 64))]), "adapters": _log_int(rng, 1, 64),
            "rank": _log_int(rng, 8, 128, 8), "width": _log_int(rng, 256, 8192, 8), "out": _log_int(rng, 256, 10240, 8), "dtype": dtype,
            "base": rng.choice(["fp32", dtype]), "without": rng.choice([0.0, 0.2])}


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(shape, gen, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=gen).mul_(scale)


def _uniform(shape, gen):
    return torch.rand(shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen, rows = _generator(seed), case["rows"]
    s = {"case": case}
    if case["op"] == "route":
        # logits of a trained router: a few experts of a row stand out; the bias evens the load out
        logits = _normal((rows, case["experts"]), gen, scale=1.5)
        if case["closed"]:
            logits[_uniform(logits.shape, gen) < case["closed"]] = -math.inf
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        s["bias"] = _normal((case["experts"],), gen, scale=0.05) if case["bias"] else None
        return s
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "experts":
        held, hidden, inter, k = case["held"], case["hidden"], case["inter"], case["top_k"]
        # normalised rows; some experts are asked more often than others; weights as the router gives them
        s["x"] = _normal((rows, hidden), gen, dtype)
        liked = _normal((rows, case["experts"]), gen) + _normal((case["experts"],), gen, scale=0.3)
        best = torch.topk(liked, k, dim=-1)
        ids = best.indices.to(torch.int32)
        if case["closed"]:
            ids[_uniform(ids.shape, gen) < case["closed"]] = -1
        score = 1 / (1 + torch.exp(-best.values))
        s["ids"], s["weights"] = ids, score / score.sum(-1, keepdim=True) * 2.826
        s["gate"] = _normal((held, inter, hidden), gen, dtype, hidden ** -0.5)
        s["up"] = _normal((held, inter, hidden), gen, dtype, hidden ** -0.5)
        s["down"] = _normal((held, hidden, inter), gen, dtype, inter ** -0.5)
        return s
    n, rank, width, out = case["adapters"], case["rank"], case["width"], case["out"]
    # each request has one adapter or none; its rows lie together (a decode batch: one row each)
    which = torch.randint(0, n, (case["requests"],), device="cuda", generator=gen)
    which[_uniform(which.shape, gen) < case["without"]] = -1
    ends = torch.sort(torch.randint(0, rows, (case["requests"] - 1,), device="cuda", generator=gen)).values
    owner = torch.arange(rows, device="cuda") if case["requests"] == rows else torch.searchsorted(ends, torch.arange(rows, device="cuda"), right=True)
    s["ids"] = which[owner].to(torch.int32)
    s["x"] = _normal((rows, width), gen, dtype)
    s["base"] = _normal((rows, out), gen).to(DTYPES[case["base"]])
    s["a"] = _normal((n, rank, width), gen, dtype, width ** -0.5)
    s["b"] = _normal((n, out, rank), gen, dtype, 0.3 * rank ** -0.5)
    s["scales"] = 0.5 + _uniform((n,), gen)
    return s


def _plain_route(s):
    case, lowest = s["case"], torch.finfo(torch.float32).min
    logits = s["logits"].float()
    if case["score"] == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = e / e.double().sum(-1, keepdim=True).float()
    else:
        score = 1 / (1 + torch.exp(-logits))
    pick = score if s["bias"] is None else score + s["bias"]
    pick = torch.where(torch.isnan(pick), lowest, pick)
    pick = torch.where(logits == -math.inf, -math.inf, pick)
    groups, size = case["groups"], case["experts"] // case["groups"]
    if groups > 1:
        # a group stands with the sum of its two best
        best = pick.view(-1, groups, size).topk(min(2, size), dim=-1).values
        second = best[..., -1] if size > 1 else torch.full_like(best[..., 0], -math.inf)
        stands = best[..., 0] + torch.where(second == -math.inf, 0.0, second)
        kept = torch.sort(stands, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = torch.zeros_like(stands, dtype=torch.bool).scatter_(1, kept, True)
        pick = torch.where(open_.repeat_interleave(size, dim=1), pick, -math.inf)
    top = torch.sort(pick, dim=-1, descending=True, stable=True)
    ids, none = top.indices[:, :case["top_k"]], top.values[:, :case["top_k"]] == -math.inf
    weights = torch.where(none, 0.0, score.gather(1, ids))
    weights = weights / (weights.sum(-1, keepdim=True) + 1e-20)
    return torch.where(none, -1, ids).to(torch.int32), weights * 2.826


def _gated(rows, gate, up, down):
    """rows [e, n, hidden] through the networks of e experts."""
    g, u = torch.bmm(rows, gate.float().transpose(1, 2)), torch.bmm(rows, up.float().transpose(1, 2))
    return torch.bmm(g / (1 + torch.exp(-g)) * u, down.float().transpose(1, 2))


def _plain_experts(s):
    x, case = s["x"].float(), s["case"]
    rows, k, held = case["rows"], case["top_k"], case["held"]
    slot = s["ids"].reshape(-1).long() - case["first"]
    none = (slot < 0) | (slot >= held) | (s["ids"].reshape(-1) < 0)
    token = torch.arange(rows * k, device=x.device) // k
    if rows * k <= held:
        # fewer slots than experts: each slot takes its expert's weights
        e = torch.where(none, 0, slot)
        y = _gated(x[token].unsqueeze(1), s["gate"][e], s["up"][e], s["down"][e]).squeeze(1)
    else:
        # every expert takes its slots, padded to the fullest
        e = torch.where(none, held, slot)
        order = torch.argsort(e, stable=True)
        count = torch.zeros(held + 1, dtype=torch.long, device=x.device).scatter_add_(0, e, torch.ones_like(e))
        place = torch.empty_like(order).scatter_(0, order, torch.arange(rows * k, device=x.device) - (count.cumsum(0) - count)[e[order]])
        most = max(1, int(count[:held].max()))
        place = torch.where(none, held * most, e * most + place)
        padded = torch.zeros((held * most + 1, case["hidden"]), device=x.device)
        padded[place] = x[token]
        y = _gated(padded[:-1].view(held, most, -1), s["gate"], s["up"], s["down"]).view(held * most, -1)[place.clamp(max=held * most - 1)]
    y = torch.where(none.unsqueeze(1), 0.0, y * s["weights"].reshape(-1, 1))
    return y.view(rows, k, -1).sum(1).to(s["x"].dtype)


def _plain_adapters(s):
    n, rank, width = s["a"].shape
    u = (s["x"].float() @ s["a"].float().view(n * rank, width).T).view(-1, n, rank) * s["scales"].view(1, n, 1)
    mine = s["ids"].view(-1, 1) == torch.arange(n, device=u.device, dtype=torch.int32)
    u = torch.where(mine.unsqueeze(2), u, 0.0).view(-1, n * rank)
    return (s["base"].float() + u @ s["b"].float().transpose(1, 2).reshape(n * rank, -1)).to(s["base"].dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        import hy3_b200
        if case["op"] == "route":
            return hy3_b200.route(s["logits"], s["bias"], top_k=case["top_k"], score=case["score"], groups=case["groups"],
                                  top_groups=case["top_groups"], renormalize=True, scale=2.826)
        if case["op"] == "experts":
            return hy3_b200.experts(s["x"], s["ids"], s["weights"], s["gate"], s["up"], s["down"], first_expert=case["first"])
        return hy3_b200.adapters(s["x"], s["base"], s["a"], s["b"], s["ids"], s["scales"])
    return {"route": _plain_route, "experts": _plain_experts, "adapters": _plain_adapters}[case["op"]](s)


def _some(n, p):
    """How many of n things at least one of draws finds that each find one with probability p."""
    return n * (1 - (1 - p[0] / n) ** p[1])


def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": float(rows * case["experts"] * size + (4 * case["experts"] if case["bias"] else 0) + rows * case["top_k"] * 8),
                "flops": float(rows * case["experts"] * 4)}
    if case["op"] == "experts":
        hidden, inter, k = case["hidden"], case["inter"], case["top_k"]
        slots = rows * k * (1 - case["closed"]) * case["held"] / case["experts"]
        # the experts that some row asks for (as many as an even choice finds), the rows in and out, the slots
        used = _some(case["held"], (k * (1 - case["closed"]) * case["held"] / case["experts"], rows))
        return {"bytes": used * 3.0 * hidden * inter * 2 + rows * hidden * 4.0 + rows * k * 8.0, "flops": slots * 6.0 * hidden * inter}
    width, out, rank = case["width"], case["out"], case["rank"]
    used = _some(case["adapters"], (1 - case["without"], case["requests"]))
    with_one = rows * (1 - case["without"])
    return {"bytes": used * (width + out) * rank * 2.0 + with_one * width * 2.0 + rows * out * 2.0 * (4 if case["base"] == "fp32" else 2) + rows * 4.0,
            "flops": with_one * 2.0 * rank * (width + out)}


def _exact_route(s, case):
    logits = s["logits"].double()
    score = torch.softmax(logits, -1) if case["score"] == "softmax" else torch.sigmoid(logits)
    pick = score.clone()
    if s["bias"] is not None:
        pick += s["bias"].double()
    pick[logits == -math.inf] = -math.inf
    if case["groups"] > 1:
        size = case["experts"] // case["groups"]
        stands = torch.stack([torch.where(p[:, :2] == -math.inf, 0.0, p[:, :2]).sum(-1) + torch.where(p[:, 0] == -math.inf, -math.inf, 0.0)
                              for p in (q.sort(dim=-1, descending=True).values for q in pick.split(size, dim=1))], dim=1)
        for g in range(case["groups"]):
            # a group is out if as many others as may stay are better, or as good and before it
            better = (stands > stands[:, g:g + 1]).sum(1) + (stands[:, :g] == stands[:, g:g + 1]).sum(1)
            pick[better >= case["top_groups"], g * size:(g + 1) * size] = -math.inf
    top = torch.sort(pick, dim=-1, descending=True, stable=True)
    weights = score.gather(1, top.indices[:, :case["top_k"]])
    weights[top.values[:, :case["top_k"]] == -math.inf] = 0
    # which experts are chosen is a matter of the scores in 32 bits: no value here
    return None, 2.826 * weights / (weights.sum(-1, keepdim=True) + 1e-20)


def _exact_experts(s, case):
    y = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
    for e in range(case["held"]):
        row, j = torch.nonzero(s["ids"] == case["first"] + e, as_tuple=True)
        if len(row):
            x = s["x"][row].double()
            h = torch.nn.functional.silu(x @ s["gate"][e].double().T) * (x @ s["up"][e].double().T)
            y.index_add_(0, row, s["weights"][row, j].double().unsqueeze(1) * (h @ s["down"][e].double().T))
    return y


def _exact_adapters(s, case):
    y = s["base"].double()
    for i in range(case["adapters"]):
        row = torch.nonzero(s["ids"] == i).squeeze(1)
        y[row] += float(s["scales"][i]) * ((s["x"][row].double() @ s["a"][i].double().T) @ s["b"][i].double().T)
    return y


def exact(case, seed):
    if work(case)["flops"] > 7e14:
        return None
    return {"route": _exact_route, "experts": _exact_experts, "adapters": _exact_adapters}[case["op"]](prepare(case, seed), case)
