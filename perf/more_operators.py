"""Performance cases of weights in 4 bits and of what is asked of the logits that they give.

  quantize4  a weight matrix -> 4-bit codes and a scale for each group of neighbours in a row (`hy3_b200.quantize4`)
  linear4    rows through such a matrix: a projection, or the output head (`hy3_b200.linear4`)
  logprobs   rows of logits -> log probabilities of given tokens, entropy, the best alternatives (`hy3_b200.logprobs`)

Where `own` is false, the operators run in their plain form: elementary torch operations in 32 bits (sums of exponentials in 64).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # loading a checkpoint: the output head (120832 tokens), the largest matrix of the model
        {"name": "quantize4_head", "op": "quantize4", "out": 120832, "width": 4096, "group": 64, "from": "bf16", "dtype": "bf16"},
        # an odd matrix of a small model from fp32, its last group not full
        {"name": "quantize4_odd", "op": "quantize4", "out": 1001, "width": 1056, "group": 128, "from": "fp32", "dtype": "fp16"},
        # one token of one conversation, the query, key and value projection; the attention takes fp32 rows
        {"name": "linear4_1_qkv", "op": "linear4", "rows": 1, "width": 4096, "out": 10240, "group": 64, "dtype": "bf16", "result": "fp32"},
        # the same token at the output head, fp32 logits
        {"name": "linear4_1_head", "op": "linear4", "rows": 1, "width": 4096, "out": 120832, "group": 64, "dtype": "bf16", "result": "fp32"},
        # a small server: 8 conversations, the output projection of the attention
        {"name": "linear4_8_o", "op": "linear4", "rows": 8, "width": 8192, "out": 4096, "group": 128, "dtype": "bf16", "result": "bf16"},
        # batched serving: 64 sequences, a token each
        {"name": "linear4_64_qkv", "op": "linear4", "rows": 64, "width": 4096, "out": 10240, "group": 64, "dtype": "bf16", "result": "fp32"},
        # the largest chunk of a prompt that the backend takes, the output projection of the attention
        {"name": "linear4_2048_o", "op": "linear4", "rows": 2048, "width": 8192, "out": 4096, "group": 128, "dtype": "bf16", "result": "bf16"},
        # odd sizes: a small model in fp16, short groups
        {"name": "linear4_333_odd", "op": "linear4", "rows": 333, "width": 1056, "out": 1001, "group": 32, "dtype": "fp16", "result": "fp16"},
        # one streamed token with 20 alternatives
        {"name": "logprobs_1_top20", "op": "logprobs", "rows": 1, "vocab": 120832, "asked": 1, "top_k": 20, "dtype": "fp32", "closed": 0.0, "padded": 0.0},
        # batched serving with 5 alternatives, 4 drafted tokens asked for, 16-bit logits, most tokens closed by a grammar
        {"name": "logprobs_64_top5", "op": "logprobs", "rows": 64, "vocab": 120832, "asked": 4, "top_k": 5, "dtype": "bf16", "closed": 0.9, "padded": 0.0},
        # a prompt's log likelihood: a chunk of 2048 tokens, some of them padding
        {"name": "logprobs_2048", "op": "logprobs", "rows": 2048, "vocab": 120832, "asked": 1, "top_k": 0, "dtype": "fp32", "closed": 0.0, "padded": 0.05},
        # a small vocabulary of an odd size, so that rows start anywhere
        {"name": "logprobs_333_odd", "op": "logprobs", "rows": 333, "vocab": 32003, "asked": 1, "top_k": 1, "dtype": "fp16", "closed": 0.0, "padded": 0.0},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, step * int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step))))


def draw(rng):
    kind = rng.choice(["quantize4", "linear4", "linear4", "linear4", "logprobs", "logprobs"])
    dtype, group = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([32, 64, 128])
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 160000)
        # no more logits than the largest listed case's
        rows = _log_int(rng, 1, min(8192, 2048 * 120832 // vocab))
        return {"op": kind, "rows": rows, "vocab": vocab, "asked": rng.choice([1, 1, 4]), "top_k": rng.choice([0, 1, 5, 20, 32]),
                "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "closed": rng.choice([0.0, 0.0, 0.9]), "padded": rng.choice([0.0, 0.1])}
    width, out = _log_int(rng, 256, 16384, 32), _log_int(rng, 64, 131072)
    # no larger a matrix than the output head
    out = min(out, 120832 * 4096 // width)
    if kind == "quantize4":
        return {"op": kind, "out": out, "width": width, "group": group, "from": rng.choice([dtype, dtype, "fp32"]), "dtype": dtype}
    # no more operations than the largest listed chunk's
    rows = _log_int(rng, 1, min(4096, max(1, 2048 * 8192 * 4096 // (width * out))))
    return {"op": kind, "rows": rows, "width": width, "out": out, "group": group, "dtype": dtype, "result": rng.choice([dtype, dtype, "fp32"])}


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(shape, gen, dtype=torch.float32, scale=1.0):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=gen).mul_(scale)


def _uniform(shape, gen):
    return torch.rand(shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = _generator(seed)
    s = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a trained head: many unlikely tokens, one that stands out in most rows
        logits = _normal((rows, vocab), gen, scale=2.5)
        likely = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
        logits.scatter_add_(1, likely, 14 * _uniform((rows, 1), gen))
        tokens = torch.randint(0, vocab, (rows, case["asked"]), device="cuda", generator=gen)
        tokens[:, :1] = torch.where(_uniform((rows, 1), gen) < 0.5, likely, tokens[:, :1])
        if case["closed"]:
            shut = _uniform(logits.shape, gen) < case["closed"]
            shut.scatter_(1, likely, False)
            logits[shut] = -math.inf
        if case["padded"]:
            tokens[_uniform((rows,), gen) < case["padded"]] = -1
        s["logits"], s["tokens"] = logits.to(DTYPES[case["dtype"]]), tokens.to(torch.int32)
        return s
    out, width, dtype = case["out"], case["width"], DTYPES[case["dtype"]]
    groups = -(-width // case["group"])
    if case["op"] == "quantize4":
        # weights of a trained layer: each row on a scale of its own
        s["w"] = (_normal((out, width), gen, scale=width ** -0.5) * (0.5 + _uniform((out, 1), gen))).to(DTYPES[case["from"]])
        return s
    # rows behind a norm; codes as normal weights have them, a scale for each group
    s["x"] = _normal((case["rows"], width), gen, dtype)
    codes = _normal((out, width), gen, torch.float16, 2.9).round_().clamp_(-8, 7).add_(8).to(torch.uint8).view(out, width // 2, 2)
    s["codes"] = codes[..., 0] | codes[..., 1] << 4
    s["scales"] = ((0.5 + _uniform((out, groups), gen)) * (width ** -0.5 / 2.9)).to(dtype)
    return s


def _plain_quantize4(s):
    case = s["case"]
    out, width, group = case["out"], case["width"], case["group"]
    groups = -(-width // group)
    w = torch.nn.functional.pad(s["w"], (0, groups * group - width)).float().view(out, groups, group)
    lowest, highest = w.amin(-1), w.amax(-1)
    # the value of the largest magnitude becomes the code 0, -8 steps; the scale has its sign turned
    scales = (torch.where(highest > -lowest, highest, lowest) / -8).to(DTYPES[case["dtype"]])
    steps = w / scales.float().unsqueeze(-1)
    steps = torch.where(torch.isfinite(steps) & torch.isfinite(scales).unsqueeze(-1), steps, 0.0)
    codes = (torch.round(steps).clamp_(-8, 7) + 8).to(torch.uint8).view(out, groups * group)[:, :width].reshape(out, width // 2, 2)
    return codes[..., 0] | codes[..., 1] << 4, scales


def _weights(codes, scales, group, dtype):
    """The matrix that codes and scales stand for."""
    steps = torch.stack([codes & 15, codes >> 4], dim=-1).view(codes.shape[0], -1).to(dtype) - 8
    return steps * scales.to(dtype).repeat_interleave(group, dim=1)[:, :steps.shape[1]]


def _plain_linear4(s):
    w = _weights(s["codes"], s["scales"], s["case"]["group"], torch.float32)
    return (s["x"].float() @ w.T).to(DTYPES[s["case"]["result"]])


def _plain_logprobs(s):
    case = s["case"]
    logits, tokens, vocab = s["logits"].float() + 0.0, s["tokens"].long(), case["vocab"]
    below = logits - logits.amax(-1, keepdim=True)
    e = torch.exp(below)
    total = e.double().sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e > 0, below * e, 0.0).double().sum(-1, keepdim=True) / total).float().squeeze(1)
    asked = (below.gather(1, tokens.clamp(min=0)).double() - log_total).float()
    asked = torch.where(tokens < 0, 0.0, asked)
    if case["top_k"] == 0:
        return asked, entropy, torch.empty((case["rows"], 0), dtype=torch.int32, device=e.device), torch.empty((case["rows"], 0), device=e.device)
    # larger logits first, of equal ones the lower index: keys of 32 bits of order and 32 of the index turned round
    bits = logits.view(torch.int32).long()
    key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits) * 2 ** 32 + (vocab - torch.arange(vocab, device=e.device))
    ids = torch.topk(key, case["top_k"], dim=-1).indices
    best = (below.gather(1, ids).double() - log_total).float()
    return asked, entropy, torch.where(best == -math.inf, -1, ids).to(torch.int32), best


def run(state):
    s, case = state, state["case"]
    if own:
        import hy3_b200
        if case["op"] == "quantize4":
            return hy3_b200.quantize4(s["w"], group=case["group"], dtype=DTYPES[case["dtype"]])
        if case["op"] == "linear4":
            return hy3_b200.linear4(s["x"], s["codes"], s["scales"], out_dtype=DTYPES[case["result"]])
        return hy3_b200.logprobs(s["logits"], s["tokens"], top_k=case["top_k"])
    return {"quantize4": _plain_quantize4, "linear4": _plain_linear4, "logprobs": _plain_logprobs}[case["op"]](s)


def work(case):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # an exponential, a sum and a weighted sum of every logit
        return {"bytes": float(rows * vocab * (4 if case["dtype"] == "fp32" else 2) + rows * (8 * case["asked"] + 4 + 8 * case["top_k"])), "flops": rows * vocab * 5.0}
    out, width = case["out"], case["width"]
    packed = out * width / 2 + out * -(-width // case["group"]) * 2
    if case["op"] == "quantize4":
        return {"bytes": out * width * (4.0 if case["from"] == "fp32" else 2.0) + packed, "flops": out * width * 4.0}
    rows = case["rows"]
    return {"bytes": packed + rows * width * 2.0 + rows * out * (4.0 if case["result"] == "fp32" else 2.0), "flops": 2.0 * rows * out * width}


def _exact_quantize4(s, case):
    # the scales before their rounding; codes are counted in steps of the rounded ones: no value here
    parts = [part.double() for part in s["w"].split(case["group"], dim=1)]
    far = [torch.where(p.max(1).values > -p.min(1).values, p.max(1).values, p.min(1).values) for p in parts]
    return None, torch.stack(far, dim=1) / -8


def _exact_linear4(s, case):
    x, step = s["x"].double(), max(1, (1 << 26) // case["width"])
    y = torch.empty((case["rows"], case["out"]), dtype=torch.float64, device="cuda")
    for o in range(0, case["out"], step):
        byte = s["codes"][o:o + step].int()
        w = torch.empty((byte.shape[0], case["width"]), dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = byte % 16 - 8, byte // 16 - 8
        for g, scale in enumerate(s["scales"][o:o + step].double().unbind(1)):
            w[:, g * case["group"]:(g + 1) * case["group"]] *= scale.unsqueeze(1)
        y[:, o:o + step] = x @ w.T
    return y


def _exact_logprobs(s, case):
    asked, entropy, best = [], [], []
    for logits, tokens in zip(s["logits"].split(64), s["tokens"].long().split(64)):
        logp = torch.log_softmax(logits.double(), -1)
        asked.append(torch.where(tokens < 0, 0.0, logp.gather(1, tokens.clamp(min=0))))
        entropy.append(-torch.where(logp == -math.inf, 0.0, logp.exp() * logp).sum(-1))
        best.append(logp.topk(case["top_k"], dim=-1).values)
    # which of equal logits come first is a matter of their indices: no value here
    return torch.cat(asked), torch.cat(entropy), None, torch.cat(best)


def exact(case, seed):
    return {"quantize4": _exact_quantize4, "linear4": _exact_linear4, "logprobs": _exact_logprobs}[case["op"]](prepare(case, seed), case)
