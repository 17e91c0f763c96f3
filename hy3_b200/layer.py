"""The operators beside the attention in a layer, on torch CUDA tensors: routing to experts, the experts' products, and low-rank adapters.

They are functions, without a context: work is enqueued on torch's current stream of the tensors' device, outputs and workspaces come
from torch's allocator, nothing is copied to the host or kept between calls, and calls can be captured in a graph.  Sizes and pointers
that the library refuses raise `Hy3AttnError`, tensors of another kind than stated `AssertionError`, and so do tensors that require gradients,
outside of torch.no_grad(): there is no backward pass.  include/hy3_attn.h has the semantics in full.
"""
from ._lib import Hy3AttnError, load_library, load_native

SCORES = {"sigmoid": 0, "softmax": 1}

_raw_stream = None


def _stream(t):
    """The current stream of t's device, as an integer (a tensor elsewhere is refused behind this)."""
    global _raw_stream
    if not t.is_cuda:
        return 0
    if _raw_stream is None:
        import torch
        _raw_stream = torch._C._cuda_getCurrentRawStream
    return _raw_stream(t.device.index)


def _out(r):
    if type(r) is int:
        raise Hy3AttnError(r, load_library().hy3a_last_error(None).decode())
    return r


def route(logits, bias=None, top_k=8, score="sigmoid", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """Routes rows to experts: logits [rows, experts] fp32 / fp16 / bf16 (row stride free), bias fp32 [experts] or None -> (ids int32
    [rows, top_k], weights fp32 [rows, top_k]).

    Scores s = sigmoid or softmax of the logits; s + bias picks, s weighs.  A logit of -inf closes its expert for the row; with groups > 1
    only the experts of the best `top_groups` groups of neighbours stay open (a group stands with the sum of its two best, whatever the score).  The `top_k`
    best in descending order, ties to the lowest index; -1 with weight 0 where none is left.  Weights are divided by their sum if
    `renormalize`, times `scale`."""
    return _out(load_native().route(_stream(logits), logits, bias, top_k, SCORES[score], groups, top_groups, renormalize, scale))


def experts(x, ids, weights, gate, up, down, first_expert=0, out=None):
    """Rows through their experts' gated feed-forward networks: out[t] = sum_j weights[t, j] * down_e (silu(gate_e x[t]) * (up_e x[t])),
    e = ids[t, j] - first_expert.

    x [rows, hidden] fp16 or bf16 (row stride free), ids int32 and weights fp32 [rows, top_k] (as `route` gives them), gate and up
    [held, inter, hidden], down [held, hidden, inter] of x's type, dense.  Sums are fp32; between the two products the gated ones are rounded to
    x's type (fp16: on a scale of each slot; fewer than 32 slots in all keep twice the bits).  Slots of experts that are not held here are left out: ranks that
    split the experts add their outputs up.  Returns out [rows, hidden] of x's type."""
    return _out(load_native().experts(_stream(x), x, ids, weights, gate, up, down, first_expert, out))


def adapters(x, base, a, b, ids, scales, out=None):
    """Each row's low-rank adapter added to what a shared projection gave it: out[t] = base[t] + scales[i] * b_i (a_i x[t]), i = ids[t].

    x [rows, width], a [adapters, rank, width], b [adapters, out_width, rank] fp16 or bf16, base [rows, out_width] of the same type or
    fp32 (row strides of x, base and out free), ids int32 [rows] (-1: none), scales fp32 [adapters].  Returns out (may be base), of base's type."""
    return _out(load_native().adapters(_stream(x), x, base, a, b, ids, scales, out))


def layer_sync(device=None):
    """Waits for torch's current stream on `device` (default: the current one), and raises `Hy3AttnError` if a bounded device-side wait of
    `experts` or `adapters` ran out there since the last call."""
    import torch
    with torch.cuda.device(device):
        rc = load_library().hy3a_layer_sync(torch.cuda.current_stream().cuda_stream)
    if rc:
        _out(rc)
