"""The operators beside the attention, on torch CUDA tensors: routing to experts, the experts' products, and low-rank adapters; weights in 4 bits and
rows' products with them; log probabilities of logits.

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


def quantize4(w, group=64, dtype=None):
    """Weights in 4 bits: w [out_width, width] fp32 / fp16 / bf16 (row stride free) -> (codes uint8 [out_width, width / 2], scales [out_width, groups]).

    Each `group` (32, 64 or 128) neighbours of a row share a scale s of type `dtype` (fp16 or bf16; default: w's, bf16 for fp32), a weight is (q - 8) * s, and a
    byte has the codes q of two neighbours, the first in its low half.  The value of the largest magnitude gets q = 0, 8 steps from 0: s is minus an eighth of it.
    width is a multiple of 32 (the last group may be short).  A group with a NaN or an infinity has a scale that is not finite."""
    return _out(load_native().quantize4(_stream(w), w, group, dtype))


def linear4(x, codes, scales, out_dtype=None, out=None):
    """Rows times a matrix in 4 bits: out[t, o] = sum_k (q[o, k] - 8) * s[o, k / group] * x[t, k], codes and scales as `quantize4` gives them.

    x [rows, width] fp16 or bf16 (row stride free), scales of x's type; the group's size follows from their number.  The result [rows, out_width] is of x's type,
    or fp32 (`out_dtype`, or out's).  Sums are fp32.  In calls of more than 16 rows with a result of x's type each weight is rounded to that type once (an error like that of
    the result's own rounding; an fp32 result has none of it).  out must not overlap x, codes or scales.  Returns out."""
    return _out(load_native().linear4(_stream(x), x, codes, scales, out_dtype, out))


def logprobs(logits, tokens=None, top_k=0):
    """Log probabilities under softmax: logits [rows, vocab] fp32 / fp16 / bf16 (row stride free), tokens int32 [rows] or [rows, asked] or None -> (log
    probabilities of the tokens, of their shape (None without), entropy [rows], ids int32 [rows, top_k], their log probabilities [rows, top_k]), fp32.

    The top_k (at most 32) most likely tokens in descending order, ties to the lowest index.  A logit of -inf closes its token: -inf if it is asked for, and
    where no open one is left the ids are -1, with -inf.  A row without open tokens has the entropy 0.  The token -1 asks for none and gets 0, others outside
    the vocabulary get NaN.  Rows with a NaN or +inf get NaN; their ids are in range, NaN below every number."""
    return _out(load_native().logprobs(_stream(logits), logits, tokens, top_k))


def layer_sync(device=None):
    """Waits for torch's current stream on `device` (default: the current one), and raises `Hy3AttnError` if a bounded device-side wait of
    `experts`, `adapters` or `linear4` ran out there since the last call."""
    import torch
    with torch.cuda.device(device):
        rc = load_library().hy3a_layer_sync(torch.cuda.current_stream().cuda_stream)
    if rc:
        _out(rc)
