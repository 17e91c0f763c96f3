"""The operators together: examples/decoder_layer.py against the same layer in 64 bits.

Tolerance.  Between the operators rows are rounded to bf16 (2^-9 of their size on average at most): the norm's output twice, the projections'
outputs, the attention's output, the experts' products and sums; about eight roundings in a row, none of which is amplified (weights scale by
1 / sqrt(width)), and int8 or fp16 caches add less (int8: 0.5 / 127 of a row's largest value, 3 of its mean, a code, on K and V: 2^-7 each).  The residual
stream passes unrounded.  So rows agree to sqrt(8) 2^-9 + 2 2^-7 < 2.5 % of what the layer adds in quadratic mean; 4 % are allowed.  Which experts a row
takes may hang on a rounding, so the reference takes the experts that the layer took, having checked that their scores are the best to 2 %.
"""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def rotate(x, pos):
    """rotate_half RoPE of [n, heads, 128] rows at positions pos."""
    import torch
    f = 1.0 / (11158840.0 ** (torch.arange(64, dtype=torch.float64, device=x.device) / 64))
    a = pos.double().view(-1, 1) * f
    c, s = a.cos().unsqueeze(1), a.sin().unsqueeze(1)
    lo, hi = x[..., :64], x[..., 64:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def reference(layer, x, adapter, ids=None, weights=None):
    """Rows x [n, hidden] of one request in 64 bits; with ids and weights [n, k] the rows' experts."""
    import torch
    import torch.nn.functional as F
    d = lambda t: t.double()  # noqa: E731
    x = d(x)
    n = x.shape[0]

    def norm(v, w, eps=1e-5):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w

    def adapted(v, w, a, b):
        y = v @ d(w).T
        return y if adapter < 0 else y + d(layer.scales[adapter]) * (v @ d(a[adapter]).T) @ d(b[adapter]).T
    q, k, v = adapted(norm(x, d(layer.norm1)), layer.qkv, layer.qkv_a, layer.qkv_b).split([8192, 1024, 1024], dim=1)
    pos = torch.arange(n, device=x.device)
    q, k, v = rotate(norm(q.reshape(n, 64, 128), 1.0), pos), rotate(norm(k.reshape(n, 8, 128), 1.0), pos), v.reshape(n, 8, 128)
    scores = torch.einsum("qgjd,kgd->gjqk", q.view(n, 8, 8, 128), k) / math.sqrt(128)
    p = torch.softmax(scores.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf), -1)
    x1 = x + adapted(torch.einsum("gjqk,kgd->qgjd", p, v).reshape(n, 8192), layer.o, layer.o_a, layer.o_b)
    h = norm(x1, d(layer.norm2))
    score = torch.sigmoid(h @ d(layer.router).T)
    if ids is None:
        return x1, h, score
    y = F.silu(h @ d(layer.shared_gate).T) * (h @ d(layer.shared_up).T) @ d(layer.shared_down).T
    for e in range(layer.gate.shape[0]):
        r, j = torch.nonzero(ids == e, as_tuple=True)
        if len(r):
            y[r] += d(weights)[r, j].unsqueeze(1) * ((F.silu(h[r] @ d(layer.gate[e]).T) * (h[r] @ d(layer.up[e]).T)) @ d(layer.down[e]).T)
    return x1 + y, h, score


@pytest.mark.parametrize("kv", ["int8", "fp16"])
def test_layer_against_64_bits(cuda, example, kv):
    import torch
    import hy3_b200
    layer = example.DecoderLayer(hidden=512, experts=24, top_k=4, inter=192, adapters=3, rank=8, requests=3, max_tokens_per_seq=256, chunk=64, kv_dtype=kv, seed=4)
    gen = torch.Generator(device=cuda).manual_seed(9)
    adapter, lengths, steps = [1, -1, 2], [5, 70, 1], 3
    rows = [torch.randn((n + steps, 512), device=cuda, generator=gen) for n in lengths]
    for s in range(3):
        layer.prompt(s, rows[s][:lengths[s]], adapter[s])
    for i in range(steps):
        at = [n + i for n in lengths]
        x = torch.stack([rows[s][at[s]] for s in range(3)])
        got, ids, weights = layer.step([0, 1, 2], at, x, torch.tensor(adapter, dtype=torch.int32, device=cuda))
        for s in range(3):
            part = rows[s][:at[s] + 1]
            _, _, score = reference(layer, part, adapter[s])
            c = (score + layer.bias.double())[-1]
            assert float(c[ids[s].long()].min()) >= float(c.topk(4).values[-1]) - 0.02 and len(set(ids[s].tolist())) == 4
            taken = score[-1][ids[s].long()]
            assert bool(((weights[s].double() - taken / taken.sum() * 2.826).abs() <= 0.02 * weights[s]).all())
            every = torch.full((at[s] + 1, 4), -1, dtype=torch.int32, device=cuda)
            every[-1] = ids[s]
            w = torch.zeros((at[s] + 1, 4), device=cuda)
            w[-1] = weights[s]
            want = reference(layer, part, adapter[s], every, w)[0][-1]
            added, off = want - x[s].double(), got[s].double() - want
            assert float(off.norm() / added.norm()) <= 0.04, (i, s, float(off.norm() / added.norm()))
    layer.ctx.sync()
    hy3_b200.layer_sync()
    layer.close()
