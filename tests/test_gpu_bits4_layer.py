"""Weights in 4 bits as they are used: examples/decoder_layer.py with its shared projections in 4 bits, and the output head with what is asked of its logits, against
64 bits on the weights that the codes stand for.

The layer: test_gpu_decoder_layer.py's tolerance and reference, whose weights are those here.  The head: rows are rounded to bf16.  The steps of a
value in [2^e, 2^(e+1)) are 2^(e-7), so its rounding is uniform over +-2^(e-8), at most +-2^-8 of the value (all of it at 2^e, half of that below 2^(e+1)), in quadratic mean 2^-8 / sqrt(3) of it
at most.  The roundings are independent: a logit is off by 2^-8 / sqrt(3) of sqrt(sum w^2 x^2) in quadratic mean at most, and six times that is allowed, which a sum of bounded
terms like these passes with a chance below 2 exp(-18) (Hoeffding's lemma; 4e-8, for 1.4 million logits).  (2^-9 / sqrt(3) would be the mean at the upper end of each binade, the least, not the most.)  Log probabilities and
entropy change by no more than the largest change of a logit allows (a logit less log sum exp: |d log p| <= 2 max |d l|; |d H| <= 2 max |d l| (1 + H)).  What logprobs says of the logits that linear4
gave is exact to fp32.
"""
import pytest

from test_gpu_decoder_layer import example, reference  # noqa: F401
from test_gpu_linear4 import weights
from test_gpu_logprobs import near
from test_gpu_logprobs import reference as of_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,chunk", [("int8", 64), ("fp16", 256)])
def test_prompts_and_steps(cuda, example, kv, chunk):  # noqa: F811
    import torch
    import hy3_b200
    layer = example.DecoderLayer(hidden=512, experts=24, top_k=4, inter=192, adapters=3, rank=8, requests=3, max_tokens_per_seq=512, chunk=chunk, kv_dtype=kv, seed=6, bits4=True)
    for name, at in (("qkv", "qkv"), ("o", "o"), ("gate", "shared_gate"), ("up", "shared_up"), ("down", "shared_down")):
        setattr(layer, at, weights(*layer.bits4[name], 64))          # what the reference multiplies with
    gen = torch.Generator(device=cuda).manual_seed(11)
    lengths, adapters, rows = [300, 5, 1], [2, -1, 0], []
    for s in range(3):
        rows.append(torch.randn((lengths[s] + 2, 512), device=cuda, generator=gen))
        routed = []
        got = layer.prompt(s, rows[s][:lengths[s]], adapters[s], routed)
        ids, w = (torch.cat(t) for t in zip(*routed))
        x = rows[s][:lengths[s]]
        want = reference(layer, x, adapters[s], ids, w)[0]
        added, off = want - x.double(), got.double() - want
        assert float(off.norm() / added.norm()) <= 0.04, (s, float(off.norm() / added.norm()))
    for i in range(2):
        at = [n + i for n in lengths]
        x = torch.stack([rows[s][at[s]] for s in range(3)])
        got, ids, w = layer.step([0, 1, 2], at, x, torch.tensor(adapters, dtype=torch.int32, device=cuda))
        for s in range(3):
            every, ws = torch.full((at[s] + 1, 4), -1, dtype=torch.int32, device=cuda), torch.zeros((at[s] + 1, 4), device=cuda)
            every[-1], ws[-1] = ids[s], w[s]
            want = reference(layer, rows[s][:at[s] + 1], adapters[s], every, ws)[0][-1]
            added, off = want - x[s].double(), got[s].double() - want
            assert float(off.norm() / added.norm()) <= 0.04, (i, s, float(off.norm() / added.norm()))
    layer.ctx.sync()
    hy3_b200.layer_sync()
    layer.close()


@pytest.mark.parametrize("rows", [1, 8, 60])
def test_output_head(cuda, example, rows):  # noqa: F811
    import torch
    import hy3_b200
    head = example.OutputHead(hidden=512, vocab=20011, group=32, seed=3)
    gen = torch.Generator(device=cuda).manual_seed(rows)
    x = 3 * torch.randn((rows, 512), device=cuda, generator=gen)
    tokens = torch.randint(0, 20011, (rows,), device=cuda, generator=gen).to(torch.int32)
    logits = head.logits(x)
    asked, entropy, ids, top = head.answer(x, tokens, 7)
    want_asked, want_entropy, want_ids, want_top = of_logits(logits, tokens, 7)
    near(asked, want_asked)
    near(entropy, want_entropy)
    near(top, want_top)
    assert torch.equal(ids.long(), want_ids)
    h = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5) * head.norm.double()
    w = weights(head.codes, head.scales, 32)
    exact = h @ w.T
    limit = 6 * 2.0 ** -8 / 3 ** 0.5 * (h.square() @ w.square().T).sqrt()
    assert bool(((logits.double() - exact).abs() <= limit).all())
    logp = torch.log_softmax(exact, -1)
    most = limit.amax(-1)
    assert bool(((asked.double() - logp.gather(1, tokens.long().view(-1, 1)).squeeze(1)).abs() <= 2 * most).all())
    exact_entropy = -(logp.exp() * logp).sum(-1)
    assert bool(((entropy.double() - exact_entropy).abs() <= 2 * most * (1 + exact_entropy)).all())
    # the tokens taken are the best there are, as far as the logits tell
    best = exact.gather(1, ids.long())
    assert bool((best.amin(-1) >= exact.topk(7, dim=-1).values[:, -1] - 2 * most).all())
    hy3_b200.layer_sync()


def test_a_step_in_a_graph(cuda, example):  # noqa: F811
    """Projection, head and log probabilities captured together, replayed on other rows; two graphs in turn."""
    import torch
    head = example.OutputHead(hidden=256, vocab=9001, group=64, seed=5)
    x, y = torch.randn((3, 256), device=cuda), torch.randn((40, 256), device=cuda)
    then_x, then_y = torch.randn_like(x), torch.randn_like(y)
    want_x, want_y = head.answer(then_x, top_k=4), head.answer(then_y, top_k=4)
    graphs, outs = [], []
    for t in (x, y):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(head.answer(t, top_k=4))
    x.copy_(then_x)
    y.copy_(then_y)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, (want_x, want_y)):
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
