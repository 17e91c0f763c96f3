"""Prompts through examples/decoder_layer.py: every row that its operators give behind one another, against the same layer in 64 bits.

Chunks of 64 to 256 rows take the forms of many rows (lists of experts and adapters, tiles), one launch behind another without a pause.  Tolerance: that of
test_gpu_decoder_layer.py, 4 % of what the layer adds in quadratic mean, over all rows of a prompt; a single row, whose few dozen roundings do not average out as
well, twice that.
"""
import pytest

from test_gpu_decoder_layer import example, reference  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,chunk", [("int8", 64), ("fp16", 256)])
def test_prompts_against_64_bits(cuda, example, kv, chunk):  # noqa: F811
    import torch
    import hy3_b200
    layer = example.DecoderLayer(hidden=512, experts=24, top_k=4, inter=192, adapters=3, rank=8, requests=3, max_tokens_per_seq=512, chunk=chunk, kv_dtype=kv, seed=5)
    gen = torch.Generator(device=cuda).manual_seed(10)
    for s, (n, adapter) in enumerate(((300, 2), (64, -1), (7, 0))):
        x = torch.randn((n, 512), device=cuda, generator=gen)
        routed = []
        got = layer.prompt(s, x, adapter, routed)
        ids, weights = (torch.cat(t) for t in zip(*routed))
        assert ids.shape == weights.shape == (n, 4) and got.shape == x.shape
        _, _, score = reference(layer, x, adapter)
        c = score + layer.bias.double()
        assert bool((c.gather(1, ids.long()).amin(1) >= c.topk(4, dim=1).values[:, -1] - 0.02).all()) and bool((ids.sort(1).values.diff(dim=1) > 0).all())
        taken = score.gather(1, ids.long())
        assert bool(((weights.double() - taken / taken.sum(1, keepdim=True) * 2.826).abs() <= 0.02 * weights).all())
        want = reference(layer, x, adapter, ids, weights)[0]
        added, off = want - x.double(), got.double() - want
        assert float(off.norm() / added.norm()) <= 0.04, (s, float(off.norm() / added.norm()))
        assert float((off.norm(dim=1) / added.norm(dim=1)).max()) <= 0.08, (s, float((off.norm(dim=1) / added.norm(dim=1)).max()))
    layer.ctx.sync()
    hy3_b200.layer_sync()
    layer.close()
