"""examples/decoder_layer.py with its shared projections in 4 bits keeps them in 4 bits alone."""
import pytest

from test_gpu_decoder_layer import example  # noqa: F401

pytestmark = pytest.mark.gpu


def test_no_16_bit_copy_is_kept(cuda, example):  # noqa: F811
    import torch
    sizes = []
    for bits4 in (False, True):
        before = torch.cuda.memory_allocated()
        layer = example.DecoderLayer(hidden=1024, experts=4, top_k=2, inter=512, adapters=1, rank=8, requests=1, max_tokens_per_seq=128, chunk=16, bits4=bits4)
        sizes.append(torch.cuda.memory_allocated() - before)
        got = layer.prompt(0, torch.randn((20, 1024), device=cuda), 0)
        assert bool(torch.isfinite(got).all())
        layer.close()
        del layer, got
    weights = (80 * 128 + 64 * 128 + 3 * 512) * 1024
    # 2 bytes a weight, and 1 / 2 + 2 / 64; torch rounds allocations up to 512 bytes
    assert sizes[0] - sizes[1] >= weights * (2 - 0.5 - 2 / 64) - 20 * 512
