"""hy3_b200.experts over and over with few slots an expert, where most of a tile's rows are not there: no wait runs out (`layer_sync` would say so), and the
bits stay."""
import pytest

from test_gpu_experts import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,experts,top_k,hidden,inter,times", [(40, 16, 1, 512, 520, 4000), (8, 48, 8, 2048, 1536, 1500), (64, 96, 8, 1024, 1536, 800), (300, 4, 1, 264, 2048, 3000),
                                                                 (700, 12, 1, 512, 1032, 2000)])
def test_many_calls(cuda, dtype, rows, experts, top_k, hidden, inter, times):
    import torch
    import hy3_b200
    args = make(rows, experts, top_k, hidden, inter, dtype)
    want = hy3_b200.experts(*args)
    other = torch.zeros((), dtype=torch.int64, device=cuda)
    for _ in range(times):
        other += (hy3_b200.experts(*args) != want).any()
    hy3_b200.layer_sync()
    assert bool(torch.isfinite(want).all()) and int(other) == 0
