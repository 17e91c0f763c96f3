"""linear4 where a pair of CTAs has many tiles of a few steps each, numbers of steps that the teams which make weights do not divide among them: many launches behind each other have the same bits, no wait
runs out, and results are the definition's.  (Tolerances: test_gpu_linear4.py.)"""
import pytest

from test_gpu_linear4 import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width,out,group,result", [(2698, 448, 16942, 64, "float32"), (128, 1000 // 32 * 32, 40003, 32, "float32"), (500, 160, 30000, 128, "float32"), (100, 320, 60000, 64, "bfloat16"),
                                                         (128, 704, 40000, 32, "bfloat16"), (1500, 192, 5000, 64, "bfloat16"), (90, 96, 70001, 32, "bfloat16"), (40, 32, 90000, 32, "float32")])
def test_many_launches_have_the_same_bits(cuda, rows, width, out, group, result):
    import torch
    import hy3_b200
    args = make(rows, width, out, group)
    first = hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result))
    check(first[:, :5000], args[0], args[1][:5000], args[2][:5000], group)
    check(first[:, -300:], args[0], args[1][-300:], args[2][-300:], group)
    for _ in range(60):
        for _ in range(8):
            last = hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result))
        assert torch.equal(last, first)
    hy3_b200.layer_sync()
