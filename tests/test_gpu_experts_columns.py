"""hy3_b200.experts where columns and slots are of very different sizes: the bound of test_gpu_experts.py holds element by element, whatever the columns
beside an element, or other slots' shares of it, hold."""
import pytest

from test_gpu_experts import check, make

pytestmark = pytest.mark.gpu


def run(args):
    import hy3_b200
    return hy3_b200.experts(*args)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,experts,top_k,hidden,inter", [(1, 4, 2, 64, 32), (3, 8, 8, 136, 72), (4, 8, 8, 136, 72), (40, 5, 2, 520, 264), (700, 6, 2, 264, 136)])
def test_columns_beside_large_ones(cuda, dtype, rows, experts, top_k, hidden, inter):
    """A few rows of down are 2^8 to 2^14 times the others, as channels of trained models are."""
    args = make(rows, experts, top_k, hidden, inter, dtype, 11)
    for i, at in enumerate(range(5, hidden, 32)):
        args[5][:, at] *= 2.0 ** (8 + 2 * (i % 4))
    check(run(args), args)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 15, 16, 300])
def test_large_columns_that_cancel(cuda, dtype, rows):
    """Two experts that differ in the small rows of down alone, taken with weights 1 and -1: the large columns are 0, the small ones are not."""
    import torch
    args = list(make(rows, 2, 2, 192, 104, dtype, 12))
    for t in args[3:]:
        t[1] = t[0]
    args[5][1] = args[5][0].flip(0)
    for at in range(7, 192, 48):
        args[5][:, at] = args[5][0, at] * 2.0 ** 12
    args[1][:] = torch.tensor([0, 1], dtype=torch.int32)
    args[2][:] = torch.tensor([1.0, -1.0])
    got = run(args)
    check(got, args)
    assert float(got[:, 8:40].float().abs().mean()) > 0.01
