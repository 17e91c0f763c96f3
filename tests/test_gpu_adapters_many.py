"""hy3_b200.adapters with about as many adapters as rows, and with more adapters than rows are listed by: bounds as in test_gpu_adapters.py."""
import pytest

from test_gpu_adapters import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("base", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,n", [(193, 200), (300, 400), (300, 299), (2000, 2040), (2000, 2047), (3000, 2048), (4096, 5000)])
def test_as_many_adapters_as_rows(cuda, rows, n, base):
    import torch
    import hy3_b200
    args = make(rows, n, 8, 64, 72, base=base)
    check(hy3_b200.adapters(*args), args)
    args[4][:] = torch.randperm(n, device=cuda)[torch.arange(rows, device=cuda) % n].to(torch.int32)        # each row another one
    check(hy3_b200.adapters(*args), args)
    args[4][1::2] = -1
    check(hy3_b200.adapters(*args), args)
