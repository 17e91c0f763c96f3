"""hy3_b200.adapters with infinite weights: where the definition gives an infinity or a number, so does the call."""
import math

import pytest

from test_gpu_adapters import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,base", [("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows,rank,out", [(1, 8, 264), (8, 40, 72), (64, 24, 520), (150, 136, 136), (300, 16, 264), (700, 200, 1032)])
def test_infinite_weights_keep_their_sign(cuda, dtype, base, rows, rank, out):
    """One infinite weight in b makes a column infinite, of the sign of u times that weight; the others stay as they are."""
    import torch
    import hy3_b200
    args = make(rows, 4, rank, 72, out, dtype, base, seed=3)
    x, rest, a, b, ids, s = args
    ids[:] = torch.arange(rows, device=cuda) % 4
    spots = ((0, 9, 3), (1, 40, rank - 1), (2, out - 1, 5))
    for i, (e, n, r) in enumerate(spots):
        b[e, n, r] = -math.inf if i == 1 else math.inf
    got = hy3_b200.adapters(*args)
    for e, n, r in spots:
        u = s[e].double() * (x[e::4].double() @ a[e, r].double())
        assert bool((u != 0).all()) and torch.equal(got[e::4, n].double(), torch.sign(u) * b[e, n, r].double())
        got[e::4, n] = 0
        rest[e::4, n] = 0
        b[e, n] = 0
    check(got, args)
