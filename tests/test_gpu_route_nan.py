"""hy3_b200.route with groups of nothing but NaN: such a group still stands before one whose experts are all closed, so that NaN is not lost."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups,size", [(2, 1), (2, 16), (8, 32), (3, 5)])
def test_groups_of_nan_stand_before_closed_ones(cuda, dtype, groups, size):
    import torch
    import hy3_b200
    l = torch.full((3, groups * size), -math.inf, device=cuda, dtype=getattr(torch, dtype))
    l[0, (groups - 1) * size:] = math.nan          # the last group, all of it
    l[1, -1] = math.nan                            # and one of it
    l[2] = math.nan
    l[2, 0] = -math.inf
    for bias in (None, torch.zeros(groups * size, device=cuda)):
        for score in ("sigmoid", "softmax"):
            k = min(4, size)
            ids, w = (t.cpu() for t in hy3_b200.route(l, bias, top_k=k, score=score, groups=groups, top_groups=1))
            first = (groups - 1) * size
            assert ids[0].tolist() == list(range(first, first + k)) and torch.isnan(w[0]).all(), (score, bias is None)
            assert ids[1, 0] == groups * size - 1 and bool((ids[1, 1:] == -1).all()) and math.isnan(w[1, 0])
            assert bool((ids[2] >= 0).any()) and math.isnan(w[2, 0])
