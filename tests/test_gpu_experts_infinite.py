"""hy3_b200.experts with infinite weights: where the definition gives an infinity or a number, so does the call, with few slots and with many."""
import math

import pytest

from test_gpu_experts import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 7, 31, 32, 200])
def test_infinite_weights_keep_their_sign(cuda, dtype, rows):
    """One infinite weight in down makes a column infinite, of the sign of h times that weight; one in up makes a row's h infinite there."""
    import torch
    import hy3_b200
    x, ids, w, gate, up, down = make(rows, 4, 1, 136, 72, dtype, 21)
    ids[:, 0] = torch.arange(rows, device=cuda) % 4
    w[:] = 0.75
    clean = down.clone()
    down[0, 9, 3], down[1, 40, 70] = math.inf, -math.inf
    got = hy3_b200.experts(x, ids, w, gate, up, down)
    want = torch.zeros(got.shape, dtype=torch.float64, device=cuda)
    for r in range(rows):
        e = r % 4
        g, u = gate[e].double() @ x[r].double(), up[e].double() @ x[r].double()
        want[r] = 0.75 * (down[e].double() @ (g / (1 + torch.exp(-g)) * u))
    far = torch.isinf(want)
    assert int(far.sum()) == sum(1 for r in range(rows) if r % 4 < 2) and not torch.isnan(want).any()
    assert torch.equal(got.double()[far], want[far]) and bool(torch.isfinite(got[~far]).all())
    safe = got.clone()
    safe[far] = 0
    down[0, 9], down[1, 40], clean[0, 9], clean[1, 40] = 0, 0, 0, 0
    safe[0::4, 9] = 0
    safe[1::4, 40] = 0
    check(safe, (x, ids, w, gate, up, clean))
    up[2, 5, 0] = math.inf
    got = hy3_b200.experts(x, ids, w, gate, up, down)[2::4]
    if len(got):
        r = torch.arange(2, rows, 4, device=cuda)
        g = x[r].double() @ gate[2, 5].double()
        sign = torch.sign(x[r, 0].double()) * torch.sign(g)
        want = sign.unsqueeze(1) * torch.sign(down[2, :, 5].double()) * math.inf
        assert torch.equal(got.double(), want)
