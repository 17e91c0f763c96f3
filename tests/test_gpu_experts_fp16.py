"""hy3_b200.experts on fp16 rows whose gated products are far from 1.

The bound of test_gpu_experts.py, but what the rounding of h to fp16 leaves of small values (2^-25 there) is no more than 2^-38 of the slot's largest, since
the largest is brought near the top of the type's range first (step 2^-24 at a largest of 2^14 and more: 2^-25 2^-14 = 2^-39, and one power of two for where a
largest value lies within its own).
"""
import pytest

from test_gpu_experts import C, TINY, V, make

pytestmark = pytest.mark.gpu


def reference_of_range(x, ids, w, gate, up, down):
    """(y, bound), fp64: h keeps 2^-38 of its row's largest in the place of 2^-25."""
    import torch
    v = V[str(x.dtype).split(".")[1]]
    rows, hidden = x.shape
    inter, k = gate.shape[1], ids.shape[1]
    y = torch.zeros((rows, hidden), dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(gate.shape[0]):
        r, j = torch.nonzero(ids == e, as_tuple=True)
        if not len(r):
            continue
        xe, G, U, D = x[r].double(), gate[e].double(), up[e].double(), down[e].double()
        g, u = xe @ G.T, xe @ U.T
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * u.abs() * hidden * C * (xe.abs() @ G.abs().T) + s.abs() * hidden * C * (xe.abs() @ U.abs().T) + 2.0 ** -20 * h.abs()
        dh = dh + v * (h.abs() + dh) + 2.0 ** -38 * (h.abs() + dh).amax(1, keepdim=True)
        wt = w[r, j].double().unsqueeze(1)
        y.index_add_(0, r, wt * (h @ D.T))
        err.index_add_(0, r, wt.abs() * (dh @ D.abs().T + inter * C * ((h.abs() + dh) @ D.abs().T)))
        mag.index_add_(0, r, wt.abs() * (h @ D.T).abs())
    err = err + k * 2.0 ** -23 * (mag + err)
    return y, err + v * (y.abs() + err) + TINY


@pytest.mark.parametrize("rows", [1, 15, 16, 400])
@pytest.mark.parametrize("s,d", [(2.0 ** 8, 2.0 ** -12), (2.0 ** -10, 2.0 ** 16)])
def test_fp16_beyond_its_range_between_the_products(cuda, rows, s, d):
    """The gated products may be larger than fp16 holds (s^2 times the usual), and much smaller, as long as the result is not."""
    import torch
    import hy3_b200
    args = list(make(rows, 3, 2, 264, 136, "float16", 13))
    args[0], args[3], args[4], args[5] = args[0] * s, args[3] / s, args[4] * s, args[5] * d
    assert all(bool(torch.isfinite(t).all()) for t in args)
    got = hy3_b200.experts(*args)
    want, bound = reference_of_range(*args)
    far = (got.double() - want).abs()
    assert float(want.abs().max()) < 60000 and bool((far <= bound).all()), "off by %.3g where %.3g is allowed" % (float(far.max()), float(bound.flatten()[(far - bound).argmax()]))
