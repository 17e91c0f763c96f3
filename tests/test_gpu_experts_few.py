"""hy3_b200.experts with few slots: h is kept as two numbers of the rows' type."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,first,rest", [("bfloat16", 2.0 ** -8, 2.0 ** -16), ("float16", 2.0 ** -11, 2.0 ** -22)])
@pytest.mark.parametrize("rows", [1, 3, 15])
def test_what_cancels_between_experts(cuda, dtype, first, rest, rows):
    """x picks one column of gate and up, down is the identity, and two experts whose up differs a little are subtracted: an element is h0 - h1, rounded
    once (`first`), up to what two numbers leave of h (`rest` of each) and the exponential, the quotient and two products in fp32 (2^-19 of each, |g| < 8).
    One number would leave `first` of each."""
    import torch
    import hy3_b200
    gen = torch.Generator(device=cuda).manual_seed(rows)
    n, t = 256, getattr(torch, dtype)
    g = torch.randn(n, device=cuda, generator=gen).to(t)
    u = (1 + torch.rand(n, device=cuda, generator=gen)).to(t)
    gate, up = torch.zeros(2, 2, n, n, dtype=t, device=cuda)
    gate[:, :, 0], up[0, :, 0], up[1, :, 0] = g, u, u * (1 + 2.0 ** -6)
    x = torch.zeros(rows, n, dtype=t, device=cuda)
    x[:, 0] = 1
    down = torch.eye(n, dtype=t, device=cuda).repeat(2, 1, 1)
    ids = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda).repeat(rows, 1)
    w = torch.tensor([[1.0, -1.0]], device=cuda).repeat(rows, 1)
    a = g.double() * torch.sigmoid(g.double())
    h0, h1 = a * up[0, :, 0].double(), a * up[1, :, 0].double()
    far = (hy3_b200.experts(x, ids, w, gate, up, down).double() - (h0 - h1)).abs()
    bound = first * (h0 - h1).abs() + (1 + first) * (rest + 2.0 ** -19) * (h0.abs() + h1.abs()) + (2.0 ** -25 if dtype == "float16" else 0)
    assert bool((far <= bound).all())
