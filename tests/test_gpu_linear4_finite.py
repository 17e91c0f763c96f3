"""linear4's results do not turn infinite, or NaN, with the number of rows: a group's sum of steps beyond fp32 whose product with its scale is not, weights beyond fp32, infinite scales.  (Tolerances: test_gpu_linear4.py.)"""
import pytest

from test_gpu_linear4 import check, make, weights

pytestmark = pytest.mark.gpu
CALLS = [(1, 500), (1, 15000), (2, 500), (8, 500), (9, 500), (16, 500), (16, 9000), (17, 500), (40, 500), (40, 30001), (300, 500)]


@pytest.mark.parametrize("result", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,out", CALLS)
@pytest.mark.parametrize("width,group", [(544, 64), (512, 32), (8224, 128)])
def test_large_rows_with_small_scales(cuda, rows, out, width, group, result):
    """x of 2^120 to 2^127, scales of 2^-20 and less: 8 x is beyond fp32, and so are sums of a group, no result is."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, width, out, group)
    large = torch.where(x > 0, 1.0, -1.0) * (1 + x.abs() % 1) * 2.0 ** 126
    x = torch.where(torch.arange(rows, device=cuda).view(-1, 1) % 3 < 2, large, large * 2.0 ** -6).to(x.dtype)
    scales = (scales * 2.0 ** -15).to(x.dtype)
    scales[3 % out] = 0
    args = x, codes, scales, group
    check(hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result)), *args)
    # one such row beside ordinary ones
    if rows > 1:
        mixed = make(rows, width, out, group)[0]
        mixed[rows // 2] = x[0]
        args = mixed, codes, scales, group
        check(hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result)), *args)


@pytest.mark.parametrize("result", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,out", CALLS)
def test_large_scales_with_small_rows(cuda, rows, out, result):
    """Scales of 2^125 to 2^127, with which up to 8 steps are beyond fp32 (and beyond bf16), and rows of 2^-30; what quantize4 makes of the largest fp32 numbers is of that kind."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 544, out, 32)
    x = (x * 2.0 ** -30).to(x.dtype)
    scales[:, ::3] = ((1 + scales[:, ::3].abs() % 1) * 2.0 ** 126).to(scales.dtype)
    args = x, codes, scales, group
    check(hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result)), *args)
    w = torch.randn((64, 512), device=cuda)
    w[::2, 5::32] = torch.finfo(torch.float32).max
    codes, scales = hy3_b200.quantize4(w, 32, torch.bfloat16)
    assert bool((scales.float()[::2] == -2.0 ** 125).all())
    args = x[:, :512], codes, scales, 32
    check(hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result)), *args)


@pytest.mark.parametrize("dtype,result", [("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows,out", CALLS)
def test_infinite_scales(cuda, rows, out, dtype, result):
    """The definition's sum of infinite terms: infinite where they have one sign, NaN where they have both, or a code is 8."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 544, out, 32, dtype)
    x[0] = x[0].abs() + 0.125
    scales[:8, 2] = float("inf")
    scales[4:8, 2] *= -1
    codes[:2, 32:48] = 0x91          # steps of both signs
    codes[2:4, 32:48] = 0xfc         # of one
    codes[4:6, 32:48] = 0x37
    codes[6:8, 32:48] = 0x83         # and some 0
    scales[9, 1] = float("nan")
    got = hy3_b200.linear4(x, codes, scales, out_dtype=getattr(torch, result))
    want = x.double() @ weights(codes, scales, group).T
    assert bool(torch.isinf(want[0, 2:6]).all()) and bool(torch.isnan(want[0, [0, 1, 6, 7, 9]]).all())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite].double(), want[infinite])
    rest = [o for o in range(min(out, 2000)) if o > 9]
    check(got[:, rest], x, codes[rest], scales[rest], group)
