"""linear4 where a pair of CTAs has many tiles of a few steps each, numbers of steps that the teams which make weights do not divide among them: many launches behind each other have the same bits, no wait
runs out, and results are the definition's.  (Tolerances: test_gpu_linear4.py.)"""
import pytest

from test_gpu_linear4 import check, make, weights

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


@pytest.mark.parametrize("rows,result", [(256, "bfloat16"), (128, "float32"), (200, "float32")])
def test_nothing_finite_in_the_largest_tiles(cuda, rows, result):
    """Every result of tiles of 256 rows (fp32: 128) of the largest width is computed again; a pair of CTAs has two such tiles and more: no wait runs out, and the next call is as ever."""
    import torch
    import hy3_b200
    gen = torch.Generator(device=cuda).manual_seed(rows)
    width, out = 65536, 37888
    codes = torch.randint(0, 256, (out, width // 2), device=cuda, generator=gen, dtype=torch.uint8)
    scales = torch.randn((out, width // 64), device=cuda, generator=gen).bfloat16()
    x = torch.randn((rows, width), device=cuda, generator=gen).bfloat16()
    x[:, 64] = float("inf")
    hy3_b200.layer_sync()
    got = hy3_b200.linear4(x, codes, scales, out_dtype=getattr(torch, result))
    hy3_b200.layer_sync()
    sign = (((codes[:, 32] & 15).double() - 8) * scales[:, 1].double()).sign()
    want = torch.where(sign == 0, float("nan"), sign * float("inf")).to(got.dtype)
    assert torch.equal(torch.nan_to_num(got, 7.0, 1.0, -1.0), torch.nan_to_num(want, 7.0, 1.0, -1.0).expand_as(got))
    args = make(rows, 544, 30000)
    check(hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result)), *args)


@pytest.mark.parametrize("dtype,result", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("rows,out", [(300, 20001), (64, 40000)])
def test_what_is_not_finite_among_several_tiles(cuda, rows, out, dtype, result):
    """An infinity in one row, a NaN in another, weights beyond the type's range in some outputs: settled in their places, all else as if alone, in odd and in even output widths."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 544, out, 32, dtype)
    scales.clamp_(-0.5, 0.5)
    x[7, 40] = float("inf")
    x[rows - 1, 3] = float("nan")
    scales[out - 5, 3], scales[out // 2, 0] = float("inf"), float("nan")
    got = hy3_b200.linear4(x, codes, scales, out_dtype=getattr(torch, result))
    w = weights(codes, scales, group)
    want = x[7].double() @ w.T
    assert torch.equal(torch.isnan(got[7]), torch.isnan(want)) and torch.equal(torch.nan_to_num(got[7].double(), 0, 1, -1).sign()[torch.isinf(want)], torch.nan_to_num(want, 0, 1, -1).sign()[torch.isinf(want)])
    assert bool(torch.isnan(got[rows - 1]).all()) and bool(torch.isnan(got[:, out // 2]).all()) and not torch.isfinite(got[:, out - 5]).any()
    r, o = torch.ones(rows, dtype=torch.bool, device=cuda), torch.ones(out, dtype=torch.bool, device=cuda)
    r[[7, rows - 1]], o[[out - 5, out // 2]] = False, False
    check(got[r][:, o], x[r], codes[o], scales[o], group)
    hy3_b200.layer_sync()
