"""hy3_b200.linear4 against the definition in 64 bits, element by element.

With A = sum of |weight| |x| over an element's products, and half a step of the result's type added (fp32 2^-24, bf16 2^-8, fp16 2^-11; fp16 2^-25 where subnormal), the bound is
  up to 16 rows:
    8 steps of a group's sum on the tensor cores, 2^-22 of it each: 2^-19 A; the groups' sums in fp32, one after the other and where warps or blocks meet: (groups + 20) 2^-24 A;
  more rows, results in fp32 (weights as two numbers that are exact together):
    64 steps of the sum over 512 k's, 2^-22 of it each (half as many of fp16's 256): 2^-16 A; these sums in fp32: (width / 512 + 20) 2^-24 A (fp16: at most 256 sums, within the first term's room);
  more rows, results of the rows' type:
    a rounding of the weights, 2^-8 A (bf16) or 2^-11 A (fp16); a step of the sum for 16 products, 2^-22 of it each: (width / 16 + 20) 2^-22 A.
"""
import pytest

pytestmark = pytest.mark.gpu
V = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}


def weights(codes, scales, group):
    import torch
    q = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1).double() - 8
    return q * scales.double().repeat_interleave(group, 1)[:, :q.shape[1]]


def make(rows, width, out, group=64, dtype="bfloat16", seed=0, device="cuda"):
    import torch
    gen = torch.Generator(device=device).manual_seed(seed + rows + width * 3 + out * 7)
    t = getattr(torch, dtype)
    x = torch.randn((rows, width), device=device, generator=gen).to(t)
    codes = torch.randint(0, 256, (out, width // 2), device=device, generator=gen, dtype=torch.uint8)
    scales = (torch.randn((out, -(-width // group)), device=device, generator=gen) * width ** -0.5).to(t)
    return x, codes, scales, group


def bound(y, a, x, scales, result):
    if x.shape[0] <= 16:
        sums = 2.0 ** -19 + (scales.shape[1] + 20) * 2.0 ** -24
    elif result == "float32":
        sums = 2.0 ** -16 + (x.shape[1] / 512 + 20) * 2.0 ** -24
    else:
        sums = V[result] + (x.shape[1] / 16 + 20) * 2.0 ** -22
    # (fp32 sums among the subnormal numbers round to multiples of 2^-149, each of them)
    return sums * a + V[result] * y.abs() + (2.0 ** -25 if result == "float16" else 0) + (scales.shape[1] + 40) * 2.0 ** -150


def check(got, x, codes, scales, group):
    import torch
    w = weights(codes, scales, group)
    y, a = x.double() @ w.T, x.double().abs() @ w.abs().T
    result = str(got.dtype).split(".")[1]
    far, limit = (got.double() - y).abs(), bound(y, a, x, scales, result)
    assert got.shape == y.shape and bool(torch.isfinite(got).all())
    assert bool((far <= limit).all()), "off by %.3g where %.3g is allowed" % (float(far.max()), float(limit.flatten()[(far - limit).argmax()]))


SIZES = [(1, 32, 1, 32), (1, 32, 16, 64), (1, 4096, 1024, 64), (2, 96, 17, 32), (3, 160, 300, 128), (5, 1056, 1001, 32), (7, 8192, 296, 128), (8, 4128, 333, 64), (8, 12288, 100, 32), (4, 8224, 2500, 128),
         (9, 512, 264, 64), (16, 2048, 520, 128), (17, 96, 31, 32), (33, 1056, 1001, 128), (64, 4096, 640, 64), (100, 8192, 129, 32), (128, 256, 128, 64), (257, 1056, 515, 64),
         (300, 4096, 256, 128), (1000, 160, 24, 32), (2049, 544, 300, 64), (1, 65536, 150, 128), (130, 16384, 72, 32),
         (1, 256, 15000, 32), (1, 1056, 14400, 64), (1, 4096, 16001, 128), (1, 8192, 15001, 64), (1, 8192, 15000, 32), (1, 12288, 15000, 64), (64, 4096, 5000, 64), (16, 4096, 20000, 128), (15, 8192, 50, 64),
         (17, 96, 20001, 32), (40, 2048, 30000, 128), (600, 288, 10000, 64), (2100, 448, 3001, 32), (300, 4128, 10003, 64), (129, 1024, 19500, 32), (3, 8224, 2500, 32), (12, 4064, 3000, 64), (2, 672, 9, 32)]


@pytest.mark.parametrize("dtype,result", [("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16"), ("float16", "float32")])
@pytest.mark.parametrize("rows,width,out,group", SIZES)
def test_sizes(cuda, rows, width, out, group, dtype, result):
    import torch
    import hy3_b200
    args = make(rows, width, out, group, dtype)
    got = hy3_b200.linear4(*args[:3], out_dtype=getattr(torch, result))
    assert got.dtype == getattr(torch, result)
    check(got, *args)


@pytest.mark.parametrize("rows", [1, 8, 13, 40, 300])
def test_strides_and_out(cuda, rows):
    """Rows of a wider matrix, a result in a part of another, one row for all; what lies beside the result stays."""
    import torch
    import hy3_b200
    x, codes, scales, group = args = make(rows, 1056, 203, 64)
    for result in (torch.bfloat16, torch.float32):
        want = hy3_b200.linear4(x, codes, scales, out_dtype=result)
        wide_x = torch.full((rows, 1200), float("nan"), dtype=x.dtype, device=cuda)
        wide_x[:, 16:1072] = x
        wide = torch.full((rows, 251), 7.0, device=cuda, dtype=result)
        view = wide[:, 3:206]
        got = hy3_b200.linear4(wide_x[:, 16:1072], codes, scales, out=view)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
        assert (wide[:, :3] == 7).all() and (wide[:, 206:] == 7).all()
    same = x[:1].expand(rows, -1)
    check(hy3_b200.linear4(same, codes, scales), same, codes, scales, group)
    # scales that start on any boundary of their type, and rows of them that do
    odd = torch.empty(scales.numel() + 1, dtype=scales.dtype, device=cuda)[1:].view_as(scales)
    odd.copy_(scales)
    assert torch.equal(hy3_b200.linear4(x, codes, odd), hy3_b200.linear4(*args[:3]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 8, 13, 40, 300])
def test_rows_and_outputs_do_not_touch_each_other(cuda, rows, dtype):
    """A NaN or an infinity in a row, or in an output's scales, stays there; an infinite x gives the infinity or NaN that the definition gives."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 544, 60, 32, dtype)
    x[0, 3] = float("nan")
    scales[7, 2] = float("nan")
    scales[9, 1] = float("inf")
    got = hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32)
    assert torch.isnan(got[0]).all() and torch.isnan(got[:, 7]).all() and not torch.isfinite(got[:, 9]).any()
    keep = [o for o in range(60) if o not in (7, 9)]
    if rows > 1:
        check(got[1:][:, keep], x[1:], codes[keep], scales[keep], group)
    x[0, 3] = float("inf")
    scales[7, 2], scales[9, 1] = 0.5, 0.25
    got = hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32)
    want = x[:1].double() @ weights(codes, scales, group).T
    assert torch.equal(torch.isnan(got[:1]), torch.isnan(want)) and torch.equal(torch.isinf(got[:1]), torch.isinf(want)) and torch.equal(torch.sign(got[0]).nan_to_num(), torch.sign(want[0]).float().nan_to_num())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_one_row_on_a_large_matrix(cuda, dtype):
    """Its digits: magnitudes far apart in a group, subnormal and largest numbers, zeros; what is not finite."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(1, 1024, 15000, 64, dtype)
    top = torch.finfo(x.dtype).max / 2 if dtype == "float16" else 2.0 ** 110
    small = torch.finfo(x.dtype).smallest_normal
    scales.clamp_(-0.5, 0.5)
    k = torch.arange(1024, device=cuda)
    wide = 2.0 ** -(k % 24).double()
    cases = [x.double() * wide, x.double() * small, torch.where(k % 64 == 5, top, x.double()), torch.where(k % 64 == 5, x.double(), 0.0), x.double() * 0, torch.where(k < 512, x.double(), small / 4)]
    for row in cases:
        row = row.to(x.dtype).view(1, -1)
        check(hy3_b200.linear4(row, codes, scales, out_dtype=torch.float32), row, codes, scales, group)
    # a large number whose code is 8: what is left is as exact as it would be without
    codes[:, 2] = codes[:, 2] & 0xf0 | 8
    row = torch.where(k == 4, 1000.0, x.double() * 2.0 ** -12).to(x.dtype)
    check(hy3_b200.linear4(row, codes, scales, out_dtype=torch.float32), row, codes, scales, group)
    for odd in (float("nan"), float("inf"), -float("inf")):
        row = x.clone()
        row[0, 77] = odd
        got, want = hy3_b200.linear4(row, codes, scales, out_dtype=torch.float32), row.double() @ weights(codes, scales, group).T
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0, 1, -1).sign()[~torch.isfinite(want)], want.nan_to_num(0, 1, -1).sign().float()[~torch.isfinite(want)])


@pytest.mark.parametrize("rows", [2, 40])
def test_scales_of_far_apart_sizes(cuda, rows):
    """Groups and outputs on scales 2^40 apart, rows of 2^-30 and 2^30 (bf16): each element is as exact as its own products allow."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 1024, 96, 64)
    scales[::3] *= 2.0 ** 40
    scales[:, ::5] *= 2.0 ** -40
    x[::2] *= 2.0 ** -30
    x[1::2] *= 2.0 ** 30
    for result in (torch.bfloat16, torch.float32):
        check(hy3_b200.linear4(x, codes, scales, out_dtype=result), x, codes, scales, group)


def test_all_codes_at_all_places(cuda):
    """x one at a place at a time gives the weights themselves, exactly."""
    import torch
    import hy3_b200
    for dtype in (torch.bfloat16, torch.float16):
        codes = (torch.arange(64 * 128, device=cuda) * 37 % 256).to(torch.uint8).view(64, 128)
        scales = torch.linspace(-3, 3, 64 * 4, device=cuda).view(64, 4).to(dtype)
        x = torch.eye(256, device=cuda, dtype=dtype)
        want = weights(codes, scales, 64).T.float()
        for rows in (1, 8, 100, 256):
            for r in range(0, 256, rows):
                assert torch.equal(hy3_b200.linear4(x[r:r + rows], codes, scales, out_dtype=torch.float32), want[r:r + rows])


def test_nothing_to_do_and_repeatable_bits(cuda):
    import torch
    import hy3_b200
    x, codes, scales, _ = make(600, 1024, 512)
    assert hy3_b200.linear4(x[:0], codes, scales).shape == (0, 512) and hy3_b200.linear4(x, codes[:0], scales[:0]).shape == (600, 0)
    for n in (1, 8, 64, 600):
        want = hy3_b200.linear4(x[:n], codes, scales)
        for _ in range(20):
            assert torch.equal(hy3_b200.linear4(x[:n], codes, scales), want)


def test_another_stream_and_a_graph(cuda):
    import torch
    import hy3_b200
    for rows in (1, 50, 400):
        args = make(rows, 1056, 300, 64)
        other = make(rows, 1056, 300, 64, seed=9)
        want, then = hy3_b200.linear4(*args[:3]), hy3_b200.linear4(*other[:3])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(hy3_b200.linear4(*args[:3]), want)
        torch.cuda.current_stream().wait_stream(side)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
        with torch.cuda.graph(graph):
            hy3_b200.linear4(*args[:3], out=out)
        for t, s in zip(args[:3], other[:3]):
            t.copy_(s)
        graph.replay()
        assert torch.equal(out, then)


def test_refusals(cuda):
    import torch
    import hy3_b200
    x, codes, scales, _ = make(4, 128, 40)
    for bad in (lambda: hy3_b200.linear4(x.float(), codes, scales), lambda: hy3_b200.linear4(x, codes, scales.half()), lambda: hy3_b200.linear4(x, codes.int(), scales),
                lambda: hy3_b200.linear4(x, codes[:, :48], scales), lambda: hy3_b200.linear4(x, codes, scales.repeat(1, 4)), lambda: hy3_b200.linear4(x[0], codes, scales), lambda: hy3_b200.linear4(x, codes, scales[:30]),
                lambda: hy3_b200.linear4(x, codes, scales, out_dtype=torch.float16), lambda: hy3_b200.linear4(x, codes, scales, out=torch.empty((4, 39), device=cuda)),
                lambda: hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32, out=torch.empty((4, 40), device=cuda, dtype=x.dtype)), lambda: hy3_b200.linear4(x, codes.cpu(), scales)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.linear4(torch.zeros((4, 132), dtype=x.dtype, device=cuda)[:, 4:], codes, scales)
    x.requires_grad_()
    with pytest.raises(AssertionError, match="grad"):
        hy3_b200.linear4(x, codes, scales)
    with torch.no_grad():
        assert not hy3_b200.linear4(x, codes, scales).requires_grad


def test_a_wait_that_ran_out_is_reported(cuda):
    import torch
    import hy3_b200
    hy3_b200.layer_sync()
    assert hy3_b200.load_library().hy3a_layer_wait_out(torch.cuda.current_stream().cuda_stream, 4) == 0
    with pytest.raises(hy3_b200.Hy3AttnError, match="linear4") as e:
        hy3_b200.layer_sync()
    assert e.value.code == -6
    hy3_b200.layer_sync()
