"""hy3_b200.quantize4 against its definition: scales and codes are equal, and codes stand for the nearest values."""
import pytest

pytestmark = pytest.mark.gpu


def reference(w, group, dtype):
    """(codes, scales) by the definition, group by group in fp32 as it says."""
    import torch
    out, width = w.shape
    codes, scales = [], []
    for part in w.float().split(group, dim=1):
        high, low = part.max(1).values, part.min(1).values
        far = torch.where(high > -low, high, low)
        far = torch.where(torch.isnan(part).any(1), float("nan"), far)
        s = (-far / 8).to(dtype)
        q = torch.round(part / s.float().unsqueeze(1)).clamp(-8, 7) + 8
        good = torch.isfinite(s) & (s != 0)
        codes.append(torch.where(good.unsqueeze(1), q, 8.0))
        scales.append(s)
    q = torch.cat(codes, 1).to(torch.uint8)
    return q[:, 0::2] | q[:, 1::2] << 4, torch.stack(scales, 1)


def same(a, b):
    import torch
    return bool(((a == b) | (torch.isnan(a.float()) & torch.isnan(b.float()))).all())


def check(w, group, dtype):
    import hy3_b200
    codes, scales = hy3_b200.quantize4(w, group=group, dtype=dtype)
    want_codes, want_scales = reference(w, group, dtype)
    assert same(scales, want_scales) and codes.equal(want_codes)
    return codes, scales


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("w_dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("out,width", [(1, 32), (3, 64), (1, 4096), (7, 96), (130, 1056), (1001, 160), (33, 65536), (4096, 512)])
def test_sizes(cuda, out, width, group, w_dtype, dtype):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(out + width + group)
    w = torch.randn((out, width), device=cuda, generator=gen) * width ** -0.5
    check(w.to(getattr(torch, w_dtype)), group, getattr(torch, dtype))


@pytest.mark.parametrize("w_dtype", ["float32", "bfloat16", "float16"])
def test_values_between_two_codes(cuda, w_dtype):
    """Halves of steps, and their neighbours on both sides: ties go to the even code, in steps of the rounded scale."""
    import torch
    t = getattr(torch, w_dtype)
    for s in (0.5, 0.0111, 3.3, -0.77):
        base = torch.arange(-16, 16, device=cuda, dtype=torch.float32) / 2 * s
        w = torch.stack([base, base * (1 + 2.0 ** -23), base * (1 - 2.0 ** -24), base * (1 + 2.0 ** -8), base * (1 - 2.0 ** -9)]).to(t)
        for dtype in (torch.bfloat16, torch.float16):
            check(w, 32, dtype)


def test_codes_stand_for_the_nearest_values(cuda):
    import torch
    gen = torch.Generator(device=cuda).manual_seed(5)
    w = torch.randn((64, 1024), device=cuda, generator=gen)
    codes, scales = check(w, 64, torch.bfloat16)
    q = torch.stack([codes & 15, codes >> 4], -1).view(64, 1024).double() - 8
    s = scales.double().repeat_interleave(64, 1)
    # half a step; towards the end with 7 the scale's own rounding (2^-8 of 8 steps) and a whole one
    off = (w.double() - q * s).abs() / s.abs()
    inner = q < 7
    assert float(off[inner & (q > -8)].max()) <= 0.5 + 2.0 ** -20
    assert float(off[~inner].max()) <= 1 + 8 * 2.0 ** -8 and float(off[q == -8].max()) <= 0.5 + 2.0 ** -20


def test_zeros_ties_and_what_is_not_finite(cuda):
    import torch
    import hy3_b200
    inf, nan = float("inf"), float("nan")
    w = torch.zeros((9, 128), device=cuda)
    w[1, 5] = 2.0
    w[2, 5] = -2.0
    w[3, 5], w[3, 70] = 2.0, -2.0        # as far on both sides: the positive scale
    w[3, 9] = -2.0
    w[4, 5] = inf
    w[5, 5] = -inf
    w[6, 5] = nan
    w[7, 5], w[7, 64] = 1e-30, 4.0
    w[8, :] = 70000.0
    for group in (32, 64, 128):
        for dtype in (torch.bfloat16, torch.float16):
            codes, scales = check(w, group, dtype)
            assert (codes[0] == 0x88).all() and not scales[0].any() and not torch.signbit(scales[0].float()).any()
            assert scales[1, 0] == -0.25 and scales[2, 0] == 0.25 and scales[3, 0] == 0.25
            assert not torch.isfinite(scales[4:7, 0]).any() and (codes[4:7, :group // 2] == 0x88).all()
    huge = torch.full((1, 32), 3e38, device=cuda)
    codes, scales = hy3_b200.quantize4(huge, 32, torch.float16)      # the scale does not fit fp16
    assert torch.isinf(scales).all() and (codes == 0x88).all()
    tiny = torch.full((1, 32), 1e-9, device=cuda)
    check(tiny, 32, torch.float16)                                     # it is 0 there
    check(tiny * 200, 32, torch.float16)                               # it is subnormal


def test_strides_defaults_and_no_rows(cuda):
    import torch
    import hy3_b200
    gen = torch.Generator(device=cuda).manual_seed(1)
    wide = torch.randn((70, 400), device=cuda, generator=gen)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        v = wide.to(t)[:, 8:264]
        assert all(torch.equal(a, b) for a, b in zip(hy3_b200.quantize4(v), hy3_b200.quantize4(v.contiguous())))
        assert hy3_b200.quantize4(v)[1].dtype == (torch.float16 if t == torch.float16 else torch.bfloat16) and hy3_b200.quantize4(v)[1].shape == (70, 4)
        for row in (v[:1].expand(5, -1),):          # one row for all
            assert torch.equal(hy3_b200.quantize4(row)[0], hy3_b200.quantize4(row.contiguous())[0])
    codes, scales = hy3_b200.quantize4(wide[:0, :64])
    assert codes.shape == (0, 32) and scales.shape == (0, 1)


def test_refusals(cuda):
    import torch
    import hy3_b200
    w = torch.randn((8, 128), device=cuda)
    for bad in (lambda: hy3_b200.quantize4(w[:, :48]), lambda: hy3_b200.quantize4(w, group=16), lambda: hy3_b200.quantize4(w[:, 1:33]), lambda: hy3_b200.quantize4(w, group=0)):
        with pytest.raises(hy3_b200.Hy3AttnError):
            bad()
    for bad in (lambda: hy3_b200.quantize4(w.double()), lambda: hy3_b200.quantize4(w, dtype=torch.float32), lambda: hy3_b200.quantize4(w[0]), lambda: hy3_b200.quantize4(w.T)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        hy3_b200.quantize4(w, dtype="bf16")
    with pytest.raises(AssertionError, match="grad"):
        hy3_b200.quantize4(w.requires_grad_())
