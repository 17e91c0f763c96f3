"""hy3_b200.adapters against the definition in 64 bits, element by element.

The bound of an element, with c = 2^-22 a step of an fp32 sum on the tensor cores, K = width, and all products of absolute values:
    u = scale A x has an error of at most (K + 2) c |scale| |A| |x|; it enters the second product as a value rounded to the rows' type and the
    rounded rest, which leaves 2^-16 (bf16) or 2^-21 (fp16) of the row's largest |u|;
    the second sum adds 2 rank c; base + it and the way to base's type a rounding each (fp32 2^-24, bf16 2^-8, fp16 2^-11; fp16 2^-25 where
    subnormal).
"""
import pytest

pytestmark = pytest.mark.gpu
V = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}
REST = {"bfloat16": 2.0 ** -16, "float16": 2.0 ** -21}
C, TINY = 2.0 ** -22, 2.0 ** -25


def name(t):
    return str(t.dtype).split(".")[1]


def reference(x, base, a, b, ids, scales):
    import torch
    y, err = base.double(), torch.zeros(base.shape, dtype=torch.float64, device=base.device)
    rank, width = a.shape[1:]
    for i in range(a.shape[0]):
        r = torch.nonzero(ids == i).squeeze(1)
        if not len(r):
            continue
        s, xe, A, B = float(scales[i]), x[r].double(), a[i].double(), b[i].double()
        u = s * (xe @ A.T)
        du = (width + 2) * C * abs(s) * (xe.abs() @ A.abs().T)
        du = du + REST[name(x)] * (u.abs() + du).amax(1, keepdim=True)
        y[r] += u @ B.T
        err[r] = du @ B.abs().T + 2 * rank * C * ((u.abs() + du) @ B.abs().T)
    return y, err + (2.0 ** -24 + V[name(base)]) * (y.abs() + base.double().abs() + err) + (TINY if name(base) == "float16" else 0)


def make(rows, n, rank, width, out, dtype="bfloat16", base="float32", runs=False, seed=0, device="cuda"):
    import torch
    gen = torch.Generator(device=device).manual_seed(seed + rows * 5 + n)
    t = getattr(torch, dtype)

    def normal(*shape, scale=1.0):
        return scale * torch.randn(shape, device=device, generator=gen)
    ids = torch.randint(-1, n, (rows,), device=device, generator=gen).to(torch.int32)
    if runs:
        ids = ids.sort().values
    return (normal(rows, width).to(t), normal(rows, out).to(getattr(torch, base)), normal(n, rank, width, scale=width ** -0.5).to(t),
            normal(n, out, rank, scale=rank ** -0.5).to(t), ids, 0.5 + torch.rand(n, device=device, generator=gen))


def check(got, args, rows=None):
    import torch
    want, bound = reference(*args)
    far = (got.double() - want).abs()
    if rows is not None:
        far, bound = far[rows], bound[rows]
    assert bool(torch.isfinite(far).all())
    assert bool((far <= bound).all()), "off by %.3g where %.3g is allowed" % (float(far.max()), float(bound.flatten()[(far - bound).argmax()]))


@pytest.mark.parametrize("dtype,base", [("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("rows,n,rank,width,out,runs", [
    (1, 1, 8, 8, 8, False), (1, 8, 16, 4096, 1024, False), (2, 3, 24, 264, 72, False), (7, 2, 40, 1032, 520, False), (8, 64, 64, 512, 256, False), (33, 5, 72, 136, 264, True),
    (64, 40, 64, 2048, 512, False), (100, 3, 128, 640, 328, True), (257, 4, 32, 512, 1032, True), (300, 30, 16, 256, 512, False), (1000, 7, 256, 320, 200, True), (2049, 2, 8, 4096, 264, True)])
def test_sizes(cuda, dtype, base, rows, n, rank, width, out, runs):
    import hy3_b200
    args = make(rows, n, rank, width, out, dtype, base, runs)
    check(hy3_b200.adapters(*args), args)


@pytest.mark.parametrize("rows", [1, 20, 400])
def test_rows_without_an_adapter_are_base(cuda, rows):
    import torch
    import hy3_b200
    x, base, a, b, ids, s = make(rows, 4, 32, 512, 264)
    x[:] = float("nan")
    base[0, 0] = float("inf")
    for none in (-1, 4, -2 ** 31, 2 ** 31 - 1):
        ids[:] = none
        assert torch.equal(hy3_b200.adapters(x, base, a, b, ids, s), base)


@pytest.mark.parametrize("rows", [3, 64, 700])
def test_in_place_and_strides(cuda, rows):
    """out may be base; rows of a wider matrix, as q, k and v lie in one projection's rows."""
    import torch
    import hy3_b200
    args = make(rows, 5, 16, 256, 136)
    want = hy3_b200.adapters(*args)
    x, base = args[:2]
    wide_x = torch.full((rows, 320), float("nan"), dtype=x.dtype, device=cuda)
    wide_x[:, 8:264] = x
    wide = torch.zeros((rows, 204), device=cuda)
    wide[:, 4:140] = base
    view = wide[:, 4:140]
    got = hy3_b200.adapters(wide_x[:, 8:264], view, *args[2:], out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
    assert (wide[:, :4] == 0).all() and (wide[:, 140:] == 0).all()
    got = hy3_b200.adapters(x, base[:1].expand(rows, -1), *args[2:])       # one base row for all
    check(got, (x, base[:1].expand(rows, -1)) + args[2:])


@pytest.mark.parametrize("rows", [8, 30, 500])
def test_what_is_not_finite_stays_where_it_is(cuda, rows):
    """A NaN row and an adapter of infinities reach their own rows, also where others share the tile."""
    import torch
    import hy3_b200
    args = make(rows, 5, 16, 256, 136)
    x, base, a, b, ids, s = args
    ids[:] = torch.arange(rows, device=cuda) % 5
    x[3] = float("nan")
    a[1], b[2] = float("inf"), float("nan")
    got = hy3_b200.adapters(*args)
    touched = (ids == 1) | (ids == 2)
    touched[3] = True
    assert not torch.isfinite(got[touched]).all(1).any()
    clean = [t.clone() for t in args]
    clean[0][3] = 0
    clean[2][1], clean[3][2] = 0, 0
    assert torch.isfinite(got[~touched]).all()
    check(got.nan_to_num(0, 0, 0), clean, rows=~touched)


def test_fp16_beyond_its_range_between_the_products(cuda):
    """u may be larger than fp16 holds, and much smaller."""
    import hy3_b200
    for big in (2.0 ** 12, 2.0 ** -12):
        args = list(make(40, 3, 16, 512, 72, "float16"))
        args[0] = args[0] * big
        args[2] = args[2] * big
        args[3] = args[3] / big
        args[5] = args[5] / big
        check(hy3_b200.adapters(*args), args)


def test_no_rows_and_repeatable_bits(cuda):
    import torch
    import hy3_b200
    args = make(600, 9, 64, 1024, 512)
    x, base, a, b, ids, s = args
    assert hy3_b200.adapters(x[:0], base[:0], a, b, ids[:0], s).shape == (0, 512)
    for n in (1, 64, 600):
        want = hy3_b200.adapters(x[:n], base[:n], a, b, ids[:n], s)
        for _ in range(10):
            assert torch.equal(hy3_b200.adapters(x[:n], base[:n], a, b, ids[:n], s), want)


def test_another_stream_and_a_graph(cuda):
    import torch
    import hy3_b200
    args = make(48, 6, 32, 512, 264)
    want = hy3_b200.adapters(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hy3_b200.adapters(args[0] + 0, *args[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = hy3_b200.adapters(*args)
    for i in (0, 1, 4):
        args[i].copy_(args[i].flip(0))
    graph.replay()
    check(held, args)


def test_refusals(cuda):
    import torch
    import hy3_b200
    x, base, a, b, ids, s = make(4, 3, 16, 64, 72)
    for rank in (4, 20, 264):
        with pytest.raises(hy3_b200.Hy3AttnError):
            hy3_b200.adapters(*make(4, 3, rank, 64, 72))
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.adapters(*make(4, 3, 16, 60, 72))
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.adapters(*make(4, 3, 16, 64, 76))
    for bad in ((x.float(), base, a, b, ids, s), (x, base.half(), a, b, ids, s), (x, base[:3], a, b, ids, s), (x, base, a.half(), b, ids, s), (x, base, a, b[:2], ids, s),
                (x, base, a, b, ids.long(), s), (x, base, a, b, ids, s.half()), (x, base, a, b, ids.cpu(), s), (x, base, a.transpose(1, 2), b, ids, s)):
        with pytest.raises(AssertionError):
            hy3_b200.adapters(*bad)
    with pytest.raises(AssertionError):
        hy3_b200.adapters(x, base, a, b, ids, s, out=torch.empty((4, 72), dtype=x.dtype, device=cuda))


@pytest.mark.parametrize("rows,n,out", [(9, 1, 264), (40, 2047, 72), (40, 2048, 72), (600, 3000, 136), (513, 500, 1032), (5000, 3, 136)])
def test_many_adapters_and_rows_in_any_order(cuda, rows, n, out):
    """Adapters beyond those whose rows can be listed, rows of one adapter that lie apart, and rows shared by several blocks of the plan."""
    import torch
    import hy3_b200
    args = list(make(rows, n, 8, 64, out))
    check(hy3_b200.adapters(*args), args)
    turn = torch.randperm(rows, device=cuda)
    want = hy3_b200.adapters(*args)
    got = hy3_b200.adapters(args[0][turn].contiguous(), args[1][turn].contiguous(), args[2], args[3], args[4][turn].contiguous(), args[5])
    assert torch.equal(got, want[turn])


@pytest.mark.parametrize("rows", [300, 1100])
def test_long_rows_in_place_in_any_order(cuda, rows):
    """Rows that are fetched and stored by their numbers, some of them twice, where the output lies over base."""
    import torch
    import hy3_b200
    for base in ("float32", "bfloat16"):
        args = make(rows, 7, 40, 128, 1096, base=base)
        want = hy3_b200.adapters(*args)
        check(want, args)
        got = args[1].clone()
        hy3_b200.adapters(args[0], got, *args[2:], out=got)
        assert torch.equal(got, want)
