"""hy3_b200.experts against the definition in 64 bits, element by element.

The bound of an element, with v the rounding of the rows' type (bf16 2^-8, fp16 2^-11), c = 2^-22 a step of an fp32 sum on the tensor cores, and
all products of absolute values:
    gate and up come out with an error of at most K c (|gate| |x|) and K c (|up| |x|), K = hidden; silu has a slope of at most 1.1, so
    h = silu(g) u with dh = 1.1 |u| dg + |silu(g)| du + 8 * 2^-23 |h| (silu's own steps);
    h is rounded (v |h|, in fp16 2^-25 more for what is subnormal); down's sum adds I c |down| |h|, I = inter;
    the sum over the slots top_k * 2^-23 of its terms, and the result is rounded (v |y|, and the subnormal 2^-25).
"""
import pytest

pytestmark = pytest.mark.gpu
V = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
C, TINY = 2.0 ** -22, 2.0 ** -25


def reference(x, ids, w, gate, up, down, first=0):
    """(y, bound), fp64 on the CPU's or GPU's side of the inputs."""
    import torch
    v = V[str(x.dtype).split(".")[1]]
    rows, hidden = x.shape
    inter, k = gate.shape[1], ids.shape[1]
    y = torch.zeros((rows, hidden), dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(gate.shape[0]):
        r, j = torch.nonzero(ids == first + e, as_tuple=True)
        if not len(r):
            continue
        xe, G, U, D = x[r].double(), gate[e].double(), up[e].double(), down[e].double()
        g, u = xe @ G.T, xe @ U.T
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * u.abs() * hidden * C * (xe.abs() @ G.abs().T) + s.abs() * hidden * C * (xe.abs() @ U.abs().T) + 2.0 ** -20 * h.abs()
        dh = dh + v * (h.abs() + dh) + TINY
        wt = w[r, j].double().unsqueeze(1)
        y.index_add_(0, r, wt * (h @ D.T))
        dy = wt.abs() * (dh @ D.abs().T + inter * C * ((h.abs() + dh) @ D.abs().T))
        err.index_add_(0, r, dy)
        mag.index_add_(0, r, wt.abs() * (h @ D.T).abs())
    err = err + k * 2.0 ** -23 * (mag + err)
    return y, err + v * (y.abs() + err) + TINY


def make(rows, experts, top_k, hidden, inter, dtype="bfloat16", seed=0, device="cuda"):
    import torch
    gen = torch.Generator(device=device).manual_seed(seed + rows * 7 + experts)
    t = getattr(torch, dtype)

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(shape, device=device, generator=gen)).to(t)
    x = normal(rows, hidden)
    ids = torch.randint(0, experts, (rows, top_k), device=device, generator=gen).to(torch.int32)
    w = torch.rand((rows, top_k), device=device, generator=gen) - 0.2
    return x, ids, w, normal(experts, inter, hidden, scale=hidden ** -0.5), normal(experts, inter, hidden, scale=hidden ** -0.5), normal(experts, hidden, inter, scale=inter ** -0.5)


def check(got, args, first=0, rows=None):
    import torch
    want, bound = reference(*args, first=first)
    far = (got.double() - want).abs()
    if rows is not None:
        far, bound = far[rows], bound[rows]
    assert bool(torch.isfinite(far).all())
    assert bool((far <= bound).all()), "off by %.3g where %.3g is allowed" % (float(far.max()), float(bound.flatten()[(far - bound).argmax()]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,experts,top_k,hidden,inter", [
    (1, 1, 1, 8, 8), (1, 4, 2, 64, 32), (1, 192, 8, 256, 128), (2, 8, 3, 136, 72), (7, 5, 1, 1032, 200), (8, 16, 8, 512, 264), (33, 3, 2, 96, 40),
    (64, 192, 8, 128, 64), (100, 2, 2, 264, 136), (129, 7, 4, 512, 256), (300, 1, 1, 256, 72), (333, 10, 3, 1032, 200), (513, 3, 2, 128, 520), (1500, 4, 4, 320, 192)])
def test_sizes(cuda, dtype, rows, experts, top_k, hidden, inter):
    import hy3_b200
    args = make(rows, experts, top_k, hidden, inter, dtype)
    check(hy3_b200.experts(*args), args)


@pytest.mark.parametrize("rows", [3, 40, 700])
def test_slots_without_an_expert(cuda, rows):
    """-1, experts of other ranks and anything else outside are left out; a row of them alone is 0, whatever lay in out."""
    import torch
    import hy3_b200
    args = make(rows, 12, 4, 256, 136)
    x, ids, w = args[:3]
    ids[::2, 1] = -1
    ids[1::2, 2] = 12
    ids[0] = -1
    ids[rows - 1] = torch.tensor([-7, 12, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    w[ids < 0] = float("nan")
    out = torch.full_like(x, float("nan"))
    got = hy3_b200.experts(*args, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (got[0] == 0).all() and (got[rows - 1] == 0).all()
    check(got, args)
    # a rank that holds experts 5 to 8
    part = (x, ids, w) + tuple(t[5:9].contiguous() for t in args[3:])
    check(hy3_b200.experts(*part, first_expert=5), part, first=5)
    # nobody's rows
    none = torch.full_like(ids, 40)
    assert (hy3_b200.experts(x, none, w, *args[3:]) == 0).all()


@pytest.mark.parametrize("rows", [5, 70, 1100])
def test_all_rows_to_one_expert(cuda, rows):
    import hy3_b200
    args = make(rows, 9, 2, 256, 136, "float16", 5)
    args[1][:, 0] = 4
    args[1][:, 1] = 4          # twice, and with two weights
    check(hy3_b200.experts(*args), args)


def test_no_rows(cuda):
    import hy3_b200
    args = make(4, 3, 2, 64, 32)
    assert hy3_b200.experts(args[0][:0], args[1][:0], args[2][:0], *args[3:]).shape == (0, 64)


@pytest.mark.parametrize("rows", [4, 48, 600])
def test_strides(cuda, rows):
    import torch
    import hy3_b200
    args = make(rows, 6, 2, 136, 72)
    want = hy3_b200.experts(*args)
    wide = torch.full((rows, 200), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 16:152] = args[0]
    out = torch.zeros((rows, 160), dtype=torch.bfloat16, device=cuda)
    hy3_b200.experts(wide[:, 16:152], *args[1:], out=out[:, 8:144])
    assert torch.equal(out[:, 8:144], want) and (out[:, :8] == 0).all() and (out[:, 144:] == 0).all()


@pytest.mark.parametrize("rows", [6, 90, 900])
def test_what_is_not_finite_stays_where_it_is(cuda, rows):
    """A row of NaN and an expert of infinities reach the rows that use them, and no others."""
    import torch
    import hy3_b200
    args = make(rows, 8, 2, 192, 104)
    x, ids = args[0], args[1]
    x[rows // 2] = float("nan")
    args[3][3], args[5][3] = float("inf"), float("nan")
    ids[0] = torch.tensor([1, 2], dtype=torch.int32)
    got = hy3_b200.experts(*args)
    touched = (ids == 3).any(1)
    touched[rows // 2] = True
    assert not torch.isfinite(got[touched]).all(1).any() or int(touched.sum()) == 0
    clean = [t.clone() for t in args]
    clean[0][rows // 2] = 0
    clean[3][3], clean[5][3] = 0, 0
    assert torch.isfinite(got[~touched]).all()
    check(got.nan_to_num(0, 0, 0), clean, rows=~touched)


@pytest.mark.parametrize("rows,experts", [(1, 192), (9, 32), (64, 24), (1024, 12)])
def test_repeatable_bits(cuda, rows, experts):
    import torch
    import hy3_b200
    args = make(rows, experts, 8, 512, 264)
    want = hy3_b200.experts(*args)
    for _ in range(20):
        assert torch.equal(hy3_b200.experts(*args), want)


def test_results_do_not_hang_on_other_rows(cuda):
    """A row's result is the same bits, wherever in its batch it lies."""
    import torch
    import hy3_b200
    args = make(400, 6, 2, 256, 136)
    want = hy3_b200.experts(*args)
    turn = torch.randperm(400, device=cuda)
    got = hy3_b200.experts(args[0][turn].contiguous(), args[1][turn].contiguous(), args[2][turn].contiguous(), *args[3:])
    assert torch.equal(got, want[turn])


def test_another_stream_and_a_graph(cuda):
    import torch
    import hy3_b200
    args = make(50, 16, 4, 256, 136)
    want = hy3_b200.experts(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = hy3_b200.experts(args[0] + 0, *args[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = hy3_b200.experts(*args)
    for t in args[:3]:
        t.copy_(t.flip(0))         # other routing, too
    graph.replay()
    assert torch.equal(held, want.flip(0))


def test_refusals(cuda):
    import torch
    import hy3_b200
    x, ids, w, gate, up, down = make(4, 3, 2, 64, 32)
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.experts(x, ids, w, gate, up, down, first_expert=-1)
    bad = make(4, 3, 2, 60, 32)
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.experts(*bad)
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.experts(*make(4, 3, 33, 64, 32))
    shifted = torch.zeros(4 * 64 + 1, dtype=x.dtype, device=cuda)[1:].view(4, 64)
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.experts(shifted, ids, w, gate, up, down)
    for a in ((x.float(), ids, w, gate, up, down), (x, ids.long(), w, gate, up, down), (x, ids, w.half(), gate, up, down), (x, ids[:3], w, gate, up, down),
              (x, ids, w, gate.half(), up, down), (x, ids, w, gate, up[:2], down), (x, ids, w, gate, up, down.transpose(1, 2)), (x, ids.cpu(), w, gate, up, down)):
        with pytest.raises(AssertionError):
            hy3_b200.experts(*a)
    with pytest.raises(AssertionError):
        hy3_b200.experts(x, ids, w, gate, up, down, out=torch.empty((4, 63), dtype=x.dtype, device=cuda))
