"""hy3_b200.route against the definition in 64 bits.

Tolerances.  A weight is s / sum * scale with s = 1 / (1 + exp(-l)) or exp(l - m) / sum: expf is good to 2 ulp, each of the at most 5 further
operations and the sum of up to 32 positive terms to half an ulp a step, 12 ulp of 2^-23 together = 1.5e-6; a softmax's l - m, up to 32 here, is
rounded to half of 2^-19, which enters exp as a relative 1e-6: 2.5e-6.  Which experts are taken is exact, but two whose scores in 64 bits
lie within 1e-6 (a score is at most 1 + |bias| < 2, its 32-bit error 4 ulp) may stand in either order.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
NEAR, RTOL = 1e-6, {"sigmoid": 1.5e-6, "softmax": 2.5e-6}


def reference(logits, bias, top_k, score, groups, top_groups):
    """Selection scores (closed: -inf) and scores in 64 bits."""
    import torch
    l = logits.double()
    s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)
    c = s + (0 if bias is None else bias.double())
    c = torch.where(l == -math.inf, -math.inf, c)
    size = c.shape[1] // groups
    if groups > 1:
        for row in c:
            per = row.view(groups, size)
            best = per.sort(dim=1, descending=True).values[:, :2]
            stands = [float(b[b > -math.inf].sum()) if bool((b > -math.inf).any()) else -math.inf for b in best]
            keep = sorted(range(groups), key=lambda g: (-stands[g], g))[:top_groups]
            for g in range(groups):
                if g not in keep:
                    per[g] = -math.inf
    return c, s


def check(logits, bias, top_k, score="sigmoid", groups=1, top_groups=1, renormalize=True, scale=2.826):
    import torch
    import hy3_b200
    ids, w = hy3_b200.route(logits, bias, top_k=top_k, score=score, groups=groups, top_groups=top_groups, renormalize=renormalize, scale=scale)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == (logits.shape[0], top_k)
    ids, w = ids.cpu().long(), w.cpu().double()
    c, s = reference(logits.cpu(), None if bias is None else bias.cpu(), top_k, score, groups, top_groups)
    want = c.sort(dim=1, descending=True, stable=True)
    n_open = (c > -math.inf).sum(1)
    for r in range(logits.shape[0]):
        n = min(top_k, int(n_open[r]))
        assert (ids[r, n:] == -1).all() and (w[r, n:] == 0).all(), r
        got = ids[r, :n]
        assert len(set(got.tolist())) == n and bool(((got >= 0) & (got < c.shape[1])).all())
        assert float((c[r, got] - want.values[r, :n]).abs().max() if n else 0) <= NEAR, (r, got, want.indices[r, :n])
        x = s[r, got]
        x = (x / (x.sum() + 1e-20) if renormalize else x) * scale
        assert bool(((w[r, :n] - x).abs() <= RTOL[score] * x.abs() + 1e-37).all()), (r, w[r], x)
    return ids, w


def make(rows, experts, dtype, seed, closed=0.0, device="cuda"):
    import torch
    gen = torch.Generator(device=device).manual_seed(seed)
    l = 1.5 * torch.randn((rows, experts), device=device, generator=gen)
    if closed:
        l[torch.rand(l.shape, device=device, generator=gen) < closed] = -math.inf
    return l.to(dtype), 0.05 * torch.randn(experts, device=device, generator=gen)


@pytest.mark.parametrize("experts,top_k", [(1, 1), (7, 7), (8, 2), (32, 1), (33, 4), (97, 6), (192, 8), (256, 32), (500, 10), (1024, 3)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_sizes_and_types(cuda, experts, top_k, score, dtype):
    import torch
    l, bias = make(13, experts, getattr(torch, dtype), experts + top_k)
    check(l, bias, top_k, score)
    check(l, None, top_k, score, renormalize=False, scale=1.0)


@pytest.mark.parametrize("experts,groups,top_groups,top_k", [(8, 8, 3, 2), (64, 2, 1, 8), (96, 3, 2, 6), (160, 5, 2, 6), (256, 8, 4, 8), (256, 32, 5, 8), (1000, 20, 1, 7), (192, 1, 1, 8)])
@pytest.mark.parametrize("closed", [0.0, 0.4, 0.95])
def test_groups_and_closed_experts(cuda, experts, groups, top_groups, top_k, closed):
    import torch
    for score in ("sigmoid", "softmax"):
        l, bias = make(37, experts, torch.float32, experts + groups, closed)
        check(l, bias if score == "sigmoid" else None, top_k, score, groups, top_groups)


def test_one_row_and_none(cuda):
    import torch
    import hy3_b200
    l, bias = make(1, 192, torch.float32, 3)
    check(l, bias, 8)
    ids, w = hy3_b200.route(l[:0], bias)
    assert ids.shape == w.shape == (0, 8)


def test_ties_go_to_the_lowest_index(cuda):
    import torch
    import hy3_b200
    for experts in (40, 192, 300):
        for dtype in (torch.float32, torch.bfloat16):
            l = torch.zeros((3, experts), device=cuda, dtype=dtype)
            l[1, 5::7] = 1.0
            l[2, experts - 1] = 2.0
            for score in ("sigmoid", "softmax"):
                ids = hy3_b200.route(l, top_k=8, score=score)[0].cpu().tolist()
                assert ids[0] == list(range(8))
                ones = list(range(5, experts, 7))[:8]
                assert ids[1] == ones + [i for i in range(experts) if i % 7 != 5][:8 - len(ones)]
                assert ids[2] == [experts - 1] + list(range(7))
    # and so do groups that stand equally
    ids = hy3_b200.route(torch.zeros((1, 64), device=cuda), top_k=4, groups=8, top_groups=2)[0].cpu().tolist()
    assert ids == [[0, 1, 2, 3]]


def test_rows_without_open_experts(cuda):
    import torch
    import hy3_b200
    l = torch.full((4, 96), -math.inf, device=cuda)
    l[1, 17] = 0.5
    l[2] = torch.finfo(torch.float32).min       # open, with a score of 0
    l[3, 90:] = 1.0
    for score in ("sigmoid", "softmax"):
        for groups, top_groups in ((1, 1), (4, 2)):
            ids, w = hy3_b200.route(l, top_k=8, score=score, groups=groups, top_groups=top_groups, scale=2.0)
            ids, w = ids.cpu(), w.cpu()
            assert (ids[0] == -1).all() and (w[0] == 0).all()
            assert ids[1].tolist() == [17] + [-1] * 7 and w[1].tolist() == [2.0] + [0.0] * 7
            assert ids[2].tolist() == list(range(8)) and torch.isfinite(w[2]).all()
            assert ids[3].tolist() == list(range(90, 96)) + [-1] * 2 and abs(float(w[3].sum()) - 2.0) < 1e-5
    # a bias of -inf closes an expert for every row, one of the lowest value puts it behind the others
    bias = torch.zeros(96, device=cuda)
    bias[:90] = -math.inf
    bias[95] = torch.finfo(torch.float32).min
    ids = hy3_b200.route(torch.zeros((2, 96), device=cuda), bias, top_k=8)[0].cpu().tolist()
    assert ids == [[90, 91, 92, 93, 94, 95, -1, -1]] * 2


def test_nan_ranks_last_and_shows(cuda):
    import torch
    import hy3_b200
    l = torch.zeros((4, 64), device=cuda)
    l[0] = math.nan
    l[1, 3] = math.nan
    l[2, 3] = math.inf
    l[3, 8:] = -math.inf
    l[3, 0] = math.nan
    ids, w = (t.cpu() for t in hy3_b200.route(l, top_k=8, score="sigmoid"))
    assert ids[0].tolist() == list(range(8)) and torch.isnan(w[0]).all()
    assert ids[1].tolist() == [0, 1, 2, 4, 5, 6, 7, 8] and torch.isfinite(w[1]).all()
    assert ids[2].tolist() == [3, 0, 1, 2, 4, 5, 6, 7] and torch.isfinite(w[2]).all()
    assert ids[3].tolist() == [1, 2, 3, 4, 5, 6, 7, 0] and torch.isnan(w[3]).all()
    ids, w = (t.cpu() for t in hy3_b200.route(l, top_k=8, score="softmax", groups=4, top_groups=2))
    for r in (0, 1, 2):
        assert bool(((ids[r] >= 0) & (ids[r] < 64)).all()) and torch.isnan(w[r]).all()


def test_row_stride_and_offsets_beyond_32_bits(cuda):
    import torch
    l, bias = make(20, 208, torch.float32, 9)
    wide = torch.full((20, 333), math.nan, device=cuda)
    wide[:, 5:213] = l
    a, b = check(l, bias, 8), check(wide[:, 5:213], bias, 8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    stride = (1 << 31) // 19 + 3
    big = torch.empty(19 * stride + 64, dtype=torch.float16, device=cuda)
    far = big.as_strided((20, 64), (stride, 1))
    far.copy_(l[:, :64])
    assert 19 * stride > 1 << 31
    check(far, None, 4)


def test_another_stream_and_a_graph(cuda):
    import torch
    import hy3_b200
    l, bias = make(300, 192, torch.float32, 21)
    want = hy3_b200.route(l, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moved = l + 0
        got = hy3_b200.route(moved, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = hy3_b200.route(l, bias)
    l.copy_(l.flip(0))
    graph.replay()
    assert torch.equal(held[0], want[0].flip(0)) and torch.equal(held[1], want[1].flip(0))


def test_refusals(cuda):
    import torch
    import hy3_b200
    l = torch.zeros((2, 64), device=cuda)
    for kw in ({"top_k": 0}, {"top_k": 33}, {"groups": 3}, {"groups": 64}, {"groups": 8, "top_groups": 9}, {"groups": 8, "top_groups": 0}, {"groups": 16, "top_groups": 1, "top_k": 5}):
        with pytest.raises(hy3_b200.Hy3AttnError):
            hy3_b200.route(l, **kw)
    with pytest.raises(hy3_b200.Hy3AttnError):
        hy3_b200.route(torch.zeros((2, 1025), device=cuda))
    with pytest.raises(KeyError):
        hy3_b200.route(l, score="tanh")
    for bad in (l.double(), l[0], l.t(), l.cpu()):
        with pytest.raises((AssertionError, IndexError, TypeError)):
            hy3_b200.route(bad)
    for bias in (torch.zeros(63, device=cuda), torch.zeros(64, device=cuda, dtype=torch.float16), torch.zeros(64)):
        with pytest.raises(AssertionError):
            hy3_b200.route(l, bias)
