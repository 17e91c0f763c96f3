"""hy3_b200.experts at the ends of what it takes, across the number of slots at which its form changes, and on two streams at once: bounds as in
test_gpu_experts.py."""
import pytest

from test_gpu_experts import check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,experts,top_k,hidden,inter", [(40, 1024, 8, 64, 32), (3, 1024, 8, 64, 32), (1, 40, 31, 136, 72), (31, 40, 1, 136, 72), (2, 5, 32, 264, 136), (50, 60, 32, 264, 136), (2, 6, 2, 5120, 2560),
                                                             (70, 6, 2, 5120, 2560), (20, 3, 2, 8, 8200), (3, 3, 2, 8, 8200), (20, 3, 2, 16392, 8), (3, 3, 2, 16392, 8)])
def test_ends(cuda, dtype, rows, experts, top_k, hidden, inter):
    """1024 experts held, 32 choices, 31 slots of as many experts, long rows and long gated products."""
    import torch
    import hy3_b200
    args = make(rows, experts, top_k, hidden, inter, dtype, 31)
    if rows * top_k == 31:
        args[1].view(-1)[:] = torch.randperm(experts, device=cuda)[:31].to(torch.int32)
    check(hy3_b200.experts(*args), args)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_row_in_small_and_large_calls(cuda, dtype):
    """From 32 slots on h has one number of the rows' type in the place of two: a row differs by no more than both may be off, which is far less than it is large."""
    import torch
    import hy3_b200
    args = make(32, 6, 1, 256, 136, dtype, 32)
    few = hy3_b200.experts(*(t[:31].contiguous() for t in args[:3]), *args[3:])
    many = hy3_b200.experts(*args)
    want, bound = reference(*args)
    assert bool(((few.double() - want[:31]).abs() <= bound[:31]).all()) and bool(((many.double() - want).abs() <= bound).all())
    assert float((few.double() - many[:31].double()).norm()) <= 2 * {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype] * float(want.norm())
    for n in (33, 40, 400):          # above the line the bits stay
        more = [torch.cat([t] * 13)[:n].contiguous() for t in args[:3]]
        assert torch.equal(hy3_b200.experts(*more, *args[3:])[:32], many)


def test_two_streams_at_once(cuda):
    """Calls on two streams, whose workspaces and waits are their own, give what they give alone."""
    import torch
    import hy3_b200
    jobs = [make(60, 24, 4, 512, 264, "bfloat16", 33), make(500, 5, 2, 264, 520, "float16", 34)]
    want = [hy3_b200.experts(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    off = [torch.zeros((), dtype=torch.int64, device=cuda) for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(200):
        for j, w, s, o in zip(jobs, want, streams, off):
            with torch.cuda.stream(s):
                o += (hy3_b200.experts(*j) != w).any()
    for s in streams:
        s.synchronize()
    hy3_b200.layer_sync()
    assert [int(o) for o in off] == [0, 0]
