"""quantize4, linear4 and logprobs in calls that their documentation allows and ordinary use seldom makes: rows that nobody wrote, far apart rows, one row for all, two streams at once, a first call
within a capture.  Tolerances are those of test_gpu_linear4.py and test_gpu_logprobs.py."""
import os
import subprocess
import sys

import pytest

from test_gpu_linear4 import bound, check, make, weights
from test_gpu_logprobs import near
from test_gpu_logprobs import reference as of_logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("result", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,out", [(1, 700), (5, 700), (16, 700), (40, 700), (300, 700), (40, 20001), (300, 10001)])
def test_rows_that_nobody_wrote(cuda, rows, out, result):
    """Every other row has a NaN, every sixth an infinity and no NaN: NaN where x has one, the definition's infinities and NaN, and the others as if alone."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, 1056, out)
    x[::2, 77] = float("nan")
    x[1::6, 5] = float("inf")
    got = hy3_b200.linear4(x, codes, scales, out_dtype=getattr(torch, result))
    assert bool(torch.isnan(got[::2]).all())
    w = weights(codes, scales, group)
    sign = w[:, 5].sign()
    for r in range(1, rows, 6):
        assert bool((got[r].double()[sign != 0] == (sign * float("inf"))[sign != 0]).all()) and bool(torch.isnan(got[r][sign == 0]).all())
    rest = [r for r in range(1, rows, 2) if r % 6 != 1]
    if rest:
        y, a = x[rest].double() @ w.T, x[rest].double().abs() @ w.abs().T
        assert bool(((got[rest].double() - y).abs() <= bound(y, a, x, scales, result)).all())


@pytest.mark.parametrize("result", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows", [1, 16, 40])
def test_nothing_finite_in_long_rows(cuda, rows, result):
    """An infinity in every row, so that every result is computed again: this ends well within the bound of what waits for it meanwhile."""
    import torch
    import hy3_b200
    gen = torch.Generator(device=cuda).manual_seed(rows)
    width, out = (4096 if rows == 1 else 65536), 20000
    codes = torch.randint(0, 256, (out, width // 2), device=cuda, generator=gen, dtype=torch.uint8)
    scales = torch.randn((out, width // 64), device=cuda, generator=gen).bfloat16()
    x = torch.randn((rows, width), device=cuda, generator=gen).bfloat16()
    x[:, 64] = float("inf")
    got = hy3_b200.linear4(x, codes, scales, out_dtype=getattr(torch, result))
    hy3_b200.layer_sync()
    sign = (((codes[:, 32] & 15).double() - 8) * scales[:, 1].double()).sign()
    assert bool((got[:, sign != 0].double() == (sign * float("inf"))[sign != 0]).all()) and bool(torch.isnan(got[:, sign == 0]).all())


@pytest.mark.parametrize("rows", [3, 16, 40])
def test_one_row_for_all_and_rows_far_apart(cuda, rows):
    """x expanded from one row; rows of x and of the result further apart than 2^32 bytes allow in 32 bits."""
    import torch
    import hy3_b200
    x, codes, scales, group = make(1, 512, 300)
    check(hy3_b200.linear4(x.expand(rows, 512), codes, scales, out_dtype=torch.float32), x.expand(rows, 512), codes, scales, group)
    x = make(rows, 512, 300)[0]
    step = ((1 << 32) // (rows - 1) + 512) // 8 * 8
    room = torch.empty((rows - 1) * step + 512, dtype=torch.bfloat16, device=cuda)
    assert room.numel() > 1 << 32
    far = room.as_strided((rows, 512), (step, 1))
    far.copy_(x)
    check(hy3_b200.linear4(far, codes, scales), x, codes, scales, group)
    out = room.as_strided((rows, 300), (step, 1))
    hy3_b200.linear4(x, codes, scales, out=out)
    check(out.contiguous(), x, codes, scales, group)


def test_logits_and_weights_far_apart(cuda):
    import torch
    import hy3_b200
    rows, step = 5, ((1 << 32) // 4 + 4096) // 8 * 8
    gen = torch.Generator(device=cuda).manual_seed(2)
    values = torch.randn((rows, 1024), device=cuda, generator=gen).bfloat16()
    room = torch.empty(4 * step + 1024, dtype=torch.bfloat16, device=cuda)
    far = room.as_strided((rows, 1024), (step, 1))
    far.copy_(values)
    tokens = torch.arange(rows, dtype=torch.int32, device=cuda)
    got, want = hy3_b200.logprobs(far, tokens, 3), of_logits(values, tokens, 3)
    near(got[0], want[0])
    near(got[1], want[1])
    assert torch.equal(got[2].long(), want[2])
    assert all(torch.equal(a, b) for a, b in zip(hy3_b200.quantize4(far), hy3_b200.quantize4(values)))


@pytest.mark.parametrize("rows", [1, 400])
def test_nan_ranks_below_the_lowest_number(cuda, rows):
    """Masks of the type's lowest value beside NaN: the masked tokens come before, in order, then NaN by index, then nothing."""
    import torch
    import hy3_b200
    logits = torch.full((rows, 3001), float("-inf"), device=cuda)
    logits[:, 5] = logits[:, 2999] = float("nan")
    logits[:, 40] = logits[:, 2000] = torch.finfo(torch.float32).min
    logits[:, 1000] = 1.0
    _, entropy, ids, top = hy3_b200.logprobs(logits, top_k=6)
    assert bool((ids == torch.tensor([1000, 40, 2000, 5, 2999, -1], dtype=torch.int32, device=cuda)).all())
    assert bool(torch.isnan(entropy).all()) and bool(torch.isnan(top[:, :5]).all())


def test_two_streams_at_once(cuda):
    import torch
    import hy3_b200
    sets = [make(rows, 2048, out) for rows, out in ((64, 3000), (200, 5000), (1, 20000), (9, 4000))]
    want = [hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32) for x, codes, scales, _ in sets]
    asked = [hy3_b200.logprobs(w, top_k=5) for w in want]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[] for _ in sets]
    for _ in range(10):
        for i, (x, codes, scales, _) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                y = hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32)
                got[i].append((y, hy3_b200.logprobs(y, top_k=5)))
    torch.cuda.synchronize()
    for i in range(len(sets)):
        for y, a in got[i]:
            assert torch.equal(y, want[i]) and all(torch.equal(p, q) for p, q in zip(a[1:], asked[i][1:]))
    hy3_b200.layer_sync()


FIRST = """
import torch, hy3_b200
x, w = torch.randn((%d, 256), device="cuda").bfloat16(), torch.randn((900, 256), device="cuda").bfloat16()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    codes, scales = hy3_b200.quantize4(w)
    y = hy3_b200.linear4(x, codes, scales, out_dtype=torch.float32)
    answer = hy3_b200.logprobs(y, top_k=3)
g.replay()
torch.cuda.synchronize()
codes2, scales2 = hy3_b200.quantize4(w)
y2 = hy3_b200.linear4(x, codes2, scales2, out_dtype=torch.float32)
assert torch.equal(codes, codes2) and torch.equal(scales, scales2) and torch.equal(y, y2)
assert all(torch.equal(a, b) for a, b in zip(answer[1:], hy3_b200.logprobs(y2, top_k=3)[1:]))
hy3_b200.layer_sync()
"""


@pytest.mark.parametrize("rows", [1, 40])
def test_first_call_within_a_capture(cuda, rows):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST % rows], cwd=root, capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stderr[-2000:]
