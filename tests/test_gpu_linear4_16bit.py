"""16-bit results of calls of more than 16 rows are those of weights that are rounded to the rows' type once: with A = sum of |rounded weight| |x|, a step of the sum for 16 products, 2^-22 of it each, and half a
step of the result, ((width / 16 + 20) 2^-22) A + V |y| (+ 2^-25, fp16's subnormal numbers).  That is tight enough to see one group's scale off by a half.

Against the weights as they are, the roundings e_k add sum e_k x_k.  They are the same for equal codes of a group, but x is independent of them and its values of each other, normal with variance 1 (rounded):
a normal number of variance sum e_k^2 at most (1 + 2^-8)^2, so that 7 standard deviations are passed with a chance of 2.6e-12 each, some 1e7 results here."""
import pytest

from test_gpu_linear4 import SIZES, V, make, weights

pytestmark = pytest.mark.gpu
MANY = [s for s in SIZES if s[0] > 16]


def near(got, x, w):
    """Whether each result is that of weights w, given in 64 bits."""
    y, a = x.double() @ w.T, x.double().abs() @ w.abs().T
    result = str(got.dtype).split(".")[1]
    limit = (x.shape[1] / 16 + 20) * 2.0 ** -22 * a + V[result] * y.abs() + (2.0 ** -25 if result == "float16" else 0) + x.shape[1] * 2.0 ** -149
    return (got.double() - y).abs() <= limit


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,width,out,group", MANY)
def test_of_weights_rounded_once(cuda, rows, width, out, group, dtype):
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, width, out, group, dtype, seed=1)
    got = hy3_b200.linear4(x, codes, scales)
    w = weights(codes, scales, group)
    rounded = w.to(x.dtype).double()
    assert bool(near(got, x, rounded).all())
    e = (rounded - w).square().sum(1).sqrt() * (1 + 2.0 ** -8)
    y, a = x.double() @ w.T, x.double().abs() @ w.abs().T
    limit = 7 * e + (width / 16 + 20) * 2.0 ** -22 * a + V[dtype] * (y.abs() + 7 * e) + 2.0 ** -25
    assert bool(((got.double() - y).abs() <= limit).all())


@pytest.mark.parametrize("rows,width,out", [(40, 8192, 300), (300, 8192, 300)])
def test_one_wrong_group_is_seen(cuda, rows, width, out):
    import torch
    import hy3_b200
    x, codes, scales, group = make(rows, width, out, 64, seed=2)
    got = hy3_b200.linear4(x, codes, scales)
    wrong = scales.clone()
    wrong[:, 77] *= 1.5
    inside = near(got, x, weights(codes, wrong, group).to(x.dtype).double())
    # With scales of standard deviation d, a result's limit is about 532 2^-22 x 8192 x 4 x 0.8 x 0.8 d + 2^-8 x 90 x 4.6 d = 4.3 d, and a scale s that is off by a half moves it by 0.5 s x 8 x 4.6 = 18 s in
    # quadratic mean: 9 d and more where |s| > d / 2, so that some 4 rows of 10 stay inside.  (Scales near 0 are no mistake worth seeing.)
    plain_to_see = scales[:, 77].double().abs() > 0.5 * width ** -0.5
    assert int(plain_to_see.sum()) > out // 2 and bool(inside.double().mean(0)[plain_to_see].max() < 0.9)
    assert bool(near(got, x, weights(codes, scales, group).to(x.dtype).double()).all())
