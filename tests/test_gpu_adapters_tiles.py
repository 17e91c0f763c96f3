"""hy3_b200.adapters where tiles, ranks and columns end inside the hardware's: bounds as in test_gpu_adapters.py; and what u keeps on an fp32 base."""
import pytest

from test_gpu_adapters import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,base", [("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
@pytest.mark.parametrize("rows,n,rank,out", [(129, 1, 8, 8), (192, 1, 64, 128), (193, 1, 72, 256), (255, 2, 136, 384), (400, 3, 192, 136), (321, 2, 200, 520), (640, 90, 248, 264)])
def test_ends_of_tiles(cuda, dtype, base, rows, n, rank, out):
    """Rows of one adapter (and -1) around multiples of 64, ranks around multiples of 64, columns around multiples of 128 and 256."""
    import hy3_b200
    args = make(rows, n, rank, 72, out, dtype, base, runs=True)
    if n == 1:
        args[4][:] = 0
    check(hy3_b200.adapters(*args), args)


@pytest.mark.parametrize("rows,distinct", [(9, 9), (63, 2), (65, 65), (128, 1), (128, 128), (250, 3)])
def test_clusters_share_columns(cuda, rows, distinct):
    """Few and many tiles: the columns of one go to several clusters, or each cluster has all of them; an adapter's rows lie apart."""
    import torch
    import hy3_b200
    for base in ("float32", "bfloat16"):
        args = make(rows, 130, 24, 136, 5000, base=base)
        args[4][:] = (torch.arange(rows, device=cuda) * 7 % distinct) - int(distinct > 2)
        check(hy3_b200.adapters(*args), args)


@pytest.mark.parametrize("rows", [1, 8, 64, 300])
def test_an_fp32_base_gets_all_of_u(cuda, rows):
    """x picks a column of A and B one rank, so that an element is scale * A up to one product's rounding (2^-24), what three bf16 numbers leave of the
    row's largest (2^-25), and three sums of an fp32 accumulator (2^-22 each): 2^-20 of the row's largest in all, where two numbers leave 2^-18."""
    import torch
    import hy3_b200
    n, rank, width = 5, 40, 16
    x, base, a, b, ids, s = make(rows, n, rank, width, rank)
    ids[:] = torch.arange(rows, device=cuda) % n
    x[:] = torch.eye(width, device=cuda, dtype=x.dtype)[torch.arange(rows, device=cuda) % width]
    b[:] = torch.eye(rank, device=cuda, dtype=b.dtype)
    base[:] = 0
    want = s[ids.long(), None].double() * torch.einsum("trk,tk->tr", a[ids.long()].double(), x.double())
    got = hy3_b200.adapters(x, base, a, b, ids, s)
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 * want.abs().amax(1, keepdim=True)).all())
