"""What the C ABI of the operators beside the attention refuses, before it touches a device (runs without a GPU)."""
import pytest


@pytest.fixture(scope="module")
def lib():
    import hy3_b200
    return hy3_b200.load_library()


P = 1 << 20          # stands for an aligned device pointer; nothing here gets as far as reading it


def refused(lib, rc, text):
    assert rc == -1, rc
    message = lib.hy3a_last_error(None).decode()
    assert text in message, message


def test_route(lib):
    def call(dtype=0, rows=4, experts=192, logits=P, stride=192, bias=P, top_k=8, score=0, groups=1, top_groups=1, ids=P, weights=P):
        return lib.hy3a_route(None, dtype, rows, experts, logits, stride, bias, top_k, score, groups, top_groups, 1, 1.0, ids, weights)
    for kw, text in (({"dtype": 3}, "dtype"), ({"rows": -1}, "rows"), ({"experts": 0}, "experts"), ({"experts": 1025}, "experts"), ({"top_k": 0}, "top_k"), ({"top_k": 33}, "top_k"),
                     ({"experts": 4}, "top_k"), ({"score": 2}, "score"), ({"groups": 5}, "groups"), ({"groups": 0}, "groups"), ({"groups": 64}, "groups"),
                     ({"groups": 4, "top_groups": 5}, "top_groups"), ({"groups": 32, "top_groups": 1}, "stay"), ({"logits": None}, "NULL"), ({"ids": None}, "NULL"),
                     ({"weights": None}, "NULL"), ({"logits": P + 2}, "aligned"), ({"bias": P + 2}, "aligned"), ({"ids": P + 1}, "aligned")):
        refused(lib, call(**kw), text)
    assert call(rows=0, logits=None, ids=None, weights=None) == 0


def test_experts(lib):
    need = lib.hy3a_experts_workspace(5, 2, 64, 32, 3)
    assert need >= 5 * 2 * (64 * 4 + 32 * 2)
    assert lib.hy3a_experts_workspace(5, 2, 60, 32, 3) == 0 and lib.hy3a_experts_workspace(-1, 2, 64, 32, 3) == 0 and lib.hy3a_experts_workspace(1 << 30, 2, 64, 32, 3) == 0
    assert lib.hy3a_experts_workspace(200000, 8, 4096, 1536, 192) > 1 << 34      # sizes are counted in 64 bits

    def call(dtype=2, rows=5, top_k=2, hidden=64, inter=32, held=3, first=0, x=P, xs=64, ids=P, w=P, gate=P, up=P, down=P, out=P, os_=64, work=P, bytes_=need):
        return lib.hy3a_experts(None, dtype, rows, top_k, hidden, inter, held, first, x, xs, ids, w, gate, up, down, out, os_, work, bytes_)
    for kw, text in (({"dtype": 0}, "dtype"), ({"rows": -1}, "rows"), ({"top_k": 0}, "top_k"), ({"top_k": 33}, "top_k"), ({"hidden": 60}, "multiples"), ({"inter": 12}, "multiples"), ({"hidden": 65544, "xs": 65544}, "over"), ({"inter": 65544}, "over"), ({"rows": 1 << 27}, "many"),
                     ({"held": 0}, "held"), ({"held": 1025}, "held"), ({"first": -1}, "first_expert"), ({"first": 2 ** 31 - 2}, "first_expert"), ({"x": None}, "NULL"), ({"work": None}, "NULL"),
                     ({"x": P + 8}, "16-byte"), ({"gate": P + 2}, "16-byte"), ({"out": P + 4}, "16-byte"), ({"ids": P + 2}, "4-byte"), ({"work": P + 16}, "256-byte"), ({"xs": 68}, "strides"),
                     ({"xs": 56}, "overlap"), ({"os_": 56}, "overlap"), ({"bytes_": need - 1}, "workspace")):
        refused(lib, call(**kw), text)
    assert call(rows=0, x=None, out=None, work=None) == 0


def test_adapters(lib):
    need = lib.hy3a_adapters_workspace(5, 64, 16)
    assert need >= 5 * 16 * 4
    assert lib.hy3a_adapters_workspace(5, 64, 12) == 0 and lib.hy3a_adapters_workspace(5, 60, 16) == 0 and lib.hy3a_adapters_workspace(-1, 64, 16) == 0

    def call(dtype=2, rows=5, width=64, out_width=72, n=3, rank=16, x=P, xs=64, bt=0, base=P, bs=72, a=P, b=P, ids=P, scales=P, out=P, os_=72, work=P, bytes_=need):
        return lib.hy3a_adapters(None, dtype, rows, width, out_width, n, rank, x, xs, bt, base, bs, a, b, ids, scales, out, os_, work, bytes_)
    for kw, text in (({"dtype": 0}, "dtype"), ({"bt": 1}, "base_dtype"), ({"rows": -1}, "rows"), ({"width": 60}, "width"), ({"out_width": 12}, "out_width"), ({"width": (1 << 20) + 8}, "over"), ({"out_width": (1 << 20) + 8}, "over"), ({"n": 0}, "adapters"),
                     ({"rank": 0}, "rank"), ({"rank": 12}, "rank"), ({"rank": 264}, "rank"), ({"x": None}, "NULL"), ({"scales": None}, "NULL"), ({"x": P + 8}, "16-byte"), ({"out": P + 4}, "16-byte"),
                     ({"ids": P + 2}, "4-byte"), ({"xs": 68}, "16-byte boundaries"), ({"bs": 74}, "16-byte boundaries"), ({"os_": 64}, "overlap")):
        refused(lib, call(**kw), text)
    assert call(rows=0, x=None, base=None, out=None, work=None) == 0


def test_without_a_gpu_it_says_so(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    rc = lib.hy3a_route(None, 0, 1, 8, P, 8, None, 2, 0, 1, 1, 1, 1.0, P, P)
    assert rc == -3 and b"no CPU path" in lib.hy3a_last_error(None)
