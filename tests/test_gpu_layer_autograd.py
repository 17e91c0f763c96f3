"""The operators beside the attention compute no gradients: a call that one would be asked of is refused, and what is written into `out` counts as a change."""
import pytest

pytestmark = pytest.mark.gpu


def calls(device):
    import torch
    import hy3_b200

    def t(*shape, dtype=torch.bfloat16):
        return torch.ones(shape, dtype=dtype, device=device)
    ids = torch.zeros((4, 2), dtype=torch.int32, device=device)
    return [
        ("route", lambda l, b: hy3_b200.route(l, b, top_k=2), [t(4, 16, dtype=torch.float32), t(16, dtype=torch.float32)]),
        ("experts", lambda x, w, g, u, d: hy3_b200.experts(x, ids, w, g, u, d), [t(4, 64), t(4, 2, dtype=torch.float32), t(3, 32, 64), t(3, 32, 64), t(3, 64, 32)]),
        ("adapters", lambda x, y, a, b, s: hy3_b200.adapters(x, y, a, b, ids[:, 0].contiguous(), s), [t(4, 64), t(4, 72), t(3, 16, 64), t(3, 72, 16), t(3, dtype=torch.float32)]),
    ]


def test_inputs_that_want_gradients(cuda):
    import torch
    for name, call, args in calls(cuda):
        call(*args)
        for i, arg in enumerate(args):
            arg.requires_grad_()
            with pytest.raises(AssertionError, match=name + ".*grad"):
                call(*args)
            with torch.no_grad():
                got = call(*args)
            with torch.inference_mode():
                call(*args)
            assert not any(g.requires_grad for g in (got if isinstance(got, tuple) else (got,)))
            arg.requires_grad_(False)


def test_what_is_written_into_out_is_a_change(cuda):
    """A value that autograd keeps for a backward pass and that a call overwrites is noticed there."""
    import torch
    import hy3_b200
    ids = torch.zeros((4, 2), dtype=torch.int32, device=cuda)
    one = lambda *shape: torch.ones(shape, dtype=torch.bfloat16, device=cuda)  # noqa: E731
    for call, width in ((lambda out: hy3_b200.experts(one(4, 64), ids, torch.ones((4, 2), device=cuda), one(3, 32, 64), one(3, 32, 64), one(3, 64, 32), out=out), 64),
                        (lambda out: hy3_b200.adapters(one(4, 64), one(4, 72), one(3, 16, 64), one(3, 72, 16), ids[:, 0].contiguous(), torch.ones(3, device=cuda), out=out), 72)):
        kept, leaf = one(4, width), torch.ones((4, width), dtype=torch.bfloat16, device=cuda, requires_grad=True)
        product = (kept * leaf).sum()
        call(kept)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()
        with pytest.raises(AssertionError, match="grad"):
            call(leaf)
        with torch.inference_mode():
            assert call(one(4, width)).shape == (4, width)
