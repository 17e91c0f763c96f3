"""hy3_b200.layer_sync reports a device-side wait that ran out, once, and calls after it work."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which,name", [(0, "experts"), (1, "adapters")])
def test_a_wait_that_ran_out_is_reported_once(cuda, which, name):
    import torch
    import hy3_b200
    from test_gpu_experts import check, make
    hy3_b200.layer_sync()
    assert hy3_b200.load_library().hy3a_layer_wait_out(torch.cuda.current_stream().cuda_stream, which) == 0
    with pytest.raises(hy3_b200.Hy3AttnError, match=name) as e:
        hy3_b200.layer_sync()
    assert e.value.code == -6
    hy3_b200.layer_sync()
    args = make(50, 6, 2, 256, 136)
    check(hy3_b200.experts(*args), args)
    hy3_b200.layer_sync()


def test_refusals(cuda):
    import hy3_b200
    assert hy3_b200.load_library().hy3a_layer_wait_out(None, 2) == -1
