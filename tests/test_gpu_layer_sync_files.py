"""hy3_b200.layer_sync reads and clears what every file reports: nothing is left for the next call."""
import threading

import pytest

pytestmark = pytest.mark.gpu


def wait_out(*which):
    import torch
    import hy3_b200
    for w in which:
        assert hy3_b200.load_library().hy3a_layer_wait_out(torch.cuda.current_stream().cuda_stream, w) == 0


@pytest.mark.parametrize("which,name,where", [((5,), "linear4", 69), ((4, 5), "linear4", 49), ((5, 4), "linear4", 49), ((0, 1, 4, 5), "experts", 29), ((1, 5), "adapters", 39)])
def test_reported_once_and_all_cleared(cuda, which, name, where):
    import hy3_b200
    from test_gpu_linear4 import check, make
    hy3_b200.layer_sync()
    wait_out(*which)
    with pytest.raises(hy3_b200.Hy3AttnError, match="%s: .*where %d\\)" % (name, where)) as e:
        hy3_b200.layer_sync()
    assert e.value.code == -6
    args = make(40, 512, 300)
    check(hy3_b200.linear4(*args[:3]), *args)
    hy3_b200.layer_sync()


def test_two_threads_on_streams_of_their_own(cuda):
    """Each wait that ran out is reported to exactly one of the calls."""
    import torch
    import hy3_b200
    hy3_b200.layer_sync()
    wait_out(5)
    torch.cuda.synchronize()
    seen = []

    def ask():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                try:
                    hy3_b200.layer_sync()
                except hy3_b200.Hy3AttnError as e:
                    seen.append(e.code)

    threads = [threading.Thread(target=ask) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen == [-6]
