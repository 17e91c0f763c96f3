"""What the C ABI of weights in 4 bits and of log probabilities refuses, before it touches a device, and what Python refuses of CPU tensors (runs without a GPU)."""
import pytest

P = 1 << 20          # stands for an aligned device pointer; nothing here gets as far as reading it


@pytest.fixture(scope="module")
def lib():
    import hy3_b200
    return hy3_b200.load_library()


def refused(lib, rc, text):
    assert rc == -1, rc
    message = lib.hy3a_last_error(None).decode()
    assert text in message, message


SIZES = (({"out_width": -1}, "out_width"), ({"width": 0}, "width"), ({"width": 48}, "width"), ({"width": 65568, "stride": 65568}, "width"), ({"width": -32}, "width"),
         ({"group": 0}, "group"), ({"group": 16}, "group"), ({"group": 256}, "group"), ({"group": -64}, "group"), ({"out_width": (1 << 30) + 1}, "out_width"))


def test_quantize4(lib):
    def call(w_dtype=2, out_width=8, width=64, group=64, w=P, stride=64, dtype=2, codes=P, scales=P):
        return lib.hy3a_quantize4(None, w_dtype, out_width, width, group, w, stride, dtype, codes, scales)
    for kw, text in SIZES + (({"w_dtype": 3}, "w_dtype"), ({"w_dtype": -1}, "w_dtype"), ({"dtype": 0}, "dtype"), ({"dtype": 3}, "dtype"), ({"w": None}, "NULL"), ({"codes": None}, "NULL"),
                             ({"scales": None}, "NULL"), ({"w": P + 8}, "16-byte"), ({"codes": P + 4}, "16-byte"), ({"scales": P + 1}, "aligned"), ({"stride": 68}, "boundaries"),
                             ({"w_dtype": 0, "stride": 66}, "boundaries")):
        refused(lib, call(**kw), text)
    assert call(out_width=0, w=None, codes=None, scales=None) == 0


def test_linear4(lib):
    def call(dtype=2, rows=5, width=64, out_width=8, group=64, x=P, stride=64, codes=P, scales=P, out_dtype=2, out=P, os_=8):
        return lib.hy3a_linear4(None, dtype, rows, width, out_width, group, x, stride, codes, scales, out_dtype, out, os_)
    for kw, text in SIZES + (({"dtype": 0}, "dtype"), ({"out_dtype": 1}, "out_dtype"), ({"dtype": 1}, "out_dtype"), ({"rows": -1}, "rows"), ({"rows": (1 << 24) + 1}, "rows"), ({"x": None}, "NULL"), ({"codes": None}, "NULL"),
                             ({"scales": None}, "NULL"), ({"out": None}, "NULL"), ({"x": P + 8}, "16-byte"), ({"codes": P + 8}, "16-byte"), ({"scales": P + 1}, "aligned"),
                             ({"out": P + 1}, "aligned"), ({"out_dtype": 0, "out": P + 2}, "aligned"), ({"stride": 68}, "boundaries"), ({"os_": 7}, "overlap")):
        refused(lib, call(**kw), text)
    assert call(rows=0, x=None, out=None) == 0 and call(out_width=0, codes=None, scales=None, out=None) == 0


def test_logprobs(lib):
    def call(dtype=0, rows=5, vocab=100, logits=P, stride=100, tokens=P, asked=1, top_k=3, asked_logp=P, entropy=P, ids=P, top=P):
        return lib.hy3a_logprobs(None, dtype, rows, vocab, logits, stride, tokens, asked, top_k, asked_logp, entropy, ids, top)
    for kw, text in (({"dtype": 3}, "dtype"), ({"rows": -1}, "rows"), ({"rows": (1 << 27) + 1}, "rows"), ({"vocab": 0}, "vocab"), ({"vocab": (1 << 24) + 1}, "vocab"), ({"asked": -1}, "asked"), ({"asked": 1025}, "asked"),
                     ({"top_k": -1}, "top_k"), ({"top_k": 33}, "top_k"), ({"vocab": 2}, "top_k"), ({"logits": None}, "NULL"), ({"entropy": None}, "NULL"), ({"tokens": None}, "NULL"),
                     ({"asked_logp": None}, "NULL"), ({"ids": None}, "NULL"), ({"top": None}, "NULL"), ({"logits": P + 2}, "aligned"), ({"dtype": 2, "logits": P + 1}, "aligned"),
                     ({"tokens": P + 2}, "aligned"), ({"entropy": P + 1}, "aligned"), ({"top": P + 2}, "aligned")):
        refused(lib, call(**kw), text)
    assert call(rows=0, logits=None, tokens=None, entropy=None, ids=None, top=None) == 0


def test_tensors_elsewhere_are_refused():
    """CPU tensors, types and shapes, before anything is launched."""
    import torch
    import hy3_b200
    w = torch.ones((8, 64))
    for call in (lambda: hy3_b200.quantize4(w), lambda: hy3_b200.quantize4(None), lambda: hy3_b200.quantize4(w.int()),
                 lambda: hy3_b200.linear4(w.bfloat16(), torch.zeros((8, 32), dtype=torch.uint8), w[:, :1].bfloat16()),
                 lambda: hy3_b200.logprobs(w), lambda: hy3_b200.logprobs(w, torch.zeros(8, dtype=torch.int32), top_k=2)):
        with pytest.raises((AssertionError, AttributeError)):
            call()


def test_without_a_gpu_it_says_so(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    for rc in (lib.hy3a_quantize4(None, 2, 8, 64, 64, P, 64, 2, P, P), lib.hy3a_linear4(None, 2, 1, 64, 8, 64, P, 64, P, P, 2, P, 8),
               lib.hy3a_logprobs(None, 0, 1, 100, P, 100, P, 1, 3, P, P, P, P)):
        assert rc == -3 and b"no CPU path" in lib.hy3a_last_error(None)
