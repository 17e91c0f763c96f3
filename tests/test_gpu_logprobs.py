"""hy3_b200.logprobs against the definition in 64 bits; ids against a stable sort.

Bounds.  With d = m - l, S = sum of e^-d of the logits below the maximum, T = sum of d e^-d, Z = n + S, all relative errors of
    an exponential: 2^-22 + d 2^-23 (its function, its argument); of a step that raises m: the same with the rise, and no more steps than a thread has turns;
    sums: 2^-24 for each of a thread's logits, 64 for where threads meet.
An exponential below 2^-126, the smallest normal number, counts as 0: that is vocab 2^-126 of S at most, and 200 times as much of T (d counts up to 200).
R is the range of the open logits, no more than 100 of which counts (e^-100 is nothing beside 1)."""
import pytest

pytestmark = pytest.mark.gpu


def reference(logits, tokens, top_k):
    import torch
    l = logits.double()
    m = l.amax(-1, keepdim=True)
    none = m == -float("inf")
    d = torch.where(l == -float("inf"), 1000.0, torch.where(none, 1000.0, m - l))
    e = torch.exp(-d)
    n = (d == 0).sum(-1, keepdim=True)
    S, T, = torch.where(d > 0, e, 0.0).sum(-1, keepdim=True), (e * d).sum(-1, keepdim=True)
    Z = n + S
    log_z = torch.where(n == 1, torch.log1p(S), torch.log(Z.clamp(min=1)))
    logp = torch.where(l == -float("inf"), -float("inf"), -d - log_z)
    entropy = torch.where(none, 0.0, log_z + T / Z.clamp(min=1e-300))
    vocab, turns = l.shape[1], l.shape[1] // 16384 + 1
    R = d.masked_fill(d == 1000, 0).amax(-1, keepdim=True).clamp(max=100)
    rel = 2.0 ** -22 * (1 + T / S.clamp(min=1e-300) + turns + 8 + R) + (vocab / 512 + 64) * 2.0 ** -24
    err_z = rel * S / Z.clamp(min=1e-300) + 2.0 ** -22 * log_z + vocab * 2.0 ** -126
    err = err_z + 2.0 ** -23 * (d.clamp(max=1000) + logp.abs().nan_to_num(posinf=0))
    err_h = err_z + (rel + 2.0 ** -23 * R) * T / Z.clamp(min=1e-300) + 2.0 ** -22 * entropy + 200 * vocab * 2.0 ** -126
    order = torch.sort(l + 0.0, dim=-1, descending=True, stable=True).indices[:, :top_k]
    top = logp.gather(1, order)
    ids = torch.where(top == -float("inf"), -1, order)
    asked = None
    if tokens is not None:
        at = tokens.long().view(l.shape[0], -1)
        asked = (torch.where(at < 0, 0.0, logp.gather(1, at.clamp(min=0))), torch.where(at < 0, 0.0, err.gather(1, at.clamp(min=0))))
    return asked, (entropy.squeeze(1), err_h.squeeze(1)), ids, (top, err.gather(1, order))


def near(got, want):
    import torch
    value, limit = want
    value = value.view(got.shape)
    same = got == value.float()         # (what is too far for fp32 is -inf)
    far = (got.double() - value).abs() <= limit.view(got.shape)
    assert got.dtype == torch.float32 and bool((same | far).all()), "off by %.3g" % float((got.double() - value).abs().nan_to_num().max())


def check(logits, tokens, top_k):
    import torch
    import hy3_b200
    asked, entropy, ids, top = hy3_b200.logprobs(logits, tokens, top_k)
    want_asked, want_entropy, want_ids, want_top = reference(logits, tokens, top_k)
    if tokens is None:
        assert asked is None
    else:
        assert asked.shape == tokens.shape
        near(asked, want_asked)
    near(entropy, want_entropy)
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want_ids)
    near(top, want_top)
    return asked, entropy, ids, top


def make(rows, vocab, dtype="float32", asked=1, closed=0.0, seed=0, scale=3.0, device="cuda"):
    import torch
    gen = torch.Generator(device=device).manual_seed(seed + rows * 3 + vocab)
    logits = scale * torch.randn((rows, vocab), device=device, generator=gen)
    if closed:
        logits[torch.rand(logits.shape, device=device, generator=gen) < closed] = -float("inf")
    tokens = torch.randint(-1, vocab, (rows, asked), device=device, generator=gen).to(torch.int32)
    return logits.to(getattr(torch, dtype)), tokens


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (1, 2, 2), (3, 5, 3), (2, 33, 32), (7, 100, 0), (1, 1000, 20), (5, 4099, 5), (1, 32003, 1), (1, 120832, 20), (2, 151936, 32), (40, 32003, 5), (100, 9001, 32),
                                              (150, 16385, 1), (333, 32003, 20), (700, 129, 8), (33, 120832, 0),
                                              (1, 2049, 3), (60, 4001, 7), (700, 4096, 20), (1500, 2051, 32), (900, 8191, 1), (160, 60001, 32), (20, 250001, 16), (200, 9001, 32), (700, 20001, 31), (1000, 77, 30), (300, 40, 32)])
def test_sizes(cuda, rows, vocab, top_k, dtype):
    check(*make(rows, vocab, dtype, asked=3), top_k)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 50, 400])
def test_closed_tokens(cuda, rows, dtype):
    """Most tokens closed, fewer open ones than asked for, one, none."""
    for closed in (0.9, 0.999):
        check(*make(rows, 20011, dtype, closed=closed), 20)
    logits, tokens = make(rows, 5003, dtype)
    logits[:] = -float("inf")
    logits[0, 4999] = 2.5
    tokens[0] = 4999
    asked, entropy, ids, top = check(logits, tokens, 3)
    assert asked[0] == 0 and entropy[0] == 0 and ids[0].tolist() == [4999, -1, -1] and top[0, 0] == 0
    logits[:] = -float("inf")
    asked, entropy, ids, top = check(logits, tokens, 3)
    assert asked[0] == -float("inf") and (entropy == 0).all() and (ids == -1).all() and (top == -float("inf")).all()


@pytest.mark.parametrize("rows", [1, 60, 300])
def test_equal_logits(cuda, rows):
    """All alike, many alike at the border of the top, both zeros: the lowest index is first."""
    import torch
    logits, tokens = make(rows, 30011)
    check(torch.zeros_like(logits), tokens, 20)
    check(logits.round().clamp(-2, 2), tokens, 20)
    check((logits * 4).round() / 4, tokens, 32)
    zeros = torch.zeros_like(logits)
    zeros[:, ::2] = -0.0
    check(zeros, tokens, 5)
    check(torch.full_like(logits, -3e38), tokens, 4)
    steps = torch.arange(30011, device=cuda, dtype=torch.float32)
    check((steps / 1000).expand(rows, -1).contiguous(), tokens, 20)
    check((-steps / 1000).expand(rows, -1).contiguous(), tokens, 20)
    # the largest are all in one thread's vectors
    for period in (2048, 4096, 8192):
        logits = torch.randn((rows, 120003), device=cuda)
        logits[:, 5::period] += 20
        check(logits, tokens, 20)


@pytest.mark.parametrize("gap", [2.0, 10.0, 16.0, 40.0, 90.0, 300.0])
def test_a_token_that_is_nearly_certain(cuda, gap):
    """Its log probability is a small number, and has its digits all the same."""
    import torch
    logits, tokens = make(6, 5001, scale=0.5)
    at = torch.tensor([0, 1, 5000, 77, 2500, 4096], device=cuda)
    logits[torch.arange(6), at] = logits.max(1).values + gap
    tokens[:, 0] = at.int()
    check(logits, tokens, 2)


def test_far_apart_and_far_from_zero(cuda):
    import torch
    logits, tokens = make(20, 3001)
    check(logits * 1e4, tokens, 8)
    check(logits + 1e6, tokens, 8)
    check(logits - 3e38, tokens, 8)
    check(torch.where(logits > 0, 3e38, -3e38), tokens, 2)
    check(logits * 1e-30, tokens, 8)
    check(logits.half() * 1000, tokens, 8)


@pytest.mark.parametrize("rows", [1, 400])
def test_what_is_not_finite_stays_in_its_row(cuda, rows):
    import torch
    import hy3_b200
    inf, nan = float("inf"), float("nan")
    logits, tokens = make(rows + 4, 20011)
    tokens[:4] = 7
    logits[0, 100] = nan
    logits[1, 100] = inf
    logits[2, :] = nan
    logits[3, :] = -inf
    logits[3, 11] = nan
    logits[1, 50:60] = -inf
    asked, entropy, ids, top = hy3_b200.logprobs(logits, tokens, 4)
    assert torch.isnan(asked[:4]).all() and torch.isnan(entropy[:4]).all()
    assert torch.isnan(top[:3]).all() and torch.isnan(top[3, 0])
    assert ids[1, 0] == 100 and ids[2].tolist() == [0, 1, 2, 3] and ids[3].tolist() == [11, -1, -1, -1]
    finite = logits[0].nan_to_num(nan=-3.4e38)
    assert torch.equal(ids[0].long(), torch.sort(finite, descending=True, stable=True).indices[:4])
    rest = hy3_b200.logprobs(logits[4:].contiguous(), tokens[4:].contiguous(), 4)
    want = reference(logits[4:], tokens[4:], 4)
    near(asked[4:], want[0])
    assert torch.equal(ids[4:].long(), want[2]) and torch.equal(rest[2], ids[4:])


def test_tokens(cuda):
    import torch
    import hy3_b200
    logits, _ = make(5, 1001)
    tokens = torch.tensor([-1, 0, 1000, 1001, -2], dtype=torch.int32, device=cuda)
    asked = hy3_b200.logprobs(logits, tokens)[0]
    assert asked.shape == (5,) and asked[0] == 0 and torch.isnan(asked[3:]).all()
    many = torch.arange(1001, device=cuda, dtype=torch.int32).expand(5, -1).contiguous()
    got = hy3_b200.logprobs(logits, many[:, :1000].contiguous())[0]
    near(got, tuple(t[:, :] for t in reference(logits, many[:, :1000], 0)[0]))
    assert torch.equal(got[1, 0], asked[1])
    # log probabilities of all tokens are those of a distribution
    assert abs(float(got.double().exp().sum(1)[0]) + float(hy3_b200.logprobs(logits, many[:, 1000].contiguous())[0].double().exp()[0]) - 1) < 1e-5


def test_strides_and_boundaries(cuda):
    """Rows that start on any boundary of the type, rows of a wider matrix whose other values are NaN, one row for all."""
    import torch
    import hy3_b200
    for dtype in ("float32", "bfloat16", "float16"):
        for shift in range(0, 9):
            logits, tokens = make(9, 2011, dtype)
            wide = torch.full((9, 2077), float("nan"), dtype=logits.dtype, device=cuda)
            wide[:, shift:shift + 2011] = logits
            got = hy3_b200.logprobs(wide[:, shift:shift + 2011], tokens, 5)
            want = reference(logits, tokens, 5)
            near(got[0], want[0])
            near(got[1], want[1])
            assert torch.equal(got[2].long(), want[2])
            one = wide[2:3, shift:shift + 2011].expand(4, -1)
            assert torch.equal(hy3_b200.logprobs(one, top_k=3)[2], got[2][2, :3].expand(4, -1))


def test_no_rows_a_stream_a_graph_and_repeatable_bits(cuda):
    import torch
    import hy3_b200
    logits, tokens = make(300, 32003)
    assert [t.shape for t in hy3_b200.logprobs(logits[:0], tokens[:0], 3)] == [(0, 1), (0,), (0, 3), (0, 3)]
    for n in (1, 20, 300):
        other, _ = make(n, 32003, seed=4)
        part, which = logits[:n].clone(), tokens[:n].clone()
        want = hy3_b200.logprobs(part, which, 7)
        then = hy3_b200.logprobs(other, which, 7)
        for _ in range(10):
            assert all(torch.equal(a, b) for a, b in zip(hy3_b200.logprobs(part, which, 7), want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = hy3_b200.logprobs(part, which, 7)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = hy3_b200.logprobs(part, which, 7)
        part.copy_(other)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, then))


def test_refusals(cuda):
    import torch
    import hy3_b200
    logits, tokens = make(4, 100)
    for bad in (lambda: hy3_b200.logprobs(logits.double()), lambda: hy3_b200.logprobs(logits.T), lambda: hy3_b200.logprobs(logits[0]), lambda: hy3_b200.logprobs(logits, tokens.long()),
                lambda: hy3_b200.logprobs(logits, tokens[:3]), lambda: hy3_b200.logprobs(logits, tokens.cpu()), lambda: hy3_b200.logprobs(logits, tokens.view(2, 2))):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: hy3_b200.logprobs(logits, top_k=33), lambda: hy3_b200.logprobs(logits, top_k=-1), lambda: hy3_b200.logprobs(logits[:, :3], top_k=4), lambda: hy3_b200.logprobs(logits[:, :0])):
        with pytest.raises(hy3_b200.Hy3AttnError):
            bad()
    logits.requires_grad_()
    with pytest.raises(AssertionError, match="grad"):
        hy3_b200.logprobs(logits)
    with torch.no_grad():
        hy3_b200.logprobs(logits)
