"""Log probabilities of tokens, entropies and strongest alternatives against 64 bits.

Bounds: a weight e^(x - m) is off by 2^-21 (the exponential, its argument's rounding at the sizes that count), a thread adds V / 256
of them one after another and 64 partial sums follow, each addition off by 2^-24: so the sum's logarithm by
off = 2^-21 + (V / 256 + 64) 2^-24, and a log probability by 2^-23 of itself and of its largest term more.  An entropy has that
error on the sum and on the mean of x - m."""
import math

import pytest
import torch

from if_i_could_turn_back_time_b200 import _lib, ops

DEV = "cuda"
gpu = pytest.mark.gpu


def _check(x, tokens, got, top):
    vocab = x.shape[-1]
    off = 2.0 ** -21 + (vocab / 256 + 64) * 2.0 ** -24
    lp = torch.log_softmax(x.double(), -1)
    lp = torch.where(torch.isneginf(x).all(-1, keepdim=True), -math.inf, lp)
    largest = x.double().masked_fill(torch.isinf(x), 0).abs().amax(-1)

    def near(a, b, tol):
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        fine = torch.isfinite(b)
        assert bool(((a.double() - b).abs()[fine] <= tol.expand_as(b)[fine]).all()), ((a.double() - b).abs() / tol)[fine].max().item()

    want = lp.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]
    want = torch.where(tokens < 0, 0.0, torch.where(tokens >= vocab, math.nan, want))
    near(got.logprob, want, off + 2.0 ** -22 * (want.abs().nan_to_num(0, 0, 0) + largest))
    d = (x.double() - x.double().amax(-1, keepdim=True)).abs().nan_to_num(0, 0, 0)
    p = lp.exp()
    want = torch.special.entr(p).sum(-1)
    near(got.entropy, want, 2 * off * (1 + (p.nan_to_num(0) * d).sum(-1)) + 2.0 ** -22 * (want.abs() + 1) + 0 * largest)
    assert got.top_logprobs.shape == got.top_tokens.shape == (x.shape[0], top)
    if top:
        clean = ~torch.isnan(x).any(-1)
        order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_tokens[clean], order[clean])
        assert bool(((got.top_tokens >= 0) & (got.top_tokens < vocab)).all())
        want = lp.gather(1, got.top_tokens)
        near(got.top_logprobs, want, (off + 2.0 ** -22 * (want.abs().nan_to_num(0, 0, 0) + largest[:, None])))


CASES = [(rows, vocab, dtype, top) for rows, vocab, top in (
    (1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 31, 31), (4, 32, 32), (7, 33, 5), (1, 2047, 32), (1, 2049, 20), (3, 32000, 5), (9, 50001, 20),
    (600, 333, 8), (700, 4099, 0), (593, 2500, 32), (2, 131072, 1), (1, 70000, 0)) for dtype in (torch.float32, torch.float16, torch.bfloat16)]


@gpu
@pytest.mark.parametrize("rows,vocab,dtype,top", CASES)
def test_against_64_bits(rows, vocab, dtype, top):
    gen = torch.Generator(DEV).manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, device=DEV, generator=gen) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=gen)
    got = ops.token_logprobs(x, tokens, top)
    _check(x, tokens, got, top)
    again = ops.token_logprobs(x, tokens, top)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    if top:
        plain = ops.token_logprobs(x, tokens)
        assert plain.top_tokens.shape == (rows, 0)
        _check(x, tokens, plain, 0)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 650])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_that_go_wrong(rows, dtype):
    vocab, top = 5003, 20
    gen = torch.Generator(DEV).manual_seed(2)
    x = torch.randn(rows, vocab, device=DEV, generator=gen).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=gen)
    lowest = torch.finfo(dtype).min
    kinds = {
        "equal": lambda t: t.fill_(1.5),
        "rising": lambda t: t.copy_(torch.arange(vocab, device=DEV).float().mul(0.002)),
        "falling": lambda t: t.copy_(torch.arange(vocab, device=DEV).float().mul(-0.002)),
        "few": lambda t: t[:, 7:].fill_(-math.inf),
        "one": lambda t: (t[:, :4000].fill_(-math.inf), t[:, 4001:].fill_(-math.inf)),
        "nothing": lambda t: t.fill_(-math.inf),
        "lowest": lambda t: t[:, ::2].fill_(lowest),
        "only lowest": lambda t: t.fill_(lowest),
        "highest": lambda t: t[:, 3].fill_(torch.finfo(dtype).max),
        "zeros": lambda t: (t.zero_(), t[:, ::3].neg_()),
        "nan": lambda t: t[:, 4999].fill_(math.nan),
        "infinity": lambda t: t[:, 12].fill_(math.inf),
    }
    for change in kinds.values():
        y = x.clone()
        change(y)
        _check(y, tokens, ops.token_logprobs(y, tokens, top), top)
        mixed = x.clone()                                          # one such row among others
        change(mixed[rows // 2:rows // 2 + 1])
        got = ops.token_logprobs(mixed, tokens, top)
        _check(mixed, tokens, got, top)
    got = ops.token_logprobs(torch.full((rows, vocab), -math.inf, device=DEV, dtype=dtype), tokens, 3)
    assert torch.isneginf(got.logprob).all() and bool((got.entropy == 0).all()) and got.top_tokens[0].tolist() == [0, 1, 2]


@gpu
def test_tokens_that_are_none_or_not_there():
    x = torch.randn(6, 100, device=DEV)
    tokens = torch.tensor([-1, -100, 0, 99, 100, 2 ** 40], device=DEV)
    got = ops.token_logprobs(x, tokens, 2)
    _check(x, tokens, got, 2)
    assert got.logprob[:2].tolist() == [0, 0] and torch.isnan(got.logprob[4:]).all() and torch.isfinite(got.entropy).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_leading_dims_streams_and_graphs(dtype):
    raw = torch.randn(2, 9, 4500, device=DEV).to(dtype)
    for x in (raw[:, :, 1:4001], raw[:, ::2, 3:3330], raw[:1].expand(3, 9, 4500)[:, :, 7:], raw.transpose(1, 2)[..., :5]):
        tokens = torch.randint(0, x.shape[-1], x.shape[:-1], device=DEV)
        got = ops.token_logprobs(x, tokens, 4)
        assert got.logprob.shape == x.shape[:-1] and got.top_tokens.shape == (*x.shape[:-1], 4)
        flat = ops.TokenLogprobs(got.logprob.reshape(-1), got.entropy.reshape(-1), got.top_logprobs.reshape(-1, 4), got.top_tokens.reshape(-1, 4))
        _check(x.reshape(-1, x.shape[-1]), tokens.reshape(-1), flat, 4)
    x, tokens = raw[0, 0], torch.tensor(17, device=DEV)
    assert ops.token_logprobs(x, tokens, 2).top_logprobs.shape == (2,)
    x, tokens = raw[0].contiguous(), torch.arange(9, device=DEV)
    want = ops.token_logprobs(x, tokens, 5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.token_logprobs(x, tokens, 5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = ops.token_logprobs(x, tokens, 5)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for seed in range(3):
        x.copy_(torch.randn(x.shape, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        _check(x, tokens, held, 5)
    empty = ops.token_logprobs(raw[:0, 0], tokens[:0], 3)
    assert empty.top_tokens.shape == (0, 3)


@gpu
def test_calls_of_any_size_follow_one_another():
    """They share one buffer, with attention over the cache too: what a call leaves in it does not reach the next."""
    gen = torch.Generator(DEV).manual_seed(4)
    for rows, vocab in ((1, 100000), (500, 5000), (3, 20000), (590, 4100), (2, 131072), (64, 32000)):
        x = torch.randn(rows, vocab, device=DEV, generator=gen)
        tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=gen)
        _check(x, tokens, ops.token_logprobs(x, tokens, 20), 20)


@gpu
def test_offsets_past_32_bits():
    x = torch.zeros(40000, 65536, dtype=torch.bfloat16, device=DEV)          # 2.6e9 elements
    x[-2:] = torch.randn(2, 65536, device=DEV).bfloat16()
    tokens = torch.full((40000,), 5, device=DEV)
    got = ops.token_logprobs(x, tokens, 2)
    _check(x[-2:], tokens[-2:], ops.TokenLogprobs(*(t[-2:] for t in got)), 2)
    assert bool(((got.logprob[:-2] + math.log(65536)).abs() < 1e-4).all())


def test_refusals():
    lib, p = _lib.load(), 1 << 20
    call = lambda x=p, rows=2, vocab=5000, dtype=0, tokens=p, lp=p, top=3, tl=p, tt=p, ws=p, size=1 << 40, stride=5000: lib.jq_token_logprobs(     # noqa: E731
        x, stride, rows, vocab, dtype, tokens, lp, p, top, tl, tt, ws, size, None)
    assert call(x=None) == -1 and call(tokens=None) == -1 and call(lp=None) == -1 and call(tl=None) == -1 and call(tt=None) == -1
    assert call(rows=-1) == -2 and call(vocab=0) == -2 and call(top=33) == -2 and call(top=-1) == -2 and call(vocab=2, top=3) == -2
    assert call(dtype=3) == -4 and call(x=p + 2) == -3 and call(tokens=p + 4) == -3 and call(ws=p + 8) == -3 and call(stride=-1) == -2
    assert call(ws=None) == -1 and call(size=100) == -6 and call(vocab=(1 << 30) + 1) == -2
    assert call(rows=0) == 0
    x, tokens = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for args, text in (((x, tokens), "CUDA"), ((x, tokens.int()), "int64"), ((x, tokens[:1]), "int64"), ((x.double(), tokens), "dtype"),
                       ((x[:, :0], tokens), "one token"), ((x, tokens, 11), "top"), ((x, tokens, -1), "top")):
        with pytest.raises(RuntimeError, match=text):
            ops.token_logprobs(*args)


@pytest.mark.parametrize("rows,vocab", [(2, (1 << 32) + 10), (2, (1 << 30) + 1), ((1 << 32) + 2, 10), (1 << 31, 3)])
def test_sizes_past_32_bits_are_refused(rows, vocab):
    """(The library's counts have 32 bits: a vocabulary of 2^32 + 10 would be one of 10.)"""
    x, tokens = torch.zeros(1, 1).expand(rows, vocab), torch.zeros(1, dtype=torch.int64).expand(rows)
    with pytest.raises(RuntimeError, match="rows of"):
        ops.token_logprobs(x, tokens, 3)
