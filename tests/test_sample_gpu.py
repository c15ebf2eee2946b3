"""tsb.sample against the 64-bit oracle. Tokens are equal; a row may differ only
where u lies within 1e-9 of the border between two shares (2^-42 per token, of at
most 2^20 tokens, is 2.4e-7 of the largest weight in the worst case and 1e-9
where the roundings of the tokens do not all point the same way; the inputs are
fixed and no row here comes that near). Log probabilities are rounded once to
float32, half a step 2^-24, over a 64-bit value off by the same sums."""

import numpy as np
import pytest
import torch

from oracle import verify as oracle

pytestmark = pytest.mark.gpu


def _check(x, u, got, **params):
    tokens, logprobs = (t.cpu().numpy() for t in got)
    xs, us = x.double().cpu().numpy(), u.cpu().numpy()
    for r in range(len(us)):
        row = {k: float(v[r]) if isinstance(v, torch.Tensor) else v for k, v in params.items()}
        row["top_k"] = int(row.get("top_k", 0))
        token, logprob, margin = oracle.sample(xs[r], us[r], **row)
        if margin > 1e-9:
            assert tokens[r] == token, (r, row, us[r], margin)
        if tokens[r] == token and token >= 0:
            assert abs(logprobs[r] - logprob) <= 2.0**-23 * abs(logprob) + 3e-7, (r, logprobs[r], logprob)
        elif token < 0:
            assert tokens[r] == -1 and np.isneginf(logprobs[r])


def _logits(rows, vocab, dtype, seed, peaks=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 2 * torch.randn(rows, vocab, device="cuda", generator=g)
    if peaks:
        at = torch.randint(0, vocab, (rows, 16), device="cuda", generator=g)
        x.scatter_reduce_(1, at, 6 + 6 * torch.rand(rows, 16, device="cuda", generator=g), "amax")
    return x.to(dtype), torch.rand(rows, device="cuda", generator=g)


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 2), (3, 31), (5, 1000), (4, 4097), (33, 5003), (2, 70001)])
@pytest.mark.parametrize("params", [
    {}, {"temperature": 0.0}, {"temperature": 0.7, "top_k": 50, "top_p": 0.95}, {"temperature": 1.5, "top_p": 0.6},
    {"top_k": 1}, {"min_p": 0.05}, {"temperature": 0.8, "top_k": 700, "top_p": 0.99, "min_p": 0.001},
    {"temperature": 100.0}, {"temperature": 1e-3}, {"top_p": 1e-6}, {"top_p": 0.999999}, {"min_p": 1.0},
], ids=lambda p: ",".join(f"{k}={v}" for k, v in p.items()) or "plain")
def test_against_64_bits(dtype, rows, vocab, params):
    import tsb

    x, u = _logits(rows, vocab, dtype, seed=rows * 7 + vocab)
    _check(x, u, tsb.sample(x, u, logprobs=True, **params), **params)


@pytest.mark.parametrize("dtype", DTYPES)
def test_flat_rows(dtype):
    """No peaks and a high temperature: tens of thousands of tokens share the weight."""
    import tsb

    x, u = _logits(9, 50021, dtype, seed=1, peaks=False)
    for params in ({"temperature": 3.0}, {"temperature": 3.0, "top_k": 30000}, {"temperature": 3.0, "top_p": 0.9},
                   {"temperature": 3.0, "top_k": 40000, "top_p": 0.97, "min_p": 0.01}):
        _check(x, u, tsb.sample(x, u, logprobs=True, **params), **params)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parameters_per_row(dtype):
    import tsb

    rows = 64
    x, u = _logits(rows, 3001, dtype, seed=2)
    g = torch.Generator().manual_seed(3)
    pick = lambda v, dt: torch.tensor(v, dtype=dt)[torch.randint(0, len(v), (rows,), generator=g)].cuda()  # noqa: E731
    params = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 7, 300, 9999], torch.int32),
                  top_p=pick([1.0, 0.9, 0.3], torch.float32), min_p=pick([0.0, 0.02, 0.5], torch.float32))
    _check(x, u, tsb.sample(x, u, logprobs=True, **params), **params)
    wide = dict(params, temperature=params["temperature"].double(), top_k=params["top_k"].long())
    assert all(torch.equal(a, b) for a, b in zip(tsb.sample(x, u, logprobs=True, **params), tsb.sample(x, u, logprobs=True, **wide)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dtype):
    import tsb

    vocab = 4099
    x = torch.zeros(6, vocab, dtype=dtype, device="cuda")
    x[1, ::2] = -0.0                       # -0 and +0 are the same logit
    x[2] = torch.arange(vocab, device="cuda").remainder(3).to(dtype)
    x[3, 100:] = 5.0
    x[4] = -torch.inf
    x[4, 7::100] = 1.0
    x[5] = 3.0
    for value in (0.0, 0.2, 0.5, 0.75, 0.99999994):
        u = torch.full((6,), value, device="cuda")
        for params in ({}, {"top_k": 5}, {"top_p": 0.5}, {"temperature": 0.0}, {"top_k": 4000, "top_p": 0.25}):
            got = tsb.sample(x, u, logprobs=True, **params)
            xs = x.double().cpu().numpy()
            for r in range(6):
                name = ("temperature", "top_k", "top_p")
                filters = [params.get(k, d) for k, d in zip(name, (1.0, 0, 1.0))]
                if r in (2, 3):  # several logits, each many times
                    token, _, margin = oracle.sample(xs[r], value, *filters)
                    assert margin < 1e-9 or int(got[0][r]) == token, (r, value, params)
                    continue
                # equal shares: the borders are whole numbers of tokens, compared exactly
                order, _ = oracle.filtered(xs[r], *filters)
                want = order[min(int(np.floor(np.float64(np.float32(value)) * len(order))), len(order) - 1)]
                assert int(got[0][r]) == want, (r, value, params)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_nan_logits(dtype):
    import tsb

    inf, nan = float("inf"), float("nan")
    x, u = _logits(8, 2000, dtype, seed=4)
    x[0] = -inf                                   # nothing to choose
    x[1] = nan
    x[2] = -inf; x[2, 1234] = -3.0                # one token left
    x[3, 5] = inf                                 # takes all the weight
    x[4, ::3] = nan                               # never chosen
    x[5, 1:] = torch.finfo(dtype).min             # a mask of the type's lowest value
    x[6, ::2] = -inf
    x[7] = torch.finfo(dtype).min                 # all lowest: equal shares
    for params in ({}, {"top_k": 10, "top_p": 0.9}, {"temperature": 0.0}, {"min_p": 0.1}):
        got = tsb.sample(x, u, logprobs=True, **params)
        _check(x, u, got, **params)
        assert got[0][0] == -1 and got[0][1] == -1 and got[0][2] == 1234 and got[0][3] == 5 and got[0][5] == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens_of_nearly_one_logit(dtype):
    """More tokens in a narrow band than can be listed: equal ones, and neighbours that differ in the last bits."""
    import tsb

    vocab = 60013
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(4, vocab, device="cuda", generator=g)
    x[0, ::2] = 4.0                                                # one tie of 30000 above the rest
    x[1] = 1.0 + 1e-3 * torch.rand(vocab, device="cuda", generator=g)
    x[2] = torch.randint(0, 3, (vocab,), device="cuda", generator=g).float()
    x[3, 1000:] = -60.0                                            # tokens with hardly any weight
    x = x.to(dtype)
    for value in (0.0, 0.3, 0.77, 0.999999):
        u = torch.full((4,), value, device="cuda")
        for params in ({}, {"top_k": 5000}, {"top_k": 50000, "top_p": 0.6}, {"top_p": 0.9, "min_p": 0.02}, {"temperature": 0.3}):
            _check(x, u, tsb.sample(x, u, logprobs=True, **params), **params)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 1 << 20), (torch.float32, (1 << 20) - 3), (torch.bfloat16, 700001)])
def test_the_largest_vocabularies(dtype, vocab):
    import tsb

    x, u = _logits(2, vocab, dtype, seed=12)
    for params in ({}, {"temperature": 0.7, "top_k": 50, "top_p": 0.95}, {"top_k": 5000, "top_p": 0.9}):
        _check(x, u, tsb.sample(x, u, logprobs=True, **params), **params)
    assert tsb.sample(torch.zeros(1, (1 << 20) + 1, dtype=dtype, device="cuda"), u[:1]) is None


def test_random_numbers_at_and_past_the_ends():
    import tsb

    x, _ = _logits(6, 999, torch.float32, seed=5)
    order = x.argsort(-1, descending=True)
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, float("nan"), 1e-45], device="cuda")
    tokens = tsb.sample(x, u, top_k=3)
    assert tokens.tolist() == [int(order[r, c]) for r, c in enumerate([0, 0, 2, 2, 0, 0])]


def test_parameters_that_are_off():
    import tsb

    x, u = _logits(16, 777, torch.bfloat16, seed=6)
    want = tsb.sample(x, u, logprobs=True)
    for params in ({"top_k": -3}, {"top_k": 777}, {"top_k": 10**9}, {"top_p": 1.5}, {"top_p": float("nan")}, {"min_p": -1.0},
                   {"min_p": float("nan")}):
        assert all(torch.equal(a, b) for a, b in zip(tsb.sample(x, u, logprobs=True, **params), want))
    greedy = tsb.sample(x, u, temperature=0.0)
    for t in (-1.0, float("nan")):
        assert torch.equal(tsb.sample(x, u, temperature=t), greedy)
    assert torch.equal(tsb.sample(x, u, min_p=7.0), greedy)        # only the first is left
    assert torch.equal(tsb.sample(x, u, top_p=0.0), greedy)
    hot = tsb.sample(x, u, temperature=float("inf"))               # equal shares, in order of the logits
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1]
    at = (u.double() * 777).long()
    assert torch.equal(hot.long(), order.gather(1, at[:, None])[:, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_shapes_and_empty(dtype):
    import tsb

    x, u = _logits(6, 1025, dtype, seed=7)
    want = tsb.sample(x, u, 0.9, 40, 0.9, logprobs=True)
    wide = torch.full((6, 2049), 50.0, dtype=dtype, device="cuda")
    wide[:, 3:1028] = x
    views = [wide[:, 3:1028], x.t().contiguous().t()]
    for v in views:
        assert all(torch.equal(a, b) for a, b in zip(tsb.sample(v, u, 0.9, 40, 0.9, logprobs=True), want))
    t3 = tsb.sample(x.view(2, 3, 1025), u.view(2, 3), 0.9, 40, 0.9)
    assert t3.shape == (2, 3) and torch.equal(t3.view(-1), want[0])
    one = tsb.sample(x[0], u[0], 0.9, 40, 0.9)
    assert one.shape == () and one == want[0][0]
    assert tsb.sample(x[:0], u[:0]).shape == (0,)


def test_repeats_captures_and_streams():
    import tsb

    x, u = _logits(24, 33333, torch.bfloat16, seed=8)
    y, v = _logits(24, 33333, torch.bfloat16, seed=9)
    args = (0.9, 400, 0.95, 0.01)
    want, other = tsb.sample(x, u, *args), tsb.sample(y, v, *args)
    for _ in range(3):
        assert torch.equal(tsb.sample(x, u, *args), want)
    hx, hu = x.clone(), u.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tsb.sample(hx, hu, *args)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b, w in ((x, u, want), (y, v, other), (x, u, want)):
        hx.copy_(a)
        hu.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            eager = tsb.sample(y, v, *args)
        torch.cuda.synchronize()
        assert torch.equal(out, w) and torch.equal(eager, other)


def test_frequencies():
    """Many samples of one row follow its distribution: counts within five standard deviations."""
    import tsb

    g = torch.Generator(device="cuda").manual_seed(10)
    x = torch.tensor([[1.0, 0.0, 2.0, -1.0, 0.5]], device="cuda")
    n = 20000
    u = torch.rand(n, device="cuda", generator=g)
    tokens = tsb.sample(x.expand(n, 5).contiguous(), u)
    p = torch.softmax(x[0].double(), 0)
    counts = torch.bincount(tokens.long(), minlength=5).double()
    assert ((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_top_k_of_64_bits():
    """Values past 32 bits keep everything, as any k past the vocabulary does."""
    import tsb

    x = torch.randn(4, 500, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    u = torch.tensor([0.9, 0.99, 0.3, 0.999], device="cuda")
    k = torch.tensor([2**32 + 1, 2**40, -5, 2**31], device="cuda")
    assert torch.equal(tsb.sample(x, u, top_k=k), tsb.sample(x, u))
