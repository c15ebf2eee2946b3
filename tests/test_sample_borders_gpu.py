"""tsb.sample where a bound falls on an end: filters that leave one token, random
numbers of one and more. Every call goes through the C entry with outputs that
hold a sentinel, so that a value that was never written shows.

Precision. A token's weight is a whole number m of at least 0.989 * 2^22, rounded
to the nearest: off by 0.5 / (0.989 * 2^22) = 2^-22.98 of itself, equal logits by
the same. m comes from a float32 series whose own roundings are below 2^-6 of a
unit. Of float32 logits (and of 16-bit ones far apart) the difference to the
largest is rounded too, by 2^-24 of itself, d / temperature * 2^-24 of the weight.
Sums over the bins are whole numbers of 2^-43, each bin's rounded once, 1376 of them
2^-33.6 at most, and with top_k <= 64 every weight is a multiple of 2^-40, 64 of them
2^-35. So eps = 1.25e-7 + 2^-24 * max(d / temperature) bounds a weight's relative
error, sums' too, and a share's border c is off by c (1 - c) 2 eps <= eps / 2.
Wherever a bound lies within eps of a border, either side is right; the token then
is one of the two, and its log probability must be that of the token."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
UNWRITTEN = -77


def _draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens, logprobs) of rows x; parameters are numbers or tensors of one value per row."""
    from tsb import _lib, verify

    rows, vocab = x.shape
    token = torch.full((rows,), UNWRITTEN, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 77.0, device="cuda")
    ptr = lambda v: v.data_ptr() if isinstance(v, torch.Tensor) else None  # noqa: E731
    num = lambda v: 0 if isinstance(v, torch.Tensor) else v  # noqa: E731
    status = _lib.load().tsb_sample(x.data_ptr(), verify._LOGIT_TYPES[x.dtype], rows, vocab, x.stride(0), u.data_ptr(),
                                    ptr(temperature), num(temperature), ptr(top_k), num(top_k), ptr(top_p), num(top_p),
                                    ptr(min_p), num(min_p), token.data_ptr(), logprob.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream)
    assert status == 0
    return token, logprob


def _rows(kind, vocab, dtype):
    """Four rows, and the first token of each row's order."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(4, vocab, device="cuda", generator=g)
    if kind == "equal":
        x = torch.full((4, vocab), 1.5, device="cuda")
    elif kind == "tied":  # half of the tokens share the largest logit
        x[:, 1::2] = 6.0
    elif kind == "near":  # neighbours that differ in the last bits
        x = 1 + 1e-3 * torch.rand(4, vocab, device="cuda", generator=g)
    x = x.to(dtype)
    return x, torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, 0].int()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["flat", "equal", "tied", "near"])
@pytest.mark.parametrize("vocab", [1, 128, 129, 3000, 60013, 100003])
def test_top_p_that_leaves_one_token(dtype, kind, vocab):
    """top_p of zero, below it, and below the first token's share: the first token, with log probability 0."""
    x, first = _rows(kind, vocab, dtype)
    u = torch.tensor([0.0, 0.3, 0.7, 0.99999994], device="cuda")
    for p in (0.0, -1.0, -float("inf"), 1e-30, 5e-324):
        for temperature in (1.0, 50.0):
            for k in (0, 5, 129, 200, 5000):
                for top_p in (p, torch.full((4,), p, device="cuda")):
                    token, logprob = _draw(x, u, temperature, k, top_p)
                    assert torch.equal(token, first), (p, temperature, k, type(top_p))
                    assert (logprob == 0).all(), (p, temperature, k, type(top_p))


def test_top_p_of_zero_in_some_rows():
    """Rows of their own top_p do not change each other."""
    import tsb

    x, first = _rows("flat", 30011, torch.bfloat16)
    u = torch.tensor([0.5, 0.5, 0.9, 0.9], device="cuda")
    p = torch.tensor([0.0, 0.9, -2.0, 1.0], device="cuda")
    token, _ = _draw(x, u, 3.0, 0, p)
    assert token[0] == first[0] and token[2] == first[2]
    assert token[1] == tsb.sample(x[1:2], u[1:2], 3.0, top_p=float(p[1]))[0]
    assert token[3] == tsb.sample(x[3:], u[3:], 3.0)[0]


# ---------------------------------------------------------------- random numbers at the upper end

def _right(row, draws, temperature, top_k, top_p, min_p):
    """One row's draws (u, token, log probability) against 64 bits, within eps of the borders; what is wrong with them."""
    x, order = row
    order = order[:top_k] if top_k > 0 else order
    d = (x[order[0]] - x[order]) / temperature
    w = np.exp(-d)
    assert w[-1] > 2.0**-40  # every token has a mass, of several units
    eps = 1.25e-7 + 2.0**-24 * d[-1]
    cum = np.cumsum(w)
    fewest, most = len(w), len(w)  # how many tokens the filters keep, from and to
    if top_p < 1:
        fewest, most = (min(int(np.searchsorted(cum, (top_p + e) * cum[-1])) + 1, len(w)) for e in (-eps, eps))
    if min_p > 0:
        # the largest logit's weight is 1, without a rounding
        fewest, most = (min(n, int(((w == 1) | (w >= min_p * (1 + e))).sum())) for n, e in ((fewest, eps), (most, -eps)))
    wrong = []
    for u, token, logprob in draws:
        why = []
        for n in range(fewest, most + 1):
            if u >= 1:
                low = high = n - 1
            else:
                low, high = (min(int(np.searchsorted(cum[:n], (u + e) * cum[n - 1], side="right")), n - 1) for e in (-eps, eps))
            at = np.flatnonzero(order[low:high + 1] == token)
            if not at.size:
                why.append(("token", token, n, order[low:high + 1].tolist()))
                continue
            want = -d[low + int(at[0])] - np.log(cum[n - 1])
            # rounded once, over log(kept) to one step, weights' errors and 2^-44 of 1 / temperature
            if abs(logprob - want) <= 2.0**-24 * abs(want) + 2.0**-23 * np.log(cum[n - 1]) + 2 * eps:
                why = []
                break
            why.append(("logprob", logprob, want, n))
        if why:
            wrong.append((u, why))
    return wrong


def _in_order(x):
    return [(row, np.argsort(-row, kind="stable")) for row in x.double().cpu().numpy()]


def _check(x, us, **params):
    """Every row of x with every set of random numbers: us a list of tensors of one number per row."""
    params = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **params}
    drawn = [[u.tolist(), *(t.tolist() for t in _draw(x, u, **params))] for u in us]
    for r, row in enumerate(_in_order(x)):
        wrong = _right(row, [[v[r] for v in d] for d in drawn], **params)
        assert not wrong, (params, r, wrong)


END = [1.0, 2.0, 0.99999994, 0.9999999]  # 1 - 2^-24 and 1 - 2^-23 are the last below one
FILTERS = [{}, {"top_p": 0.9}, {"top_p": 0.9, "temperature": 0.7}, {"min_p": 0.01}, {"min_p": 0.3, "temperature": 1.5},
           {"top_p": 0.97, "min_p": 0.001}, {"top_k": 40}, {"top_k": 100}, {"top_k": 1000, "top_p": 0.95},
           {"top_k": 3000}, {"top_k": 4000, "top_p": 0.99, "min_p": 1e-4}, {"temperature": 4.0}, {"temperature": 4.0, "top_p": 0.8},
           {"temperature": 4.0, "top_k": 4500}, {"temperature": 4.0, "min_p": 0.05}, {"temperature": 4.0, "top_p": 0.95, "min_p": 0.02}]


def _in_order(x):
    return [(row, np.argsort(-row, kind="stable")) for row in x.double().cpu().numpy()]


def _ends(rows, vocab, dtype, peaks, filters):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = 1.5 * torch.randn(rows, vocab, device="cuda", generator=g)
    if peaks:
        at = torch.randint(0, vocab, (rows, 16), device="cuda", generator=g)
        x.scatter_reduce_(1, at, 4 + 4 * torch.rand(rows, 16, device="cuda", generator=g), "amax")
    x = x.clamp_min(-7).to(dtype)
    for params in filters:
        _check(x, [torch.full((rows,), value, device="cuda") for value in END], **params)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("params", FILTERS, ids=lambda p: ",".join(f"{k}={v}" for k, v in p.items()) or "plain")
def test_random_numbers_of_one(dtype, params):
    """u = 1 and the last float32 numbers below it: the last token that the filters keep, never one past it and never none."""
    _ends(100, 5003, dtype, True, [params])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,peaks", [(1, True), (2, True), (129, False), (70001, True), (60013, False)])
def test_random_numbers_of_one_over_sizes(dtype, vocab, peaks):
    _ends(3, vocab, dtype, peaks, FILTERS + [{"temperature": 4.0, "top_k": 50000}, {"temperature": 4.0, "top_k": 30000, "top_p": 0.9}])


@pytest.mark.parametrize("dtype", DTYPES)
def test_random_numbers_of_one_on_equal_and_near_logits(dtype):
    """More tokens in one bin than can be listed, and ties that a filter cuts."""
    us = [torch.full((4,), value, device="cuda") for value in (1.0, 0.99999994, 0.5, 0.0)]
    for kind in ("equal", "tied", "near"):
        for vocab in (3000, 60013):
            x, _ = _rows(kind, vocab, dtype)
            for params in ({}, {"top_k": 1500}, {"top_k": 2900}, {"top_p": 0.5}, {"top_p": 0.731}, {"top_k": 2900, "top_p": 0.7},
                           {"min_p": 0.5}, {"min_p": 1.0}, {"top_p": 0.9, "min_p": 0.9996}):
                _check(x, us, **params)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_largest_row_of_equal_weights(dtype):
    """2^20 tokens of the same weight, by equal logits or by temperature: the largest sums there are."""
    n = 1 << 20
    us = [torch.full((2,), value, device="cuda") for value in (1.0, 0.99999994, 0.5, 1e-6, 0.0)]
    x = torch.full((2, n), -3.0, device="cuda").to(dtype)
    for params in ({}, {"top_p": 0.75}, {"top_k": n - 5}, {"top_k": 700000, "top_p": 0.5}, {"min_p": 0.9}):
        _check(x, us, **params)
    x[1] = torch.arange(n, device="cuda").remainder(97).to(dtype)
    _check(x, us, temperature=1e30)


def test_two_values_near_a_border():
    """Rows of two logits, thousands of each: all weights of a kind are off by the same
    rounding, and u on both sides of the border between the kinds, a few eps away."""
    for dtype in DTYPES:
        for a, b, half in ((1.0, 0.75, 2500), (2.0, -1.0, 20000), (0.5, 0.4375, 4000)):
            x = torch.full((8, 2 * half), b, device="cuda")
            x[:, :half] = a
            x = x.to(dtype)
            border = 1 / (1 + np.exp(b - a))
            u = torch.tensor([border + e for e in (-4e-7, -2.5e-7, -1.3e-7, -6e-8, 6e-8, 1.3e-7, 2.5e-7, 4e-7)], device="cuda").float()
            for params in ({}, {"top_p": 0.999}, {"top_k": half + 77}, {"min_p": 0.01}):
                _check(x, [u], **params)
