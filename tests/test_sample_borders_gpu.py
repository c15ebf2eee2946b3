"""tsb.sample where a bound falls on an end: filters that leave one token, random
numbers of one and more. Every call goes through the C entry with outputs that
hold a sentinel, so that a value that was never written shows."""

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
