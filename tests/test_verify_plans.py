"""What a commit plan and a verify step refuse before they touch a cache, on the CPU:
the checks of the caches' tensors need no device."""

import pytest
import torch

HKV, CAP = 2, 12


@pytest.fixture
def plan(lib_built, monkeypatch):
    """PathCommit of caches that lie in host memory (the plan itself launches nothing)."""
    import tsb
    from tsb import verify

    monkeypatch.setattr(verify, "_require_cuda", lambda *ts: None)
    return tsb.PathCommit


def _cache(fmt, b=2, **other):
    """A cache of zeros, with some of its tensors replaced."""
    import tsb

    z = lambda *s, dtype: torch.zeros(b, HKV, CAP, *s, dtype=dtype)  # noqa: E731
    if fmt == "bf16":
        kind, t = tsb.KVCache, dict(keys=z(256, dtype=torch.bfloat16), values=z(256, dtype=torch.bfloat16))
    elif fmt == "ref_q8":
        kind, t = tsb.Q8KVCache, dict(keys=z(256, dtype=torch.int8), values=z(256, dtype=torch.int8),
                                      k_scale=z(dtype=torch.float32), v_scale=z(dtype=torch.float32))
    else:
        kind, t = tsb.MLXQ8KVCache, dict(keys=z(64, dtype=torch.int32), values=z(64, dtype=torch.int32))
        t.update({n: z(4, dtype=torch.bfloat16) for n in ("k_scales", "k_biases", "v_scales", "v_biases")})
    for name, change in other.items():
        t[name] = change(t[name])
    return kind(**t, offset=CAP)


BAD = [
    ("bf16", "keys", lambda t: t.float()), ("bf16", "values", lambda t: t.half()), ("bf16", "keys", lambda t: t.to(torch.int8)),
    ("bf16", "values", lambda t: t[:, :1].contiguous()), ("bf16", "keys", lambda t: t[0]),
    ("ref_q8", "keys", lambda t: t.to(torch.bfloat16)), ("ref_q8", "values", lambda t: t.float()),
    ("ref_q8", "k_scale", lambda t: t.half()), ("ref_q8", "v_scale", lambda t: t.bfloat16()),
    ("ref_q8", "v_scale", lambda t: t.double()), ("ref_q8", "k_scale", lambda t: t[:, :, :-1].contiguous()),
    ("ref_q8", "k_scale", lambda t: t[..., None].expand(-1, -1, -1, 2).contiguous()), ("ref_q8", "v_scale", lambda t: None),
    ("mlx_q8", "keys", lambda t: t.long()), ("mlx_q8", "values", lambda t: t.float()),
    ("mlx_q8", "k_scales", lambda t: t.float()), ("mlx_q8", "v_biases", lambda t: t.half()),
    ("mlx_q8", "v_scales", lambda t: t[..., :2].contiguous()), ("mlx_q8", "k_biases", lambda t: torch.cat([t, t], -1)),
    ("mlx_q8", "k_biases", lambda t: t[..., 0].contiguous()), ("mlx_q8", "v_scales", lambda t: None),
    ("bf16", "keys", lambda t: t.reshape(-1)), ("mlx_q8", "k_scales", lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)),
]


@pytest.mark.parametrize("fmt,name,change", BAD, ids=[f"{i}-{f}-{n}" for i, (f, n, _) in enumerate(BAD)])
def test_plan_refuses_tensors_of_another_kind(plan, fmt, name, change):
    """A row is moved by its format's width: tensors of another type or shape would lose
    rows, or be written past their ends."""
    good = _cache(fmt)
    plan([good])
    for caches in ([_cache(fmt, **{name: change})], [good, _cache(fmt, **{name: change})]):
        with pytest.raises(ValueError):
            plan(caches)


def test_plan_takes_every_format(plan):
    import tsb

    words = _cache("mlx_q8", keys=lambda t: t.view(torch.uint32), values=lambda t: t.view(torch.uint32))
    plan([_cache("bf16"), _cache("ref_q8"), _cache("mlx_q8"), words])
    c = _cache("bf16")
    past = tsb.KVCache(c.keys, c.values, CAP + 5)  # a plan does not read the offset
    plan([past])


# ---------------------------------------------------------------- the decoder's verify step

class _Reached(Exception):
    pass


@pytest.fixture
def decoder(monkeypatch):
    """A decoder of two layers whose layer stack ends the call: nothing runs on a device."""
    from tsb import decoder as tdec

    dec = tdec.VerifyDecoder.__new__(tdec.VerifyDecoder)
    dec.layers = [None, None]

    def stop(self, *args):
        raise _Reached

    monkeypatch.setattr(tdec.VerifyDecoder, "step_shared", stop)
    return dec


def _verify(dec, caches, commit):
    i = torch.zeros(2, 3, dtype=torch.int32)
    return dec.verify(torch.zeros(6, 8), i, i, [], caches, torch.zeros(2, dtype=torch.int32), None, torch.zeros(2, 3), commit)


@pytest.mark.parametrize("fmt", ["bf16", "ref_q8", "mlx_q8"])
def test_verify_takes_its_caches_plan_only(plan, decoder, fmt):
    """A plan of other caches would move those caches' rows and keep these as they are."""
    import copy

    caches = [_cache(fmt), _cache(fmt)]
    for good in (plan(caches), plan(caches[::-1]), plan([copy.copy(c) for c in caches])):
        with pytest.raises(_Reached):
            _verify(decoder, caches, good)
    clones = [type(c)(**{k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in vars(c).items()}) for c in caches]
    for other in (clones, [caches[0], clones[1]], caches[:1], caches + clones[:1]):
        with pytest.raises(ValueError, match="commit"):
            _verify(decoder, caches, plan(other))
    stale = plan(caches)
    caches[1].values = caches[1].values.clone()  # a cache got a new tensor: the plan still has the old one
    with pytest.raises(ValueError, match="commit"):
        _verify(decoder, caches, stale)


@pytest.fixture
def stack(lib_built, monkeypatch):
    """A decoder of two layers whose first work on the device ends the call."""
    from tsb import decoder as tdec

    def stop(self, *args):
        raise _Reached

    dec = tdec.VerifyDecoder.__new__(tdec.VerifyDecoder)
    dec.layers = [None, None]
    dec.cfg = tdec.DecoderConfig(layers=2, hidden=8, hq=4, hkv=HKV, d=256, inter=8)
    monkeypatch.setattr(tdec.VerifyDecoder, "_buffers", stop)
    return dec


def _step(dec, prefixes, caches, b=2):
    return dec.step_shared(torch.zeros(b * 3, 8), torch.zeros(b, 3, dtype=torch.int32), prefixes, caches,
                           torch.full((b,), 4, dtype=torch.int32))


@pytest.mark.parametrize("fmt", ["bf16", "ref_q8", "mlx_q8"])
def test_step_shared_refuses_caches_that_it_would_write_past(stack, fmt):
    """Every layer's nodes are written by the batch, heads and format that the call
    implies: a cache of fewer requests or heads, or of another type, is refused before
    the first layer runs."""
    pre, own = [_cache(fmt, b=1) for _ in range(2)], [_cache(fmt) for _ in range(2)]
    with pytest.raises(_Reached):
        _step(stack, pre, own)
    name = "keys" if fmt == "bf16" else "k_scale" if fmt == "ref_q8" else "k_biases"
    half = lambda t: t[:, :1].contiguous()  # noqa: E731
    tensors = [n for n, v in vars(own[0]).items() if isinstance(v, torch.Tensor)]
    bad = [_cache(fmt, b=1), _cache(fmt, b=3), _cache(fmt, **{n: half for n in tensors}),
           _cache(fmt, values=lambda t: t.double()), _cache(fmt, **{name: lambda t: t[:, :, :-1].contiguous()}),
           _cache("ref_q8" if fmt == "bf16" else "bf16")]
    for c in bad:
        with pytest.raises(ValueError):
            _step(stack, pre, [own[0], c])
    for p in (_cache(fmt), _cache(fmt, b=1, **{n: half for n in tensors}), _cache("mlx_q8" if fmt == "bf16" else "bf16", b=1)):
        with pytest.raises(ValueError):
            _step(stack, [pre[0], p], own)
    own[1].offset = CAP + 1
    with pytest.raises(ValueError):
        _step(stack, pre, own)
