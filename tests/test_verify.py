"""The operators after a verify pass and the shared-prefix attention, without a
GPU: their C entries' refusals (all before any launch), workspace sizes, the
Python refusals that need no device, and the oracle they are tested against."""

import ctypes
import itertools

import numpy as np
import pytest
import torch

from oracle import verify as overify

FAKE = 0x10000  # never dereferenced: every call fails its host-side checks


def _lib():
    from tsb import _lib

    return _lib


def _attn(lib, fmt=0, pre=None, own=None, **kw):
    L = _lib()
    a = dict(q=FAKE, sb=24 * 16 * 256, sh=16 * 256, st=256, lengths=None, parents=FAKE, bits=None, B=2, T=16, Hq=24, Hkv=4,
             D=256, tail=16, scale=0.0625, out=FAKE, lse=None, sums=None, ws=FAKE, ws_bytes=1 << 40)
    a.update(kw)
    scales = FAKE if fmt else None
    biases = FAKE if fmt == L.TSB_KV_MLX_Q8_G64 else None
    base = dict(k=FAKE, k_scales=scales, k_biases=biases, v=FAKE, v_scales=scales, v_biases=biases, capacity=1024, rows=1000)
    p, o = L.KVT(**{**base, **(pre or {})}), L.KVT(**{**base, **(own or {})})
    return lib.tsb_tree_attn_shared(a["q"], a["sb"], a["sh"], a["st"], fmt, ctypes.byref(p), ctypes.byref(o), a["lengths"],
                                    a["parents"], a["bits"], a["B"], a["T"], a["Hq"], a["Hkv"], a["D"], a["tail"],
                                    a["scale"], a["out"], a["lse"], a["sums"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(parents=None), dict(q=FAKE + 8), dict(out=FAKE + 2),
                                dict(lse=FAKE + 2), dict(sums=FAKE + 1), dict(sb=12), dict(sh=4), dict(st=255),
                                dict(B=0), dict(T=0), dict(Hq=0), dict(Hkv=0), dict(ws=FAKE + 4),
                                dict(pre=dict(rows=1025)), dict(own=dict(rows=1025)), dict(pre=dict(rows=-1)),
                                dict(pre=dict(k=None)), dict(own=dict(v=None)), dict(pre=dict(v=FAKE + 8)),
                                dict(fmt=1, pre=dict(k_scales=None)), dict(fmt=1, own=dict(v_biases=None)),
                                dict(fmt=1, pre=dict(k_scales=FAKE + 4)), dict(fmt=2, own=dict(k_scales=None)),
                                dict(fmt=2, pre=dict(v_scales=FAKE + 2))])
def test_shared_attention_contract(lib_built, kw):
    L = _lib()
    assert _attn(L.load(), **kw) == L.TSB_EINVAL


@pytest.mark.parametrize("kw", [dict(D=128), dict(Hq=22), dict(T=65, tail=65), dict(parents=None, bits=FAKE, tail=65),
                                dict(parents=None, bits=FAKE, tail=-1), dict(fmt=3), dict(fmt=-1), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=float("nan")), dict(B=1 << 14, T=64),
                                dict(own=dict(capacity=1 << 30))])
def test_shared_attention_declines(lib_built, kw):
    L = _lib()
    assert _attn(L.load(), **kw) == L.TSB_EUNSUPPORTED


def test_shared_attention_workspace(lib_built):
    L = _lib()
    lib = L.load()
    size = lib.tsb_tree_attn_shared_workspace_bytes
    need = size(2, 16, 24, 4, 256, 1000, 1000, 0)
    assert need > 0
    assert _attn(lib, ws=None) == _attn(lib, ws_bytes=need - 1) == L.TSB_EWORKSPACE
    # an 8-bit cache's rows in bf16, K and V, beside the partials
    assert size(2, 16, 24, 4, 256, 1000, 1000, 1) == need + 2 * 4 * (1000 + 2 * 1000) * 512
    assert size(0, 16, 24, 4, 256, 1000, 1000, 0) == size(2, 16, 22, 4, 256, 1000, 1000, 0) == 0
    # partials of every row: no more of them than key splits and chunks there can be
    for b, t, hkv, p, own in itertools.product((1, 7, 64), (1, 13, 64), (1, 8), (0, 1, 5003, 1 << 20), (0, 1, 333, 4096)):
        n = size(b, t, 8 * hkv, hkv, 256, p, own, 0)
        assert n % 256 == 0 and n <= (64 + 16) * b * t * 8 * hkv * 258 * 4 + 256
        assert n >= (int(p > 0) + int(own > 0)) * b * t * 8 * hkv * 258 * 4


def _sample(lib, **kw):
    a = dict(logits=FAKE, dtype=2, rows=4, vocab=1000, stride=1000, u=FAKE, token=FAKE)
    a.update(kw)
    return lib.tsb_sample(a["logits"], a["dtype"], a["rows"], a["vocab"], a["stride"], a["u"], None, 1.0, None, 0, None, 1.0,
                          None, 0.0, a["token"], None, None)


def test_sample_refusals(lib_built):
    L = _lib()
    lib = L.load()
    for kw in (dict(logits=None), dict(u=None), dict(token=None), dict(rows=0), dict(vocab=0), dict(stride=999),
               dict(dtype=L.TSB_MASK_BF16, logits=FAKE + 1), dict(dtype=L.TSB_MASK_F32, logits=FAKE + 2)):
        assert _sample(lib, **{"dtype": L.TSB_MASK_F32, **kw}) == L.TSB_EINVAL, kw
    assert _sample(lib, vocab=(1 << 20) + 1, stride=1 << 21) == L.TSB_EUNSUPPORTED
    assert _sample(lib, dtype=L.TSB_MASK_BOOL) == _sample(lib, dtype=9) == L.TSB_EUNSUPPORTED


def test_accept_refusals(lib_built):
    L = _lib()
    lib = L.load()
    for i in (0, 1, 2, 5, 6, 7):
        args = [FAKE] * 3 + [2, 4] + [FAKE] * 3
        args[i] = None
        assert lib.tsb_tree_accept(*args, None) == L.TSB_EINVAL
    assert lib.tsb_tree_accept(FAKE, FAKE, FAKE, 0, 4, FAKE, FAKE, FAKE, None) == L.TSB_EINVAL
    assert lib.tsb_tree_accept(FAKE, FAKE, FAKE, 2, 0, FAKE, FAKE, FAKE, None) == L.TSB_EINVAL
    assert lib.tsb_tree_accept(FAKE, FAKE, FAKE, 2, 65, FAKE, FAKE, FAKE, None) == L.TSB_EUNSUPPORTED


def _commit(lib, fmt=0, layers=1, planes=None, **kw):
    a = dict(B=2, Hkv=4, D=256, cap=64, T=8, lengths=FAKE, path=FAKE, n_keep=FAKE, new=None)
    a.update(kw)
    arrays = [(ctypes.c_void_p * layers)(*([x] * layers)) if x is not None else None
              for x in (planes or [FAKE] * 6)]
    return lib.tsb_kv_commit_paths(fmt, layers, *arrays, a["B"], a["Hkv"], a["D"], a["cap"], a["T"], a["lengths"], a["path"],
                                   a["n_keep"], a["new"], None)


def test_commit_refusals(lib_built):
    L = _lib()
    lib = L.load()
    for kw in (dict(B=0), dict(Hkv=0), dict(cap=0), dict(T=0), dict(lengths=None), dict(path=None), dict(n_keep=None),
               dict(new=FAKE), dict(planes=[None] + [FAKE] * 5), dict(planes=[FAKE + 8] + [FAKE] * 5),
               dict(fmt=1, planes=[FAKE, FAKE, None, FAKE, FAKE, FAKE]), dict(fmt=2, planes=[FAKE, None] + [FAKE] * 4),
               dict(fmt=1, planes=[FAKE, FAKE + 4, FAKE, FAKE, FAKE, FAKE])):
        assert _commit(lib, **kw) == L.TSB_EINVAL, kw
    for kw in (dict(D=128), dict(T=65), dict(layers=49), dict(fmt=3), dict(B=1 << 28)):
        assert _commit(lib, **kw) == L.TSB_EUNSUPPORTED, kw


def test_python_refuses_cpu_tensors(lib_built):
    import tsb

    x = torch.zeros(2, 100)
    with pytest.raises(ValueError):
        tsb.sample(x, torch.zeros(2))
    i = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        tsb.tree_accept(i, i, i)
    cache = tsb.KVCache(*(torch.zeros(1, 1, 8, 256, dtype=torch.bfloat16) for _ in range(2)), 8)
    with pytest.raises(ValueError):
        tsb.tree_flash_shared(torch.zeros(1, 2, 4, 256, dtype=torch.bfloat16), cache, cache, 1.0, parents=i[:1])
    with pytest.raises(ValueError):
        tsb.PathCommit([cache])
    with pytest.raises(ValueError):
        tsb.PathCommit([])


# ---------------------------------------------------------------- the oracle

@pytest.mark.parametrize("seed", range(6))
def test_oracle_sample_is_the_distribution(seed):
    """Over a fine grid of u the tokens come in the shares of the filtered softmax,
    and the log probabilities are those shares."""
    r = np.random.default_rng(seed)
    x = r.normal(size=12) * 2
    x[r.integers(12)] = -np.inf
    k, p, m, t = int(r.integers(0, 9)), float(r.uniform(0.5, 1.2)), float(r.uniform(0, 0.2)), float(r.uniform(0.5, 2))
    w = np.exp(x / t)
    order = np.argsort(-x, kind="stable")
    keep = [i for n, i in enumerate(order) if np.isfinite(x[i]) and (k <= 0 or n < k)]
    if p < 1:
        mass = np.cumsum(w[keep])
        keep = [i for n, i in enumerate(keep) if n == 0 or mass[n - 1] < p * mass[-1]]
    keep = [i for n, i in enumerate(keep) if n == 0 or w[i] >= m * w[keep[0]]]
    share = np.zeros(12)
    share[keep] = w[keep] / w[keep].sum()
    grid = (np.arange(4000) + 0.5) / 4000
    drawn = [overify.sample(x, u, t, k, p, m) for u in grid]
    counts = np.bincount([d[0] for d in drawn], minlength=12) / grid.size
    assert np.abs(counts - share).max() <= 1.0 / grid.size  # a token's interval holds its share of the grid, to one point
    for token, logp, _ in drawn[::97]:
        assert abs(logp - np.log(share[token])) < 1e-12


def test_oracle_accept_by_enumeration():
    """The walk against the definition: the accepted nodes are those all of whose
    steps from the root hold, following the lowest child at each."""
    r = np.random.default_rng(3)
    for _ in range(200):
        t = int(r.integers(1, 8))
        parents = [-1] + [int(r.integers(0, i)) for i in range(1, t)]
        tokens, samples = r.integers(0, 3, t).tolist(), r.integers(-1, 3, t).tolist()
        path, nxt = overify.tree_accept(tokens, parents, samples)
        assert path[0] == 0 and nxt == samples[path[-1]]
        for a, b in zip(path, path[1:]):
            assert b == min(c for c in range(t) if parents[c] == a and tokens[c] == samples[a] >= 0)
        assert not any(parents[c] == path[-1] and tokens[c] == samples[path[-1]] >= 0 for c in range(path[-1] + 1, t))
