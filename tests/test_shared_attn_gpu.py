"""tsb.tree_flash_shared against a plain implementation in 64 bits.

Tolerance (per output element, from the roundings that the kernel makes, half a
step of bf16 being 2^-8): each weight p is rounded to bf16 once before P V, at
most 2^-8 sum p|v|; the result is rounded to bf16 once, 2^-8 |out|; scores are
float32 sums of 256 products, off by at most 256 * 2^-24 * sum|q k| * scale,
which moves every weight by that factor, as does the float32 sum over n keys by
n * 2^-24. The log-sum-exp has the last two alone, and its own rounding."""

import numpy as np
import pytest
import torch

from oracle import gen

pytestmark = pytest.mark.gpu
D = 256
FORMATS = ("bf16", "mlx_q8", "ref_q8")


def _rows(shape, fmt, seed):
    """(cache tensors, values float64) of random rows."""
    import tsb

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, D, device="cuda", generator=g)
    if fmt == "bf16":
        return (x.bfloat16(),), x.bfloat16().double()
    if fmt == "ref_q8":
        q, s = tsb.quantize_rows(x)
        return (q, s), q.double() * s.double()[..., None]
    w, s, b = tsb.quantize_g64(x)
    codes = w.view(torch.uint8).double().reshape(*shape, 4, 64)
    value = (codes * s.double()[..., None] + b.double()[..., None]).float().bfloat16()
    return (w, s, b), value.double().reshape(*shape, D)


def _cache(k, v, fmt, offset):
    import tsb

    if fmt == "bf16":
        return tsb.KVCache(k[0], v[0], offset)
    if fmt == "ref_q8":
        return tsb.Q8KVCache(k[0], v[0], k[1], v[1], offset)
    return tsb.MLXQ8KVCache(k[0], v[0], k[1], k[2], v[1], v[2], offset)


def _make(fmt, hkv, b, p_cap, o_cap, p_rows, o_rows, seed=0):
    pk, pkv = _rows((1, hkv, p_cap), fmt, seed + 1)
    pv, pvv = _rows((1, hkv, p_cap), fmt, seed + 2)
    ok, okv = _rows((b, hkv, o_cap), fmt, seed + 3)
    ov, ovv = _rows((b, hkv, o_cap), fmt, seed + 4)
    return _cache(pk, pv, fmt, p_rows), _cache(ok, ov, fmt, o_rows), (pkv, pvv, okv, ovv)


def _poison(planes, rows):
    """What lies past the valid rows must not matter: NaN where the type has one."""
    for t in planes:
        t[:, :, rows:] = float("nan") if t.is_floating_point() else 0x7F


def _ancestor_sets(parents):
    t = len(parents)
    see = np.zeros((t, t), bool)
    for i in range(t):
        j = i
        while j >= 0:
            see[i, j] = True
            j = parents[j]
    return see


def _check(q, vals, p_rows, lengths, see_tail, scale, out, lse=None):
    """see_tail: per request a bool (n, tail) of which tail rows each node sees."""
    pkv, pvv, okv, ovv = vals
    b, hq, n, _ = q.shape
    g = hq // pkv.shape[1]
    for i in range(b):
        m = lengths[i]
        tail = see_tail[i].shape[1]
        k = torch.cat([pkv[0, :, :p_rows], okv[i, :, :m]], 1).repeat_interleave(g, 0)
        v = torch.cat([pvv[0, :, :p_rows], ovv[i, :, :m]], 1).repeat_interleave(g, 0)
        see = torch.ones(n, p_rows + m, dtype=torch.bool)
        own = min(m, tail)
        if own:
            see[:, p_rows + m - own:] = torch.from_numpy(see_tail[i][:, tail - own:].copy())
        see = see.cuda()
        s = torch.einsum("hnd,hkd->hnk", q[i].double(), k) * scale
        size = torch.einsum("hnd,hkd->hnk", q[i].double().abs(), k.abs()).amax(-1) * scale if p_rows + m else torch.zeros(hq, n, device="cuda")
        s = s.masked_fill(~see, -torch.inf)
        any_ = see.any(-1)[None].expand(hq, n)
        ref_lse = torch.logsumexp(s, -1) if p_rows + m else torch.full((hq, n), -torch.inf, device="cuda")
        w = torch.where(any_[..., None], torch.exp(s - torch.where(any_, ref_lse, 0.0)[..., None]), 0.0)
        ref = w @ v
        mass = w @ v.abs()
        count = p_rows + m
        slack = 256 * 2.0**-24 * size + (count + 64) * 2.0**-24  # relative, of every weight
        tol = 2.0**-8 * (mass + ref.abs()) + 2 * slack[..., None] * mass + 1e-30
        err = (out[i].double() - ref).abs()
        assert torch.isfinite(out[i].float()).all()
        assert (err <= tol).all(), f"request {i}: {float((err / tol).max())} of the tolerance"
        if lse is not None:
            got = lse[i].double()
            assert torch.equal(torch.isneginf(got), ~any_)
            off = (got - ref_lse)[any_].abs()
            assert (off <= (slack + 2.0**-20 * (1 + ref_lse.abs()))[any_]).all(), float(off.max())


def _run(fmt, b, n, hq, hkv, p_rows, lengths, p_cap=None, o_cap=None, seed=0, stats=True, poison=True):
    import tsb

    p_cap = p_cap or p_rows + 3
    o_rows = max(max(lengths), 1)
    o_cap = o_cap or o_rows + 5
    prefix, cache, vals = _make(fmt, hkv, b, p_cap, o_cap, p_rows, o_rows, seed)
    if poison:
        for c, r in ((prefix, p_rows),):
            _poison([t for t in vars(c).values() if isinstance(t, torch.Tensor)], r)
        for t in [t for t in vars(cache).values() if isinstance(t, torch.Tensor)]:
            for i, m in enumerate(lengths):
                t[i, :, m:] = float("nan") if t.is_floating_point() else 0x7F
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(b, hq, n, D, device="cuda", generator=g).bfloat16()
    rng = np.random.default_rng(seed)
    parents = np.stack([gen.tree_parents(rng, n) for _ in range(b)])
    out, lse, ones = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=torch.from_numpy(parents).cuda(),
                                           lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), stats=True)
    torch.cuda.synchronize()
    assert out.shape == q.shape and lse.shape == (b, hq, n, 1) and torch.equal(ones, torch.ones_like(lse))
    _check(q, vals, p_rows, lengths, [_ancestor_sets(p) for p in parents], D**-0.5, out, lse[..., 0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,n,hq,hkv,p_rows,lengths", [
    (1, 1, 1, 1, 1, [1]),                          # one of everything
    (3, 1, 6, 1, 70, [1, 64, 65]),                 # single tokens, tile edges
    (2, 5, 4, 2, 64, [5, 130]),
    (4, 16, 12, 2, 257, [16, 17, 100, 333]),       # packed rows cross requests and blocks
    (5, 13, 14, 2, 1000, [13, 14, 15, 16, 200]),   # odd everywhere
    (2, 64, 8, 1, 300, [64, 129]),                 # widest tree, eight heads to a key head
    (9, 3, 3, 3, 2049, [3, 4, 5, 6, 7, 8, 9, 10, 11]),  # one head to a key head
], ids=lambda v: "x".join(map(str, v)) if isinstance(v, list) else str(v))
def test_against_64_bits(fmt, b, n, hq, hkv, p_rows, lengths):
    _run(fmt, b, n, hq, hkv, p_rows, lengths)


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_prefix_and_no_own_rows(fmt):
    _run(fmt, 3, 4, 6, 2, 0, [4, 70, 9], p_cap=8)       # an empty prefix
    _run(fmt, 3, 4, 6, 2, 130, [0, 70, 4])              # a request with no rows sees the prefix alone
    _run(fmt, 2, 8, 6, 2, 65, [3, 1])                   # fewer own rows than tree nodes: the last of the tree
    _run(fmt, 2, 2, 2, 1, 0, [0, 2], p_cap=4)           # a request that sees nothing: zeros and -inf


@pytest.mark.parametrize("fmt", FORMATS)
def test_odd_capacities(fmt):
    _run(fmt, 3, 7, 4, 2, 129, [7, 71, 90], p_cap=129, o_cap=91)
    _run(fmt, 2, 7, 4, 2, 64, [7, 64], p_cap=65, o_cap=67)


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_prefix(fmt):
    """Many splits, and running maxima that grow along the keys (the largest scores come last)."""
    import tsb

    b, n, hq, hkv, p_rows, lengths = 2, 8, 8, 2, 9000, [8, 200]
    prefix, cache, vals = _make(fmt, hkv, b, p_rows, 256, p_rows, 200, seed=11)
    q = torch.randn(b, hq, n, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
    parents = np.tile(gen.chain_parents(n), (b, 1))
    for scale in (D**-0.5, 1.0, 1e-3):  # 1: near one-hot, maxima move by far more than 2^8; 1e-3: near the mean
        out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, scale, parents=torch.from_numpy(parents).cuda(),
                                            lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), stats=True)
        torch.cuda.synchronize()
        _check(q, vals, p_rows, lengths, [_ancestor_sets(p) for p in parents], scale, out, lse[..., 0])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tail", [0, 1, 9, 64])
def test_bits_and_tails(fmt, tail):
    import tsb

    b, n, hq, hkv, p_rows, lengths = 2, 6, 6, 3, 100, [70, 5]
    prefix, cache, vals = _make(fmt, hkv, b, 128, 80, p_rows, 70, seed=3)
    rng = np.random.default_rng(tail)
    see = rng.random((b, n, tail)) < 0.4
    bits = np.zeros((b, n), np.uint64)
    for i in range(b):
        for j in range(n):
            for k in range(tail):
                bits[i, j] |= np.uint64(int(see[i, j, k]) << k)
    q = torch.randn(b, hq, n, D, device="cuda").bfloat16()
    out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, torch.from_numpy(bits.view(np.int64)).cuda(), tail=tail,
                                        lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), stats=True)
    torch.cuda.synchronize()
    _check(q, vals, p_rows, lengths, list(see), D**-0.5, out, lse[..., 0])


def test_rows_that_see_nothing():
    """Masks that leave a row empty: no prefix, and no bit set."""
    import tsb

    prefix, cache, vals = _make("bf16", 1, 2, 4, 64, 0, 3)
    q = torch.randn(2, 4, 3, D, device="cuda").bfloat16()
    bits = torch.tensor([[0, 1, 7], [0, 0, 0]], device="cuda")
    out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, bits, tail=3, stats=True)
    see = [np.array([[0, 0, 0], [1, 0, 0], [1, 1, 1]], bool), np.zeros((3, 3), bool)]
    torch.cuda.synchronize()
    _check(q, vals, 0, [3, 3], see, D**-0.5, out, lse[..., 0])
    assert torch.equal(out[1], torch.zeros_like(out[1])) and torch.isneginf(lse[1]).all()


def test_lengths_default_and_bound():
    """No lengths: cache.offset for all; longer lengths than cache.offset count as it, negative ones as 0."""
    import tsb

    b, n = 3, 4
    prefix, cache, vals = _make("bf16", 2, b, 100, 90, 100, 77, seed=8)
    q = torch.randn(b, 4, n, D, device="cuda").bfloat16()
    parents = torch.arange(-1, n - 1, device="cuda", dtype=torch.int32)
    see = [_ancestor_sets(parents.tolist())] * b
    out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents, stats=True)
    torch.cuda.synchronize()
    _check(q, vals, 100, [77] * b, see, D**-0.5, out, lse[..., 0])
    lengths = torch.tensor([2**31 - 1, 78, -5], dtype=torch.int32, device="cuda")
    out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents, stats=True, lengths=lengths)
    torch.cuda.synchronize()
    _check(q, vals, 100, [77, 77, 0], see, D**-0.5, out, lse[..., 0])


def test_strided_queries_and_out():
    """Queries as a projection leaves them, (B, n, Hq, D), and a slice of wider rows; results do not change by a bit."""
    import tsb

    b, n, hq = 3, 9, 6
    prefix, cache, _ = _make("bf16", 2, b, 500, 40, 500, 33, seed=4)
    wide = torch.randn(b, n, hq, 2 * D, device="cuda").bfloat16()
    q = wide[..., :D].transpose(1, 2)
    parents = torch.from_numpy(np.stack([gen.tree_parents(np.random.default_rng(i), n) for i in range(b)])).cuda()
    want = tsb.tree_flash_shared(q.contiguous(), prefix, cache, D**-0.5, parents=parents)
    out = torch.empty_like(want)
    assert tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents, out=out) is out
    odd = torch.zeros(b * hq * n * D + 3, dtype=torch.bfloat16, device="cuda")[3:].view(b, hq, n, D).copy_(q)
    again = tsb.tree_flash_shared(odd, prefix, cache, D**-0.5, parents=parents)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_repeats_bit_for_bit_and_replays(fmt):
    """The same call gives the same bits; a captured call replays with other lengths, trees and queries; two graphs
    and an eager call on other streams do not disturb one another."""
    import tsb

    b, n, hq, hkv, p_rows = 4, 8, 8, 2, 2000
    prefix, cache, _ = _make(fmt, hkv, b, 2048, 300, p_rows, 300, seed=6)
    sets = []
    for i in range(3):
        g = torch.Generator(device="cuda").manual_seed(i)
        sets.append((torch.randn(b, hq, n, D, device="cuda", generator=g).bfloat16(),
                     torch.from_numpy(np.stack([gen.tree_parents(np.random.default_rng(10 * i + j), n) for j in range(b)])).cuda(),
                     torch.randint(n, 301, (b,), device="cuda", generator=g, dtype=torch.int32)))
    call = lambda s: tsb.tree_flash_shared(s[0], prefix, cache, D**-0.5, parents=s[1], lengths=s[2])  # noqa: E731
    want = [call(s).clone() for s in sets]
    for s, w in zip(sets, want):
        assert torch.equal(call(s), w)
    graphs = []
    for s in sets[:2]:
        held = [t.clone() for t in s]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(held)
        graphs.append((graph, held, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for first in (0, 1, 2):
        for i, (graph, held, out) in enumerate(graphs):
            for h, t in zip(held, sets[(first + i) % 3]):
                h.copy_(t)
        torch.cuda.synchronize()
        for i, (graph, held, out) in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = call(sets[(first + 2) % 3])
        torch.cuda.synchronize()
        for i, (graph, held, out) in enumerate(graphs):
            assert torch.equal(out, want[(first + i) % 3])
        assert torch.equal(eager, want[(first + 2) % 3])
    lib = tsb.load_library()
    assert lib.tsb_device_status(None, 0) == 0


def test_agrees_with_tree_flash():
    """The same rows in one cache per request through tsb.tree_flash: both within two roundings of each other."""
    import tsb

    b, n, hq, hkv, p_rows, m = 3, 8, 8, 2, 500, 44
    prefix, cache, _ = _make("bf16", hkv, b, p_rows, m, p_rows, m, seed=2)
    k = torch.cat([prefix.keys.expand(b, -1, -1, -1), cache.keys], 2).contiguous()
    v = torch.cat([prefix.values.expand(b, -1, -1, -1), cache.values], 2).contiguous()
    q = torch.randn(b, hq, n, D, device="cuda").bfloat16()
    parents = torch.from_numpy(np.stack([gen.tree_parents(np.random.default_rng(i), n) for i in range(b)])).cuda()
    one = tsb.tree_flash(q, tsb.KVCache(k, v, p_rows + m), D**-0.5, parents=parents)
    two = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents)
    torch.cuda.synchronize()
    # each is off by at most 2^-8 (sum p|v| + |out|), and sum p|v| <= max|v|
    assert (one.float() - two.float()).abs().max() <= 4 * 2.0**-8 * v.float().abs().max()


@pytest.mark.parametrize("fmt,b,n,hq,hkv,p_rows,lengths", [
    ("bf16", 70, 1, 4, 2, 130, [1 + (37 * i) % 90 for i in range(70)]),        # single tokens, many requests to a block
    ("bf16", 40, 3, 3, 3, 5, [3] * 39 + [2500]),                               # one request far longer than the others
    ("bf16", 33, 2, 8, 8, 700, [2 + (101 * i) % 260 for i in range(33)]),      # 264 own units, more than pairs of CTAs
    ("mlx_q8", 12, 32, 6, 1, 64, [32 + 64 * i for i in range(12)]),            # own rows outweigh the prefix
    ("ref_q8", 3, 1, 2, 1, 6000, [900, 1, 0]),                                 # many splits of few rows
    ("bf16", 5, 4, 4, 4, 3000, [0] * 5),                                       # no own rows at all
    ("bf16", 1, 64, 64, 8, 1, [64]),                                           # two row blocks to a request, one prefix row
], ids=lambda v: str(len(v)) if isinstance(v, list) else str(v))
def test_schedules(fmt, b, n, hq, hkv, p_rows, lengths):
    """Splits, chunks and their dealing out to the CTAs at the ends of what is possible."""
    _run(fmt, b, n, hq, hkv, p_rows, lengths, seed=21)


def test_a_request_does_not_touch_another():
    """NaN and infinite queries of one request, whose rows are packed with the others', leave those as they were."""
    import tsb

    b, n, hq, hkv = 6, 5, 4, 2
    prefix, cache, _ = _make("bf16", hkv, b, 400, 90, 400, 90, seed=13)
    q = torch.randn(b, hq, n, D, device="cuda").bfloat16()
    parents = torch.arange(-1, n - 1, device="cuda", dtype=torch.int32)
    lengths = torch.tensor([5, 90, 33, 64, 65, 17], dtype=torch.int32, device="cuda")
    want, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents, lengths=lengths, stats=True)
    bad = q.clone()
    bad[2] = float("nan")
    bad[4, 0, 0, :3] = torch.tensor([float("inf"), -float("inf"), 1.0])
    out, got, _ = tsb.tree_flash_shared(bad, prefix, cache, D**-0.5, parents=parents, lengths=lengths, stats=True)
    torch.cuda.synchronize()
    for i in (0, 1, 3, 5):
        assert torch.equal(out[i], want[i]) and torch.equal(got[i], lse[i])
    assert torch.isnan(out[2]).all() and torch.isnan(got[2]).all()  # not passed off as a row that sees nothing
    assert torch.equal(out[4, 1:], want[4, 1:]) and torch.equal(out[4, 0, 1:], want[4, 0, 1:])


def test_refusals():
    import tsb

    b, n, hq, hkv = 2, 4, 4, 2
    prefix, cache, _ = _make("bf16", hkv, b, 64, 32, 50, 20)
    q8, _, _ = _make("ref_q8", hkv, b, 64, 32, 50, 20)
    q = torch.randn(b, hq, n, D, device="cuda").bfloat16()
    parents = torch.arange(-1, n - 1, device="cuda", dtype=torch.int32)
    lengths = torch.full((b,), 9, dtype=torch.int32, device="cuda")
    call = lambda q=q, prefix=prefix, cache=cache, parents=parents, **kw: tsb.tree_flash_shared(  # noqa: E731
        q, prefix, cache, D**-0.5, parents=parents, **kw)
    assert call() is not None
    assert call(q=q.half()) is None and call(q=q[..., :128]) is None and call(q=q[:, :3]) is None and call(parents=None) is None
    assert call(q=torch.zeros(b, hq, 65, D, device="cuda", dtype=torch.bfloat16), parents=torch.zeros(65, device="cuda", dtype=torch.int32)) is None
    for bad in (lengths.long(), lengths[:1], lengths.cpu(), lengths.repeat(2)[::2]):
        with pytest.raises(ValueError):
            call(lengths=bad)
    with pytest.raises(ValueError):  # mixed formats
        call(prefix=q8)
    with pytest.raises(ValueError):  # a prefix of two requests
        call(prefix=cache)
    with pytest.raises(ValueError):  # a cache of another batch
        call(cache=prefix)
    with pytest.raises(ValueError):
        call(parents=parents[:3])
    with pytest.raises(ValueError):
        call(prefix=tsb.KVCache(prefix.keys, prefix.values, 65))
    with pytest.raises(ValueError):
        call(prefix=tsb.KVCache(prefix.keys[:, :, ::2], prefix.values[:, :, ::2], 3))
    with pytest.raises(ValueError):
        call(cache=tsb.KVCache(cache.keys.half(), cache.values.half(), 3))
    with pytest.raises(ValueError):
        call(out=torch.empty(b, hq, n, D, device="cuda"))
    with pytest.raises(ValueError):
        call(out=torch.empty(b, n, hq, D, device="cuda", dtype=torch.bfloat16).transpose(1, 2))


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_rows_at_all(fmt):
    """Both caches empty, their planes not read: zeros and -inf, where a call is the first to be captured too."""
    import tsb

    prefix, cache, _ = _make(fmt, 2, 3, 4, 4, 0, 0)
    for c in (prefix, cache):
        _poison([t for t in vars(c).values() if isinstance(t, torch.Tensor)], 0)
    q = torch.randn(3, 4, 2, D, device="cuda").bfloat16()
    parents = torch.tensor([-1, 0], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, _ = tsb.tree_flash_shared(q, prefix, cache, D**-0.5, parents=parents, stats=True)
    graph.replay()
    torch.cuda.synchronize()
    assert not out.any() and torch.isneginf(lse).all()
