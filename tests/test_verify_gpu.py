"""The walk down the drafted tree and the commit by device paths: whole numbers
and moved bytes, equal to the oracle's."""

import numpy as np
import pytest
import torch

from oracle import gen, kv, verify as oracle

pytestmark = pytest.mark.gpu


def _tree(rng, t, hit=0.6):
    parents = gen.tree_parents(rng, t)
    parents[1:] = np.where(parents[1:] < 0, 0, parents[1:])
    tokens = rng.integers(0, 50, t).astype(np.int32)
    samples = rng.integers(0, 50, t).astype(np.int32)
    for i in range(1, t):
        if rng.random() < hit:
            samples[parents[i]] = tokens[i]
    return parents, tokens, samples


def _accept(parents, tokens, samples):
    import tsb

    path, n, nxt = tsb.tree_accept(*(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (tokens, parents, samples)))
    return path.cpu().numpy(), n.cpu().numpy(), nxt.cpu().numpy()


def _check_accept(parents, tokens, samples):
    path, n, nxt = _accept(parents, tokens, samples)
    for b in range(len(n)):
        want, after = oracle.tree_accept(tokens[b], parents[b], samples[b])
        assert n[b] == len(want) and list(path[b, :n[b]]) == want and (path[b, n[b]:] == -1).all()
        assert nxt[b] == after


@pytest.mark.parametrize("b,t", [(1, 1), (1, 2), (3, 31), (5, 32), (6, 33), (70, 64), (257, 7)])
def test_accept(b, t):
    rng = np.random.default_rng(b * 100 + t)
    trees = [_tree(rng, t) for _ in range(b)]
    _check_accept(*(np.stack(x) for x in zip(*trees)))


def test_accept_whole_chains_and_nothing():
    t = 64
    parents = np.tile(gen.chain_parents(t), (2, 1))
    tokens = np.tile(np.arange(t, dtype=np.int32), (2, 1))
    samples = tokens + 1
    samples[1] = 999
    _check_accept(parents, tokens, samples)


def test_accept_equal_siblings_padding_and_bad_parents():
    # equal drafted tokens below one node: the lowest counts, and only its own subtree goes on
    parents = np.array([[-1, 0, 0, 1, 2], [-1, 0, 1, 2, 3], [-1, -1, -1, -1, -1], [-1, 4, 0, 2, 9]], np.int32)
    tokens = np.array([[9, 5, 5, 6, 6], [9, 1, 2, 3, 4], [9, -1, -1, -1, -1], [9, 5, 5, 7, 8]], np.int32)
    samples = np.array([[5, 6, 6, 0, 0], [1, 2, -1, 4, 5], [-1, -1, -1, -1, -1], [5, 6, 7, 8, 8]], np.int32)
    _check_accept(parents, tokens, samples)
    path, n, nxt = _accept(parents, tokens, samples)
    assert list(path[0, :3]) == [0, 1, 3] and n[1] == 3 and nxt[1] == -1 and n[2] == 1
    assert list(path[3, :n[3]]) == [0, 2, 3]  # node 1 names a later node as its parent, node 4 none of the tree


def test_accept_types_and_empty():
    import tsb

    parents, tokens, samples = (torch.from_numpy(a)[None].cuda() for a in _tree(np.random.default_rng(0), 20))
    want = tsb.tree_accept(tokens, parents, samples)
    got = tsb.tree_accept(tokens.long(), parents.long(), samples.long())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    path, n, nxt = tsb.tree_accept(tokens[:0], parents[:0], samples[:0])
    assert path.shape == (0, 20) and n.shape == (0,) and nxt.shape == (0,)


# ---------------------------------------------------------------- commit

def _cache(fmt, b, hkv, cap, seed):
    from tsb.decoder import TSB_KV_BF16, TSB_KV_MLX_Q8_G64, TSB_KV_REF_Q8_ROW, make_cache

    g = torch.Generator().manual_seed(seed)
    kf, vf = torch.randn(b, hkv, cap, 256, generator=g).cuda(), torch.randn(b, hkv, cap, 256, generator=g).cuda()
    return make_cache(kf, vf, cap, {"bf16": TSB_KV_BF16, "mlx_q8": TSB_KV_MLX_Q8_G64, "ref_q8": TSB_KV_REF_Q8_ROW}[fmt])


def _tensors(cache):
    return {k: t for k, t in vars(cache).items() if isinstance(t, torch.Tensor)}


def _bytes(t):
    return t.contiguous().cpu().view(torch.uint8).numpy()


def _want(cache, lengths, paths, t):
    out = {}
    for name, x in _tensors(cache).items():
        raw = _bytes(x.reshape(*x.shape[:3], -1))
        new = raw.copy()
        for b, (m, p) in enumerate(zip(lengths, paths)):
            new[b:b + 1] = kv.take_rows(raw[b:b + 1], m - t, p) if p else raw[b:b + 1]
        out[name] = new
    return out


def _commit_case(fmts, b, t, cap, lengths, paths, keep=None, hkv=2, expect=None, new=None):
    import tsb

    caches = [_cache(f, b, hkv, cap, i) for i, f in enumerate(fmts)]
    want = [_want(c, lengths, expect or paths, t) for c in caches]
    path = np.full((b, t), -1, np.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    n = np.array(keep if keep is not None else [len(p) for p in paths], np.int32)
    dev = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    plan = tsb.PathCommit(caches)
    cur = dev(lengths)
    got = plan(cur, dev(path), dev(n))
    torch.cuda.synchronize()
    assert cur.tolist() == list(lengths)
    kept = [len(p) for p in (expect or paths)]
    assert got.tolist() == (new or [m - t + k for m, k in zip(lengths, kept)])
    for c, w in zip(caches, want):
        for name, x in _tensors(c).items():
            assert np.array_equal(_bytes(x.reshape(*x.shape[:3], -1)), w[name]), name


@pytest.mark.parametrize("fmt", ["bf16", "mlx_q8", "ref_q8"])
@pytest.mark.parametrize("b,t,cap", [(1, 1, 1), (2, 4, 9), (9, 33, 77), (3, 64, 130), (40, 8, 64)])
def test_commit_paths(fmt, b, t, cap):
    rng = np.random.default_rng(b + t)
    lengths = rng.integers(t, cap + 1, b)
    lengths[0] = t
    lengths[-1] = cap
    paths = [sorted(rng.choice(t, rng.integers(0, t + 1), replace=False).tolist()) for _ in range(b)]
    _commit_case([fmt, fmt], b, t, cap, lengths.tolist(), paths)


def test_commit_whole_and_last_node():
    t = 64
    _commit_case(["bf16"], 4, t, 100, [64, 100, 70, 80], [list(range(t)), list(range(1, t)), [63], []])


def test_commit_mixed_formats_and_many_layers():
    _commit_case(["bf16", "mlx_q8", "ref_q8", "bf16"], 3, 6, 40, [6, 20, 40], [[0, 2, 5], [0], [0, 1, 2, 3]])
    _commit_case(["ref_q8"] * 50, 2, 5, 16, [5, 16], [[0, 3], [0, 1, 4]])  # more layers than one launch takes


def test_commit_paths_that_end_early_and_lengths_out_of_range():
    # counts past the path's valid part: it ends at -1, past the tree, or where it stops increasing
    _commit_case(["bf16", "mlx_q8"], 5, 6, 30, [6, 12, 30, 20, 9], [[0, 2, -1, 4], [0, 3, 6], [1, 4, 4, 5], [2, 1], [0, 1, 2]],
                 keep=[4, 3, 4, 2, 99], expect=[[0, 2], [0, 3], [1, 4], [2], [0, 1, 2]])
    _commit_case(["bf16", "ref_q8"], 4, 6, 30, [5, 31, -7, 10], [[0, 2], [0, 2], [0, 2], [0, 2]], keep=[2, 2, 2, -3],
                 expect=[[], [], [], []], new=[5, 31, -7, 4])


def test_commit_agrees_with_host_commit():
    import tsb

    paths = [[0, 3, 4], [0, 1]]
    a, b = _cache("mlx_q8", 2, 2, 50, 1), _cache("mlx_q8", 2, 2, 50, 1)
    offs = tsb.commit([a], [20, 30], paths)[0]
    path = torch.tensor([[0, 3, 4, -1, -1], [0, 1, -1, -1, -1]], dtype=torch.int32, device="cuda")
    new = tsb.commit_paths([b], torch.tensor([25, 35], device="cuda"), path, torch.tensor([3, 2], device="cuda"))
    torch.cuda.synchronize()
    assert new.tolist() == offs
    for (_, x), (_, y) in zip(sorted(_tensors(a).items()), sorted(_tensors(b).items())):
        assert torch.equal(x, y)


def test_commit_refusals():
    import tsb

    c = _cache("bf16", 2, 2, 20, 0)
    for bad in ([], [c, c], [c, _cache("bf16", 3, 2, 20, 0)], [tsb.KVCache(c.keys, c.keys, 20)],
                [tsb.KVCache(c.keys[:, :, ::2], c.values[:, :, ::2], 10)], [tsb.KVCache(c.keys[..., :128].contiguous(), c.values[..., :128].contiguous(), 20)]):
        with pytest.raises(ValueError):
            tsb.PathCommit(bad)
    plan = tsb.PathCommit([c])
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for args in ((i(3), i(2, 4), i(2)), (i(2), i(2, 65), i(2)), (i(2), i(2, 4), i(1)), (i(2), i(4), i(2)), (i(2), i(2, 0), i(2))):
        with pytest.raises(ValueError):
            plan(*args)


def test_accept_and_commit_captured():
    """Sample, walk and commit in one graph, replayed on other logits: no host read in between."""
    import tsb

    b, t, vocab, cap = 3, 12, 501, 64
    rng = np.random.default_rng(5)
    parents = np.stack([_tree(rng, t)[0] for _ in range(b)])
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens = torch.randint(0, vocab, (b, t), generator=g, device="cuda", dtype=torch.int32)
    dpar = torch.from_numpy(parents).cuda()
    sets = []
    for i in range(3):
        x = torch.randn(b, t, vocab, device="cuda", generator=g)
        child = torch.from_numpy(parents.astype(np.int64)).cuda()
        for c in range(1, t):  # a drafted child's token is likely
            x[torch.arange(b), child[:, c], tokens[:, c].long()] += 8.0
        sets.append((x, torch.rand(b, t, device="cuda", generator=g), torch.randint(t, cap + 1, (b,), generator=g, device="cuda", dtype=torch.int32)))
    caches = [_cache(f, b, 2, cap, i) for i, f in enumerate(("bf16", "mlx_q8"))]
    first = [{k: v.clone() for k, v in _tensors(c).items()} for c in caches]
    plan = tsb.PathCommit(caches)
    hx, hu, hl = (s.clone() for s in sets[0])

    def step():
        picked = tsb.sample(hx, hu, 0.9, 50, 0.95)
        path, n, nxt = tsb.tree_accept(tokens, dpar, picked)
        return picked, path, n, nxt, plan(hl, path, n)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        res = step()
    for x, u, m in sets:
        for h, s in zip((hx, hu, hl), (x, u, m)):
            h.copy_(s)
        for c, f in zip(caches, first):
            for k, v in _tensors(c).items():
                v.copy_(f[k])
        graph.replay()
        torch.cuda.synchronize()
        picked, path, n, nxt, new = (r.cpu().numpy() for r in res)
        paths = []
        for i in range(b):
            for j in range(t):
                tok, _, margin = oracle.sample(x[i, j].double().cpu().numpy(), float(u[i, j]), 0.9, 50, 0.95)
                assert picked[i, j] == tok or margin < 1e-9
            p, after = oracle.tree_accept(tokens[i].cpu().numpy(), parents[i], picked[i])
            assert list(path[i, :n[i]]) == p and nxt[i] == after
            paths.append(p)
        lens = m.tolist()
        assert new.tolist() == [k - t + len(p) for k, p in zip(lens, paths)]
        for c, f in zip(caches, first):
            for name, v in _tensors(c).items():
                old = _bytes(f[name].reshape(*v.shape[:3], -1))
                want = old.copy()
                for i, (k, p) in enumerate(zip(lens, paths)):
                    want[i:i + 1] = kv.take_rows(old[i:i + 1], k - t, p)
                assert np.array_equal(_bytes(v.reshape(*v.shape[:3], -1)), want), name
