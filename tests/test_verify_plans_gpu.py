"""Commit plans over caches of several capacities, and what a verify step with the
wrong plan leaves behind: moved bytes, equal to the oracle's."""

import numpy as np
import pytest
import torch

from oracle import kv

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "mlx_q8", "ref_q8"]


def _cache(fmt, b, hkv, cap, seed):
    import tsb
    from tsb.decoder import make_cache

    g = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(b, hkv, cap, 256, generator=g, device="cuda") for _ in range(2))
    return make_cache(k, v, cap, {"bf16": tsb.TSB_KV_BF16, "mlx_q8": tsb.TSB_KV_MLX_Q8_G64, "ref_q8": tsb.TSB_KV_REF_Q8_ROW}[fmt])


def _bytes(cache):
    return {n: t.cpu().reshape(*t.shape[:3], -1).contiguous().view(torch.uint8).numpy().copy()
            for n, t in vars(cache).items() if isinstance(t, torch.Tensor)}


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("caps", [(40, 24), (24, 40), (24, 40, 24, 33)])
def test_commit_over_capacities(fmt, caps):
    """A request is moved in every cache or in none: in none where its length fits some
    capacities only, whichever cache comes first."""
    import tsb

    b, t = 6, 5
    lengths = [5, 24, 25, 40, 41, 3]
    paths = [[0, 2, 4], [1, 3], [0, 1, 4], [2, 3], [0, 4], [1, 2]]
    caches = [_cache(fmt, b, 2, cap, i) for i, cap in enumerate(caps)]
    want = [_bytes(c) for c in caches]
    moved = [i for i, n in enumerate(lengths) if t <= n <= min(caps)]
    for w in want:
        for raw in w.values():
            for i in moved:
                raw[i:i + 1] = kv.take_rows(raw[i:i + 1], lengths[i] - t, paths[i])
    path = np.full((b, t), -1, np.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    cur = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    keep = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
    new = tsb.PathCommit(caches)(cur, torch.from_numpy(path).cuda(), keep)
    torch.cuda.synchronize()
    assert cur.tolist() == lengths
    assert new.tolist() == [n - t + len(paths[i]) if i in moved else n for i, n in enumerate(lengths)]
    for c, w in zip(caches, want):
        got = _bytes(c)
        for name in w:
            assert np.array_equal(got[name], w[name]), name


def test_commit_over_capacities_captured():
    """The same by replays of one graph, with lengths of their own."""
    import tsb

    b, t = 4, 3
    caches = [_cache(f, b, 1, cap, i) for i, (f, cap) in enumerate((("bf16", 20), ("ref_q8", 12)))]
    plan = tsb.PathCommit(caches)
    cur = torch.zeros(b, dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 2, -1]] * b, dtype=torch.int32, device="cuda")
    keep = torch.full((b,), 2, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        new = plan(cur, path, keep)
    for lengths in ([3, 12, 13, 20], [12, 0, 21, 5], [7, 8, 9, 10]):
        want = [_bytes(c) for c in caches]
        cur.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert new.tolist() == [n - 1 if 3 <= n <= 12 else n for n in lengths]
        for c, w in zip(caches, want):
            got = _bytes(c)
            for name, raw in w.items():
                for i, n in enumerate(lengths):
                    if 3 <= n <= 12:
                        raw[i:i + 1] = kv.take_rows(raw[i:i + 1], n - t, [0, 2])
                assert np.array_equal(got[name], raw), (name, lengths)
