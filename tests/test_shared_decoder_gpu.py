"""The decoder over requests that share a prefix, and a whole verify step: the
layer stack, the LM head, the sampled tokens, the walk and the commit.

The layer stack is held to the oracle's layer loop over each request's
concatenated rows, by the bar of the unshared step (2e-2 * max|ref|): the same
layers in the same precisions, with the attention's weights in one more float32
merge. What follows the logits is exact: integers from the logits at hand."""

import numpy as np
import pytest
import torch

from gpu_util import assert_close_rel, host_f32
from oracle import bf16 as obf16
from oracle import decoder as odec
from oracle import gen, kv
from oracle import verify as overify

pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "mlx_q8", "ref_q8"]


def _bf(t):
    return obf16.from_torch_bf16(t.cpu())


def _w_np(w):
    wq, s, b = w
    return wq.cpu().numpy().view(np.uint32), _bf(s), _bf(b)


def _code(fmt):
    import tsb

    return {"bf16": tsb.TSB_KV_BF16, "mlx_q8": tsb.TSB_KV_MLX_Q8_G64, "ref_q8": tsb.TSB_KV_REF_Q8_ROW}[fmt]


def _values(cache, fmt):
    """(keys, values) that a cache holds, as float64."""
    if fmt == "bf16":
        return [host_f32(t).astype(np.float64) for t in (cache.keys, cache.values)]
    if fmt == "ref_q8":
        return [q.cpu().numpy().astype(np.float64) * s.cpu().numpy().astype(np.float64)[..., None]
                for q, s in ((cache.keys, cache.k_scale), (cache.values, cache.v_scale))]
    return [kv.dequant_g64(w.cpu().numpy().view(np.uint32), _bf(s), _bf(b)).astype(np.float64)
            for w, s, b in ((cache.keys, cache.k_scales, cache.k_biases), (cache.values, cache.v_scales, cache.v_biases))]


def _planes(cache):
    return [t for t in vars(cache).values() if isinstance(t, torch.Tensor)]


def _setup(fmt, b, t, prefix, cap, layers=2, hq=4, hkv=1, seed=5):
    from tsb import decoder as tdec

    cfg = tdec.DecoderConfig(layers=layers, hidden=1024, hq=hq, hkv=hkv, d=256, inter=1024)
    weights, final_norm = tdec.random_weights(cfg, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)

    def cache(batch, rows, offset):
        k, v = (torch.randn(batch, hkv, rows, 256, device="cuda", generator=g) for _ in range(2))
        return tdec.make_cache(k, v, offset, _code(fmt))

    prefixes = [cache(1, prefix + 3, prefix) for _ in range(layers)]
    caches = [cache(b, cap, cap) for _ in range(layers)]
    rng = np.random.default_rng(seed)
    parents = np.stack([gen.tree_parents(rng, t) for _ in range(b)]).astype(np.int32)
    h0 = torch.randn(b * t, cfg.hidden, device="cuda", generator=g).to(torch.bfloat16)
    return cfg, weights, final_norm, tdec.VerifyDecoder(cfg, weights, final_norm), prefixes, caches, parents, h0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,prefix,lengths", [(8, 200, [8, 70, 33]), (1, 64, [1, 40, 64]), (5, 0, [5, 9, 61])])
def test_step_shared(fmt, t, prefix, lengths):
    b, cap = len(lengths), 72
    cfg, weights, final_norm, dec, prefixes, caches, parents, h0 = _setup(fmt, b, t, prefix, cap)
    ref = []
    for p, c in zip(prefixes, caches):
        pair = []
        for shared, own in zip(_values(p, fmt), _values(c, fmt)):
            pair.append(np.concatenate([np.repeat(shared[:, :, :prefix], b, axis=0), own], axis=2))
        ref.append(pair)
    before = [[x.clone() for x in _planes(c)] for c in caches]
    kept = [[x.clone() for x in _planes(p)] for p in prefixes]
    out = dec.step_shared(h0, torch.from_numpy(parents).cuda(), prefixes, caches,
                          torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    ocfg = {"hq": cfg.hq, "hkv": cfg.hkv, "d": cfg.d, "eps": cfg.eps, "rope_dims": cfg.rope_dims,
            "rope_base": cfg.rope_base}
    h = host_f32(h0)
    _, x = odec.rms_norm(h, host_f32(weights[0]["input_norm"]), cfg.eps)
    offsets = [prefix + n - t for n in lengths]
    for i, lw in enumerate(weights):
        p = {name: _w_np(lw[name]) for name in ("qkv", "o", "gate_up", "down")}
        p.update({name: host_f32(lw[name]) for name in ("q_norm", "k_norm", "post_norm")})
        nxt = host_f32(weights[i + 1]["input_norm"]) if i + 1 < len(weights) else host_f32(final_norm)
        h, x = odec.layer_step(h, x, p, *ref[i], parents, offsets, ocfg, nxt, kv_format=fmt)
    assert_close_rel(host_f32(out), x, 2e-2, f"shared decoder {fmt}")
    for c, old, p, same in zip(caches, before, prefixes, kept):  # only the nodes' rows were written
        for now, then in zip(_planes(c), old):
            for r, n in enumerate(lengths):
                assert torch.equal(now[r, :, :n - t], then[r, :, :n - t])
                assert torch.equal(now[r, :, n:], then[r, :, n:])
        assert all(torch.equal(a, z) for a, z in zip(_planes(p), same))


@pytest.mark.parametrize("fmt", ["bf16", "mlx_q8"])
def test_step_shared_rows_outside_the_cache(fmt):
    """Requests whose lengths leave no room for their nodes (padding of a batch, or
    past the capacity): rows outside their caches are not written, and the other
    requests' rows are what they are without them."""
    b, t, prefix, cap = 4, 4, 100, 24
    lengths = [0, 2, cap + 3, 20]  # rows -4..-1, -2..1, 23..26, 16..19
    cfg, _, _, dec, prefixes, caches, parents, h0 = _setup(fmt, b, t, prefix, cap)
    before = [[x.clone() for x in _planes(c)] for c in caches]
    dec.step_shared(h0, torch.from_numpy(parents).cuda(), prefixes, caches,
                    torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    written = [[], [0, 1], [23], [16, 17, 18, 19]]
    for c, old in zip(caches, before):
        for now, then in zip(_planes(c), old):
            for r in range(b):
                same = [i for i in range(cap) if i not in written[r]]
                assert torch.equal(now[r, :, same], then[r, :, same])


def _lm_head(vocab, hidden, seed=21):
    import tsb

    g = torch.Generator(device="cuda").manual_seed(seed)
    return tsb.quantize(torch.randn(vocab, hidden, generator=g, device="cuda") * 0.02)


@pytest.mark.parametrize("fmt,temperature", [("bf16", 0.0), ("mlx_q8", 0.7), ("ref_q8", 0.7)])
def test_verify_steps_captured(fmt, temperature):
    """Three verify steps, each as a replay of one captured graph, equal the same
    steps run eagerly, and their integers are the oracle's for the sampled tokens."""
    import tsb

    b, t, prefix, cap, vocab = 3, 6, 130, 96, 2048
    cfg, _, _, dec, prefixes, caches, parents_np, _ = _setup(fmt, b, t, prefix, cap)
    eager_dec = type(dec)(cfg, dec.layers, dec.final_norm)
    head = _lm_head(vocab, cfg.hidden)
    copies = [type(c)(**{k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in vars(c).items()}) for c in caches]
    commit, commit_e = tsb.PathCommit(caches), tsb.PathCommit(copies)
    g = torch.Generator(device="cuda").manual_seed(77)
    parents = torch.from_numpy(parents_np).cuda()
    h = torch.empty(b * t, cfg.hidden, device="cuda", dtype=torch.bfloat16)
    tokens = torch.zeros(b, t, dtype=torch.int32, device="cuda")
    u = torch.zeros(b, t, device="cuda")
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")

    def run(d, cs, cm, n):
        return d.verify(h, tokens, parents, prefixes, cs, n, head, u, cm, temperature=temperature, top_k=40, top_p=0.9)

    def fill():
        h.copy_(torch.randn(h.shape, device="cuda", generator=g))
        u.copy_(torch.rand(u.shape, device="cuda", generator=g))

    # a captured call's kernels must have run once before (attributes, addresses)
    lengths.copy_(torch.tensor([t, 40, 17], dtype=torch.int32))
    scratch = [type(c)(**{k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in vars(c).items()}) for c in caches]
    fill()
    run(dec, scratch, tsb.PathCommit(scratch), lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(dec, caches, commit, lengths)
    now = lengths.clone()
    for step in range(3):
        fill()
        # drafts that partly come true: the tokens that would be drawn, at some nodes
        peek = [type(c)(**{k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in vars(c).items()}) for c in copies]
        drawn = run(eager_dec, peek, tsb.PathCommit(peek), now).samples
        par = parents.clamp(min=0).long()
        tokens.copy_(torch.where(torch.rand(b, t, device="cuda", generator=g) < 0.8, torch.gather(drawn, 1, par), 7))
        want = run(eager_dec, copies, commit_e, now)
        lengths.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, want):
            assert torch.equal(a, e)
        for c, d in zip(caches, copies):
            assert all(torch.equal(x, y) for x, y in zip(_planes(c), _planes(d)))
        for r in range(b):
            path, nxt = overify.tree_accept(tokens[r].tolist(), parents[r].tolist(), want.samples[r].tolist())
            n = int(want.n_keep[r])
            assert want.path[r].tolist() == path + [-1] * (t - len(path)) and n == len(path)
            assert int(want.next_token[r]) == nxt and int(want.lengths[r]) == int(now[r]) - t + n
        now = want.lengths + t
    assert int((want.n_keep > 1).sum()) > 0  # the last trees were walked below their roots


def test_step_shared_refusals():
    b, t = 2, 4
    cfg, _, _, dec, prefixes, caches, parents, h0 = _setup("bf16", b, t, 64, 32)
    par = torch.from_numpy(parents).cuda()
    n = torch.full((b,), 8, dtype=torch.int32, device="cuda")
    for bad in (n.long(), n[:1], n.cpu()):
        with pytest.raises(ValueError):
            dec.step_shared(h0, par, prefixes, caches, bad)
    with pytest.raises(ValueError):
        dec.step_shared(h0, par, prefixes[:1], caches, n)
    prefixes[1].offset = 63
    with pytest.raises(ValueError):
        dec.step_shared(h0, par, prefixes, caches, n)
