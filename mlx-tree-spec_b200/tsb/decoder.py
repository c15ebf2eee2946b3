"""The verify-step decoder (the gated-q layer stack) on the library's kernels.

One step runs every layer of a gated-q decoder over the tree nodes of B
requests (M = B*T rows), as mlx-tree-spec's batch_forward does
(src/mlx_tree_spec/tree_verify.py:414-447, attention 311-367, add_rms_norm
fused_ops.py:107-154):

    x = input_norm_0(h)
    per layer:  qkv = x W_qkv^T                     (4-bit qmm; q with gate, k, v)
                q, cache <- qkv_prep(qkv)            (q/k norms, rope at depth, K/V append)
                a = tree_attention(q, cache, parents)
                r = (a * sigmoid(gate)) W_o^T        (attn_gate + 4-bit qmm)
                h, x = add_rms_norm(h, r, post_norm)
                r = swiglu(x W_gate_up^T) W_down^T   (4-bit qmm, swiglu, 4-bit qmm)
                h, x = add_rms_norm(h, r, next input norm | final norm)

Per layer that is four quantized matmuls, one attention and five small
kernels; every buffer is allocated once per (B, T), so a whole step can be
captured in one CUDA graph (no host work inside). Weights are random (config 5
is a synthetic model): N(0, 0.02) quantized to 4-bit g64, norm weights
1 + N(0, 0.1). Rope follows a Qwen3-Next-style partial rotary layout (the
first `rope_dims` of each head, base `rope_base`); the reference reads both
from its model's config.

`step` has all requests at one length. `step_shared` is the same layer stack for
requests that share a long prefix and have their own rows behind it, of lengths
that live on the device; `verify` goes on from there to the LM head, samples a
token at every node, walks the trees and keeps the accepted rows, without a host
read: the lengths it returns are the next step's, plus the next tree.
"""

from __future__ import annotations

from collections import namedtuple
from dataclasses import dataclass

import torch

from . import _lib, ops
from ._lib import TSB_KV_BF16, TSB_KV_MLX_Q8_G64, TSB_KV_REF_Q8_ROW, check
from .cache import KVCache, MLXQ8KVCache, Q8KVCache
from .quant import quantize, quantize_g64, quantize_rows
from .verify import PathCommit, sample, tree_accept

# of VerifyDecoder.verify: tree_accept's path (B, T), n_keep (B,) and next_token (B,), the
# sampled tokens (B, T) and the lengths (B,) after the commit, all int32 on the device
Verified = namedtuple("Verified", "path n_keep next_token samples lengths")


@dataclass
class DecoderConfig:
    layers: int = 16
    hidden: int = 5120
    hq: int = 24
    hkv: int = 4
    d: int = 256
    inter: int = 17408
    eps: float = 1e-6
    rope_dims: int = 64
    rope_base: float = 1e7

    @property
    def qkv_rows(self) -> int:
        return (2 * self.hq + 2 * self.hkv) * self.d


def random_weights(cfg: DecoderConfig, seed: int = 0, device="cuda", std: float = 0.02):
    """Per-layer weights {qkv, o, gate_up, down: (wq, scales, biases); q_norm,
    k_norm, input_norm, post_norm: bf16} and the final norm."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def w(n, k):
        return quantize(torch.randn(n, k, generator=gen, device=device) * std)

    def norm(n):
        return (1.0 + 0.1 * torch.randn(n, generator=gen, device=device)).to(torch.bfloat16)

    layers = []
    for _ in range(cfg.layers):
        layers.append({"qkv": w(cfg.qkv_rows, cfg.hidden), "o": w(cfg.hidden, cfg.hq * cfg.d),
                       "gate_up": w(2 * cfg.inter, cfg.hidden), "down": w(cfg.hidden, cfg.inter),
                       "q_norm": norm(cfg.d), "k_norm": norm(cfg.d),
                       "input_norm": norm(cfg.hidden), "post_norm": norm(cfg.hidden)})
    return layers, norm(cfg.hidden)


def make_cache(kf: torch.Tensor, vf: torch.Tensor, offset: int, kv_format: int = TSB_KV_BF16):
    """A layer's cache from float K/V (B, Hkv, capacity, D) in the given format."""
    if kv_format == TSB_KV_BF16:
        return KVCache(kf.to(torch.bfloat16), vf.to(torch.bfloat16), offset)
    if kv_format == TSB_KV_REF_Q8_ROW:
        kq, ks = quantize_rows(kf)
        vq, vs = quantize_rows(vf)
        return Q8KVCache(kq, vq, ks, vs, offset)
    kw, ks, kb = quantize_g64(kf)
    vw, vs, vb = quantize_g64(vf)
    return MLXQ8KVCache(kw, vw, ks, kb, vs, vb, offset)


def _planes(cache):
    """(k, k_scales, k_biases, v, v_scales, v_biases) of a cache, as ops reads them."""
    fmt = cache.kv_format
    if fmt == TSB_KV_BF16:
        return cache.keys, None, None, cache.values, None, None
    if fmt == TSB_KV_REF_Q8_ROW:
        return cache.keys, cache.k_scale, None, cache.values, cache.v_scale, None
    return cache.keys, cache.k_scales, cache.k_biases, cache.values, cache.v_scales, cache.v_biases


def _ptr(t):
    return None if t is None else t.data_ptr()


class VerifyDecoder:
    """The layer stack over one verify step's nodes."""

    def __init__(self, cfg: DecoderConfig, layers, final_norm):
        self.cfg, self.layers, self.final_norm = cfg, layers, final_norm
        self._bufs: dict = {}

    def _buffers(self, b: int, t: int, device):
        key = (b, t, str(device))
        buf = self._bufs.get(key)
        if buf is None:
            c, m = self.cfg, b * t
            e = lambda *shape, dt=torch.bfloat16: torch.empty(*shape, dtype=dt, device=device)  # noqa: E731
            buf = {"h": e(m, c.hidden), "x": e(m, c.hidden), "r": e(m, c.hidden), "qkv": e(m, c.qkv_rows),
                   "q": e(b, c.hq, t, c.d), "attn": e(b, c.hq, t, c.d), "gated": e(m, c.hq * c.d),
                   "gu": e(m, 2 * c.inter), "act": e(m, c.inter),
                   "positions": e(m, dt=torch.int32), "offsets": e(b, dt=torch.int32)}
            self._bufs[key] = buf
        return buf

    def step(self, h_in: torch.Tensor, parents: torch.Tensor, caches, prefix: int) -> torch.Tensor:
        """h_in (B*T, hidden) bf16 hidden states of the nodes (request-major);
        parents int32 (B, T); caches: one per layer, holding `prefix` rows per
        request and room for T more (their offset is set to prefix + T). The
        nodes' K/V are written at rows prefix .. prefix+T-1. Returns the final
        normed hidden states (B*T, hidden), a buffer reused by the next step."""
        b, t = parents.shape
        buf = self._buffers(b, t, h_in.device)
        _, depth = ops.ancestor_bits(parents, depth=True)
        buf["positions"].copy_((depth + prefix).reshape(-1))
        buf["offsets"].fill_(prefix)

        def attend(i, q, cache, scale, out):
            return ops.tree_flash(q, cache, scale, parents=parents, out=out)

        for cache in caches[:len(self.layers)]:
            cache.offset = prefix + t
        return self._layer_loop(h_in, b, t, buf, caches, attend)

    def step_shared(self, h_in: torch.Tensor, parents: torch.Tensor, prefixes, caches,
                    lengths: torch.Tensor) -> torch.Tensor:
        """step for requests that share a prefix: prefixes, one cache of batch 1
        per layer (all of one offset P), and each request's own rows in caches,
        one per layer with the prefix's format. lengths int32 (B,) on the device:
        a request's own rows with this step's T nodes, whose K/V are written at
        own rows lengths[b] - T .. lengths[b] - 1 and which stand at positions
        P + lengths[b] - T + depth. caches[i].offset bounds the lengths and is left
        as it is (the capacity will do). The lengths are read on the device, so a
        captured step serves every later one; they must lie in [T, offset] (rows
        outside the cache are not written, whatever the lengths are)."""
        b, t = parents.shape
        shared = int(prefixes[0].offset)
        if any(int(p.offset) != shared for p in prefixes):
            raise ValueError("step_shared: every layer's prefix must have the same rows")
        if len(prefixes) != len(self.layers) or len(caches) != len(self.layers):
            raise ValueError(f"step_shared: {len(self.layers)} layers need as many prefixes and caches")
        if (lengths.dtype != torch.int32 or lengths.shape != (b,) or not lengths.is_contiguous()
                or lengths.device != h_in.device):
            raise ValueError(f"step_shared: lengths must be a contiguous int32 tensor ({b},) on {h_in.device}")
        # a layer's rows are written before its attention looks at the caches
        for prefix, cache in zip(prefixes, caches):
            pre, own = ops._kv_planes(prefix), ops._kv_planes(cache)
            if pre[0] != own[0]:
                raise ValueError("step_shared: a layer's prefix and cache must share a format")
            ops._kv_struct("step_shared", prefix, pre, 1, self.cfg.hkv, self.cfg.d, h_in.device)
            ops._kv_struct("step_shared", cache, own, b, self.cfg.hkv, self.cfg.d, h_in.device)
        buf = self._buffers(b, t, h_in.device)
        _, depth = ops.ancestor_bits(parents, depth=True)
        torch.sub(lengths, t, out=buf["offsets"])
        buf["positions"].copy_((depth + (buf["offsets"] + shared)[:, None]).reshape(-1))

        def attend(i, q, cache, scale, out):
            return ops.tree_flash_shared(q, prefixes[i], cache, scale, parents=parents, lengths=lengths, out=out)

        return self._layer_loop(h_in, b, t, buf, caches, attend)

    def verify(self, h_in: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, prefixes, caches,
               lengths: torch.Tensor, lm_head, u: torch.Tensor, commit, temperature=1.0, top_k=0, top_p=1.0,
               min_p=0.0) -> Verified:
        """A whole verify step: step_shared, the LM head (lm_head: its quantized
        (wq, scales, biases)), a token drawn at every node with the random numbers u
        (B, T) (tsb.sample's filters; one value per node where a tensor), the walk
        along the drafted tokens (B, T), and the commit of the accepted rows.
        commit: PathCommit(caches), made once; a plan of other tensors than these
        caches' raises, before anything is written. Nothing is read on the host, so the
        step can be captured and replayed."""
        if isinstance(commit, PathCommit) and not commit.is_of(caches):
            raise ValueError("verify: commit must be the plan of these caches' tensors (PathCommit(caches))")
        b, t = parents.shape
        x = self.step_shared(h_in, parents, prefixes, caches, lengths)
        logits = ops.quantized_matmul(x, *lm_head)
        if logits is None:
            raise RuntimeError("the quantized matmul declined the LM head's shape")
        samples = sample(logits.view(b, t, -1), u, temperature, top_k, top_p, min_p)
        if samples is None:
            raise ValueError("verify: the vocabulary is larger than tsb.sample takes")
        path, n_keep, next_token = tree_accept(tokens, parents, samples)
        return Verified(path, n_keep, next_token, samples, commit(lengths, path, n_keep))

    def _layer_loop(self, h_in, b: int, t: int, buf, caches, attend) -> torch.Tensor:
        c = self.cfg
        m = b * t
        lib = _lib.load()
        st = torch.cuda.current_stream(h_in.device).cuda_stream
        h, x, r = buf["h"], buf["x"], buf["r"]
        h.copy_(h_in)
        check(lib.tsb_add_rms_norm(_ptr(h), None, _ptr(self.layers[0]["input_norm"]), None, _ptr(x), m, c.hidden,
                                   c.eps, st), "tsb_add_rms_norm")
        scale = c.d ** -0.5
        for i, lw in enumerate(self.layers):
            cache = caches[i]
            k, ks, kb, v, vs, vb = _planes(cache)
            ops.quantized_matmul_into(x, *lw["qkv"], buf["qkv"], c.qkv_rows)
            check(lib.tsb_qkv_prep(_ptr(buf["qkv"]), c.qkv_rows, b, t, c.hq, c.hkv, c.d, _ptr(lw["q_norm"]),
                                   _ptr(lw["k_norm"]), c.eps, _ptr(buf["positions"]), c.rope_dims, c.rope_base, 1.0,
                                   _ptr(buf["q"]), cache.kv_format, _ptr(k), _ptr(ks), _ptr(kb), _ptr(v), _ptr(vs),
                                   _ptr(vb), k.shape[2], _ptr(buf["offsets"]), st), "tsb_qkv_prep")
            if attend(i, buf["q"], cache, scale, buf["attn"]) is None:
                raise RuntimeError("tree attention declined the decoder's shape")
            check(lib.tsb_attn_gate(_ptr(buf["attn"]), _ptr(buf["qkv"]), c.qkv_rows, _ptr(buf["gated"]), b, t, c.hq,
                                    c.d, st), "tsb_attn_gate")
            ops.quantized_matmul_into(buf["gated"], *lw["o"], r, c.hidden)
            check(lib.tsb_add_rms_norm(_ptr(h), _ptr(r), _ptr(lw["post_norm"]), _ptr(h), _ptr(x), m, c.hidden, c.eps,
                                       st), "tsb_add_rms_norm")
            ops.quantized_matmul_into(x, *lw["gate_up"], buf["gu"], 2 * c.inter)
            check(lib.tsb_swiglu(_ptr(buf["gu"]), _ptr(buf["act"]), m, c.inter, st), "tsb_swiglu")
            ops.quantized_matmul_into(buf["act"], *lw["down"], r, c.hidden)
            nxt = self.layers[i + 1]["input_norm"] if i + 1 < len(self.layers) else self.final_norm
            check(lib.tsb_add_rms_norm(_ptr(h), _ptr(r), _ptr(nxt), _ptr(h), _ptr(x), m, c.hidden, c.eps, st),
                  "tsb_add_rms_norm")
        return x


__all__ = ["DecoderConfig", "random_weights", "make_cache", "VerifyDecoder", "Verified",
           "TSB_KV_BF16", "TSB_KV_MLX_Q8_G64", "TSB_KV_REF_Q8_ROW"]
