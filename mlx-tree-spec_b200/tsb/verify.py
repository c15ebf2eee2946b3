"""What follows a verify pass, on the device from the logits to the caches.

  sample(logits, u, temperature, top_k, top_p, min_p)   a token for every tree node
  tree_accept(tokens, parents, samples)                 the accepted path of each request's tree
  PathCommit(caches)(lengths, path, n_keep)             those rows kept in every layer's cache

Verifying by sampling: a token is drawn from the model's own distribution at
every node of the drafted tree, and the walk from the root follows the drafted
child that equals the token drawn at its parent, so the emitted tokens are
distributed as if they had been decoded one by one. The reference does the
walk and the commit's indices on the host (mlx-tree-spec
src/mlx_tree_spec/tree_verify.py:499-516); here no step reads the device, so
the whole of a verify step can be one captured graph.

As in tsb.ops, an unsupported shape or type returns None, a contract violation
raises, and work is enqueued on torch's current stream of the tensors' device.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import TSB_EUNSUPPORTED, TSB_MASK_BF16, TSB_MASK_F16, TSB_MASK_F32, check
from .ops import _GET_DEVICE, _check_planes, _kv_planes, _ptr, _require_cuda, _stream

_LOGIT_TYPES = {torch.bfloat16: TSB_MASK_BF16, torch.float16: TSB_MASK_F16, torch.float32: TSB_MASK_F32}
_MAX_LAYERS_PER_LAUNCH = 48
_MAX_VOCAB = 1 << 20


def _per_row(v, rows: int, dtype, name: str, device):
    """A sampling parameter: (device pointer or None, scalar, what keeps the pointer alive)."""
    if not isinstance(v, torch.Tensor):
        return None, v, None
    if v.device != device:
        raise ValueError(f"sample: {name} must be on {device}")
    if v.numel() != rows:
        raise ValueError(f"sample: {name} must have one value per row ({rows}), got {tuple(v.shape)}")
    if v.dtype != dtype:
        if dtype == torch.int32 and v.dtype == torch.int64:
            v = v.clamp(0, 2**31 - 1)  # a larger top_k is as good as none
        v = v.to(dtype)
    if not v.is_contiguous():
        v = v.contiguous()
    return v.data_ptr(), 0, v


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprobs: bool = False):
    """One token per row of logits (..., V), bf16, fp16 or float32, with the
    random numbers u (...,) float32 in [0, 1).

    Order a row's tokens by logit, equal ones by index; w_i = exp((x_i - max) /
    temperature). Of that order the first top_k are kept, of those the shortest
    prefix whose weight reaches top_p times theirs, of those the tokens with
    w_i >= min_p (always the first). The token is the first kept one whose
    cumulative weight exceeds u times the kept weight: u near 0 gives the likeliest.
    temperature 0 is greedy. top_k <= 0, top_p >= 1 and min_p <= 0 are off; top_p <= 0 leaves the first token.
    Each parameter is a number or a tensor of one value per row.

    Returns int32 tokens (...,), or (tokens, logprobs) with float32 log
    probabilities under the filtered distribution. Logits of -inf or NaN are
    never chosen; a row of nothing else gives -1 and -inf. None where the type
    or V (> 2^20) is not taken."""
    dt = _LOGIT_TYPES.get(logits.dtype)
    if not logits.is_cuda:
        raise ValueError("tsb operators take CUDA tensors (there is no CPU path)")
    if dt is None or logits.dim() < 1:
        return None
    dev = logits.device
    if dev.index != _GET_DEVICE():
        with torch.cuda.device(dev):
            return sample(logits, u, temperature, top_k, top_p, min_p, logprobs)
    *lead, vocab = logits.shape
    if vocab < 1:
        raise ValueError("sample: logits have no tokens")
    if vocab > _MAX_VOCAB:
        return None
    if u.dtype != torch.float32 or list(u.shape) != lead or u.device != dev:
        raise ValueError(f"sample: u must be float32 of shape {tuple(lead)} on {dev}, got {u.dtype} {tuple(u.shape)}")
    x = logits if len(lead) == 1 else logits.reshape(-1, vocab)
    rows = x.shape[0]
    stride = x.stride(0) if rows > 1 else vocab
    if stride < vocab or (vocab > 1 and x.stride(1) != 1):
        x = x.contiguous()
        stride = vocab
    t_p, t_s, t_ref = _per_row(temperature, rows, torch.float32, "temperature", dev)
    k_p, k_s, k_ref = _per_row(top_k, rows, torch.int32, "top_k", dev)
    p_p, p_s, p_ref = _per_row(top_p, rows, torch.float32, "top_p", dev)
    m_p, m_s, m_ref = _per_row(min_p, rows, torch.float32, "min_p", dev)
    if not u.is_contiguous():
        u = u.contiguous()
    token = torch.empty_like(u, dtype=torch.int32)
    logprob = torch.empty_like(u) if logprobs else None
    if rows:
        status = _lib.load().tsb_sample(x.data_ptr(), dt, rows, vocab, stride, u.data_ptr(), t_p, t_s, k_p,
                                        min(max(int(k_s), 0), vocab), p_p, p_s, m_p, m_s, token.data_ptr(), _ptr(logprob),
                                        _stream(x))
        if status:
            check(status, "tsb_sample")
            return None
    return (token, logprob) if logprobs else token


def _i32(t, shape, name: str, device):
    if t.device != device or t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)} on {device}, got {tuple(t.shape)} on {t.device}")
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def tree_accept(tokens, parents, samples):
    """The accepted path of each request's tree: from node 0, on to the lowest
    node c below the current one (parents[c] == cur, c > cur) whose drafted token
    is the one sampled at cur, until there is none.

    tokens, parents, samples (B, T) integers: the drafted tokens (-1 for a
    padding node), the parents as for tree_flash, and the token sampled after
    each node (negative: nothing follows). Returns int32 path (B, T), the
    accepted nodes and then -1; n_keep (B,), their number; next_token (B,), the
    token sampled after the last of them. None for T > 64."""
    if not tokens.is_cuda:
        raise ValueError("tsb operators take CUDA tensors (there is no CPU path)")
    dev = tokens.device
    if dev.index != _GET_DEVICE():
        with torch.cuda.device(dev):
            return tree_accept(tokens, parents, samples)
    shape = tokens.shape
    if len(shape) != 2:
        raise ValueError("tree_accept: tokens must be (B, T)")
    b, t = shape
    if t > 64:
        return None
    if t < 1:
        raise ValueError("tree_accept: a tree has at least its root")
    tok = _i32(tokens, shape, "tree_accept: tokens", dev)
    par = _i32(parents, shape, "tree_accept: parents", dev)
    smp = _i32(samples, shape, "tree_accept: samples", dev)
    path = torch.empty_like(tok)
    n_keep = tok.new_empty(b)
    nxt = tok.new_empty(b)
    if b:
        status = _lib.load().tsb_tree_accept(tok.data_ptr(), par.data_ptr(), smp.data_ptr(), b, t, path.data_ptr(),
                                             n_keep.data_ptr(), nxt.data_ptr(), _stream(tok))
        if status:
            check(status, "tsb_tree_accept")
    return path, n_keep, nxt


def _pointers(planes) -> list:
    return [t.data_ptr() for p in planes for t in p[1:] if t is not None]


class PathCommit:
    """The tree commit of a list of caches (every layer's; tree_verify.py:499-516)
    by lengths and paths on the device.

    plan = PathCommit(caches); new_lengths = plan(lengths, path, n_keep): for
    request b the last T rows of its lengths[b] are its tree's; rows
    lengths[b] - T + path[b, i], i < n_keep[b], move to lengths[b] - T + i in
    every cache, and the new length is lengths[b] - T + n_keep[b]. path (B, T)
    and n_keep (B,) are tree_accept's; a path must increase and ends where it
    does not. A request whose length is not in [T, capacity] is left as it is, in
    every cache: where capacities differ, the smallest counts.

    The plan holds the caches' tensors (not their `offset`): make it once per
    set of caches, and again if a cache gets new tensors. The caches of one
    request batch B may differ in format, heads and capacity; every tensor must
    be contiguous, of its format's type and shape."""

    def __init__(self, caches):
        self._caches = [(c, _kv_planes(c)) for c in caches]
        if not self._caches:
            raise ValueError("PathCommit: no caches")
        groups: dict = {}
        k0 = self._caches[0][1][1]
        pointers = _pointers(planes for _, planes in self._caches)
        self._pointers = frozenset(pointers)
        if len(self._pointers) < len(pointers):
            raise ValueError("PathCommit: a tensor appears twice: its rows would move twice")
        for _, planes in self._caches:
            _require_cuda(*planes[1:])
            # the same requests on the same device in every cache
            _check_planes("PathCommit", planes, k0.shape[0], None, 256, k0.device)
            groups.setdefault((planes[0], *planes[1].shape[1:3]), []).append(planes)
        self._device, self._batch = k0.device, k0.shape[0]
        caps = {cap for _, _, cap in groups}
        self._least = min(caps) if len(caps) > 1 else None
        self._launches = []
        vp = ctypes.c_void_p
        for (fmt, hkv, cap), members in groups.items():
            for i in range(0, len(members), _MAX_LAYERS_PER_LAUNCH):
                part = members[i:i + _MAX_LAYERS_PER_LAUNCH]
                arrays = [(vp * len(part))(*[_ptr(p[j]) for p in part]) if part[0][j] is not None else None
                          for j in range(1, 7)]
                self._launches.append((fmt, len(part), *arrays, self._batch, hkv, 256, cap))

    def is_of(self, caches) -> bool:
        """Whether these caches' tensors, as they are now, are the plan's."""
        return self._pointers.issuperset(now := _pointers(map(_kv_planes, caches))) and len(now) == len(self._pointers)

    def __call__(self, lengths, path, n_keep):
        dev, b = self._device, self._batch
        if dev.index != _GET_DEVICE():
            with torch.cuda.device(dev):
                return self(lengths, path, n_keep)
        if path.dim() != 2:
            raise ValueError("PathCommit: path must be (B, T)")
        t = path.shape[1]
        if not 1 <= t <= 64:
            raise ValueError(f"PathCommit: trees of 1 to 64 nodes, got {t}")
        p = _i32(path, (b, t), "PathCommit: path", dev)
        n = _i32(n_keep, (b,), "PathCommit: n_keep", dev)
        cur = _i32(lengths, (b,), "PathCommit: lengths", dev)
        new = torch.empty_like(cur)
        given = cur
        if self._least is not None:  # each launch knows its own caches' capacity
            fits = given <= self._least
            cur = torch.where(fits, given, 0)  # no tree ends there: left as it is
        commit, stream, out = _lib.load().tsb_kv_commit_paths, _stream(p), new.data_ptr()
        for args in self._launches:
            status = commit(*args, t, cur.data_ptr(), p.data_ptr(), n.data_ptr(), out, stream)
            out = None  # one launch writes the lengths
            if status and check(status, "tsb_kv_commit_paths") == TSB_EUNSUPPORTED:
                raise ValueError("PathCommit: unsupported caches")
        return new if cur is given else torch.where(fits, new, given)


def commit_paths(caches, lengths, path, n_keep):
    """PathCommit(caches)(lengths, path, n_keep), for a single commit."""
    return PathCommit(caches)(lengths, path, n_keep)
