"""The operators that end a verify step of many requests drawn from one prompt, as they are measured.

A step verifies a tree of drafted tokens for each request of a batch:

  attn    tree attention over a prompt that the whole batch shares and each request's own rows (`tsb.tree_flash_shared`)
  sample  one token for each tree node from its logits, with given random numbers (`tsb.sample`)
  accept  the walk down the tree along the sampled tokens (`tsb.tree_accept`)
  commit  the accepted nodes' rows kept in every layer's cache, lengths and paths on the device (`tsb.PathCommit`)

`run` computes them in plain torch operations, or, with `own`, through the library's own calls.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

D = 256  # head width of every cache format


def _tsb():
    if "tsb" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "mlx-tree-spec_b200"))
    import tsb

    return tsb


# ---------------------------------------------------------------- cases

def listed():
    return [
        # plain decoding of four samples of one prompt: one token each, a short prompt; the call's latency counts
        dict(name="attn-token-bf16", op="attn", fmt="bf16", batch=4, nodes=1, hq=24, hkv=4, prefix=1024, own=64, stats=False),
        # an ordinary verify step: eight requests, 16-node trees, an 8K prompt; the row statistics are asked for too
        dict(name="attn-tree-bf16", op="attn", fmt="bf16", batch=8, nodes=16, hq=24, hkv=4, prefix=8192, own=512, stats=True),
        # the largest: twelve requests with full 32-node trees over a 32K prompt
        dict(name="attn-wide-bf16", op="attn", fmt="bf16", batch=12, nodes=32, hq=24, hkv=4, prefix=32768, own=1024, stats=False),
        # a long prompt kept in 8 bits, groups of 64
        dict(name="attn-tree-mlx8", op="attn", fmt="mlx8", batch=5, nodes=32, hq=24, hkv=4, prefix=32768, own=256, stats=False),
        # odd sizes everywhere, int8 rows, seven query heads to a key head
        dict(name="attn-odd-int8", op="attn", fmt="int8", batch=7, nodes=13, hq=14, hkv=2, prefix=5003, own=333, stats=True),
        # one sequence, one token, the usual sampling settings
        dict(name="sample-one-bf16", op="sample", dtype="bfloat16", rows=1, vocab=131072, mode="usual", masked=False),
        # every node of eight 16-node trees, each row with settings of its own, a grammar's mask on the logits
        dict(name="sample-tree-bf16", op="sample", dtype="bfloat16", rows=128, vocab=131072, mode="mixed", masked=True),
        # temperature alone on flat 32-bit logits of an odd vocabulary: no filter leaves few candidates
        dict(name="sample-flat-f32", op="sample", dtype="float32", rows=48, vocab=100003, mode="flat", masked=False),
        # a few small trees, and many full ones
        dict(name="accept-small", op="accept", batch=4, nodes=16),
        dict(name="accept-full", op="accept", batch=64, nodes=64),
        # eight layers, four requests; and six layers of an 8-bit cache, 32 requests, an odd capacity
        dict(name="commit-bf16", op="commit", fmt="bf16", layers=8, batch=4, nodes=32, hkv=4, capacity=2048),
        dict(name="commit-mlx8", op="commit", fmt="mlx8", layers=6, batch=32, nodes=48, hkv=4, capacity=1001),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "sample", "sample", "sample", "accept", "commit"])
    if op == "attn":
        hkv = rng.choice([1, 2, 4, 8])
        c = dict(op="attn", fmt=rng.choice(["bf16", "bf16", "mlx8", "int8"]), batch=_log(rng, 1, 32), nodes=_log(rng, 1, 64),
                 hq=hkv * rng.randint(1, 8), hkv=hkv, prefix=_log(rng, 16, 32768), own=0, stats=rng.random() < 0.5)
        c["own"] = c["nodes"] + _log(rng, 1, 1500)
        top = 12 * 32 * 24 * (32768 + 528)
        while c["batch"] * c["nodes"] * c["hq"] * (c["prefix"] + c["own"]) > top or c["batch"] * c["hkv"] * c["own"] > 150000:
            c["batch"] = max(1, c["batch"] // 2)
            c["prefix"] = max(16, c["prefix"] * 2 // 3 + 1)
        return c
    if op == "sample":
        c = dict(op="sample", dtype=rng.choice(["bfloat16", "float16", "float32"]), rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 200000),
                 mode=rng.choice(["usual", "mixed", "flat"]), masked=rng.random() < 0.4)
        while c["rows"] * c["vocab"] > 128 * 131072:
            c["rows"] = max(1, c["rows"] // 2)
        return c
    if op == "accept":
        return dict(op="accept", batch=_log(rng, 1, 256), nodes=rng.randint(1, 64))
    return dict(op="commit", fmt=rng.choice(["bf16", "mlx8", "int8"]), layers=rng.randint(1, 8), batch=_log(rng, 1, 32),
                nodes=rng.randint(1, 64), hkv=rng.choice([1, 2, 4]), capacity=_log(rng, 128, 1024))


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _trees(batch, nodes, seed):
    """Parents int32 (batch, nodes): node 0 the root, every other below an earlier node, at most eight levels down."""
    r = np.random.default_rng(seed)
    parents = np.full((batch, nodes), -1, np.int32)
    depth = np.zeros((batch, nodes), np.int64)
    at = np.arange(batch)
    for i in range(1, nodes):
        p = r.integers(0, i, batch)
        p = np.where(depth[at, p] >= 8, 0, p)
        parents[:, i] = p
        depth[:, i] = depth[at, p] + 1
    return parents


def _planes(x, fmt):
    """A cache tensor of float rows (..., D) in a format: (data,), (codes, scales) or (words, scales, biases)."""
    if fmt == "bf16":
        return (x.bfloat16(),)
    if fmt == "int8":
        s = (x.abs().amax(-1) / 127).clamp_min(1e-6)
        return torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8), s
    g = x.reshape(*x.shape[:-1], D // 64, 64)
    b = g.amin(-1).bfloat16()
    s = ((g.amax(-1) - b.float()) / 255).bfloat16()
    q = torch.round((g - b.float()[..., None]) / s.float()[..., None]).clamp(0, 255).to(torch.uint8)
    return q.reshape(x.shape).view(torch.int32), s, b


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "attn":
        b, t, hq, hkv, n, o = (case[k] for k in ("batch", "nodes", "hq", "hkv", "prefix", "own"))
        parts = []
        for shape in ((1, hkv, n, D), (b, hkv, o, D)):
            parts += [_planes(torch.randn(shape, generator=g, device="cuda"), case["fmt"]) for _ in "kv"]
        st = dict(pk=parts[0], pv=parts[1], ok=parts[2], ov=parts[3],
                  q=torch.randn((b, hq, t, D), generator=g, device="cuda").bfloat16(),
                  lengths=torch.randint(t, o + 1, (b,), generator=g, device="cuda", dtype=torch.int32),
                  parents=torch.from_numpy(_trees(b, t, seed)).cuda())
    elif op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=g, device="cuda")
        if case["mode"] != "flat":  # a model's logits: a broad floor, and some tens of tokens that stand out
            x = 2 * x
            top = torch.randint(0, vocab, (rows, 48), generator=g, device="cuda")
            x.scatter_reduce_(1, top, 6 + 8 * torch.rand((rows, 48), generator=g, device="cuda"), "amax")
        if case["masked"]:
            x[torch.rand((rows, vocab), generator=g, device="cuda") < 0.3] = -math.inf
        st = dict(logits=x.to(getattr(torch, case["dtype"])), u=torch.rand(rows, generator=g, device="cuda"))
        if case["mode"] == "mixed":
            def pick(values, dtype):
                at = torch.randint(0, len(values), (rows,), generator=g, device="cuda")
                return torch.tensor(values, dtype=dtype, device="cuda")[at]

            st.update(temperature=pick([0.0, 0.6, 1.0, 1.0, 1.4], torch.float32), top_k=pick([0, 0, 1, 40, 1000], torch.int32),
                      top_p=pick([1.0, 0.95, 0.9, 0.5], torch.float32), min_p=pick([0.0, 0.0, 0.05], torch.float32))
        elif case["mode"] == "usual":
            st.update(temperature=0.8, top_k=50, top_p=0.95, min_p=0.0)
        else:
            st.update(temperature=1.3, top_k=0, top_p=1.0, min_p=0.0)
    elif op == "accept":
        b, t = case["batch"], case["nodes"]
        parents = _trees(b, t, seed)
        r = np.random.default_rng(seed + 1)
        tokens = r.integers(0, 131072, (b, t)).astype(np.int32)
        samples = r.integers(0, 131072, (b, t)).astype(np.int32)
        for i in range(1, t):  # most nodes' next tokens are among the drafted ones
            hit = r.random(b) < 0.5
            samples[np.arange(b)[hit], parents[hit, i]] = tokens[hit, i]
        st = dict(tokens=torch.from_numpy(tokens).cuda(), parents=torch.from_numpy(parents).cuda(), samples=torch.from_numpy(samples).cuda())
    else:
        b, t, hkv, cap = (case[k] for k in ("batch", "nodes", "hkv", "capacity"))
        layers = [[_planes(torch.randn((b, hkv, cap, D), generator=g, device="cuda"), case["fmt"]) for _ in "kv"] for _ in range(case["layers"])]
        r = np.random.default_rng(seed)
        path = np.full((b, t), -1, np.int32)
        keep = np.zeros(b, np.int32)
        for i, parents in enumerate(_trees(b, t, seed)):  # a root-to-node path of each tree
            node, up = int(r.integers(0, t)), []
            while node >= 0:
                up.append(node)
                node = int(parents[node])
            keep[i] = len(up)
            path[i, :len(up)] = up[::-1]
        st = dict(layers=layers, path=torch.from_numpy(path).cuda(), n_keep=torch.from_numpy(keep).cuda(),
                  lengths=torch.from_numpy(r.integers(t, cap + 1, b).astype(np.int32)).cuda())
        if own:  # the handle that a program keeps next to its caches
            st["plan"] = _tsb().PathCommit([_cache(k, v, case["fmt"], cap) for k, v in layers])
    st["case"] = dict(case)
    return st


# ---------------------------------------------------------------- the library's calls

def _cache(k, v, fmt, offset):
    tsb = _tsb()
    if fmt == "bf16":
        return tsb.KVCache(k[0], v[0], offset)
    if fmt == "int8":
        return tsb.Q8KVCache(k[0], v[0], k[1], v[1], offset)
    return tsb.MLXQ8KVCache(k[0], v[0], k[1], k[2], v[1], v[2], offset)


def _own(st):
    tsb, case = _tsb(), st["case"]
    op = case["op"]
    if op == "attn":
        prefix = _cache(st["pk"], st["pv"], case["fmt"], case["prefix"])
        cache = _cache(st["ok"], st["ov"], case["fmt"], case["own"])
        r = tsb.tree_flash_shared(st["q"], prefix, cache, D ** -0.5, parents=st["parents"], lengths=st["lengths"], stats=case["stats"])
        return [r[0], r[1][..., 0]] if case["stats"] else [r]
    if op == "sample":
        return list(tsb.sample(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], logprobs=True))
    if op == "accept":
        return list(tsb.tree_accept(st["tokens"], st["parents"], st["samples"]))
    return [st["plan"](st["lengths"], st["path"], st["n_keep"]), [[k, v] for k, v in st["layers"]]]


# ---------------------------------------------------------------- the plain form

def _values(planes):
    """Float values (..., D) of a cache tensor."""
    if len(planes) == 1:
        return planes[0].float()
    if len(planes) == 2:
        return planes[0].float() * planes[1][..., None]
    codes = planes[0].view(torch.uint8).float()
    codes = codes.reshape(*codes.shape[:-1], D // 64, 64)
    # the cache's value is the 16-bit one that dequantizing it gives
    return (codes * planes[1].float()[..., None] + planes[2].float()[..., None]).bfloat16().float().flatten(-2)


def _ancestors(parents):
    """bool (B, T, T): [b, i, j] where j is i or above it."""
    t = parents.shape[1]
    up = (parents[:, :, None] == torch.arange(t, device=parents.device)).double()
    return torch.linalg.matrix_power(up + torch.eye(t, dtype=torch.float64, device=parents.device), t) > 0


def _plain_attn(st):
    case = st["case"]
    b, t, hq, hkv, n, o = (case[k] for k in ("batch", "nodes", "hq", "hkv", "prefix", "own"))
    q = st["q"].float().reshape(b, hkv, hq // hkv * t, D) * D ** -0.5
    # the prefix's scores for the rows of the whole batch at once, key head by key head
    qs = q.transpose(0, 1).reshape(hkv, -1, D)
    sp = torch.matmul(qs, _values(st["pk"])[0].transpose(1, 2))
    so = torch.matmul(q, _values(st["ok"]).transpose(2, 3))
    # own rows: a node sees the rows before the last `nodes` of its request, and of those its ancestors'
    at = torch.arange(o, device="cuda")[None, :] - (st["lengths"].long()[:, None] - t)
    tree = torch.gather(_ancestors(st["parents"]), 2, at.clamp(0, t - 1)[:, None, :].expand(b, t, o))
    see = ((at < 0)[:, None, :] | tree) & (at < t)[:, None, :]
    so = so.reshape(b, hkv, -1, t, o).masked_fill(~see[:, None, None], -math.inf).reshape(b, hkv, -1, o)
    top = torch.maximum(sp.amax(-1).reshape(hkv, b, -1).transpose(0, 1), so.amax(-1))
    ps = torch.exp(sp - top.transpose(0, 1).reshape(hkv, -1, 1))
    po = torch.exp(so - top[..., None])
    total = ps.sum(-1).reshape(hkv, b, -1).transpose(0, 1) + po.sum(-1)
    out = torch.matmul(ps, _values(st["pv"])[0]).reshape(hkv, b, -1, D).transpose(0, 1)
    # rows past a request's length have no weight, whatever they hold
    out = (out + torch.matmul(po, _values(st["ov"]))) / total[..., None]
    out = out.reshape(b, hq, t, D).bfloat16()
    return [out, (top + torch.log(total)).reshape(b, hq, t)] if case["stats"] else [out]


def _column(v):
    return v[:, None].double() if isinstance(v, torch.Tensor) else v


def _plain_sample(st):
    x = st["logits"].float()
    rows, vocab = x.shape
    temperature, k, p, floor = (_column(st[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    full = torch.zeros((rows, 1), dtype=torch.float64, device=x.device)
    temperature, k, p, floor = full + temperature, full + k, full + p, full + floor
    k = torch.where(k > 0, k, vocab)
    k = torch.where(temperature > 0, k, 1)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    weight = torch.exp((x.double() - x[:, :1].double()) / torch.where(temperature > 0, temperature, 1))
    rank = torch.arange(vocab, device=x.device)
    kept = torch.where(rank < k, weight, 0)
    total = kept.sum(-1, keepdim=True)
    before = kept.cumsum(-1) - kept
    keep = (rank == 0) | (((before < p * total) | (p >= 1)) & (weight >= floor) & (rank < k))
    kept = torch.where(keep, weight, 0)
    up_to = kept.cumsum(-1)
    total = up_to[:, -1:]
    at = (up_to <= st["u"].double()[:, None] * total).sum(-1, keepdim=True)
    at = torch.minimum(at, (kept > 0).sum(-1, keepdim=True) - 1)
    return [torch.gather(order, 1, at)[:, 0].int(), torch.log(torch.gather(kept, 1, at) / total)[:, 0].float()]


def _plain_accept(st):
    tokens, parents, samples = st["tokens"], st["parents"].long(), st["samples"]
    b, t = tokens.shape
    hit = (parents >= 0) & (tokens == torch.gather(samples, 1, parents.clamp_min(0)))
    # of siblings with the same token the first counts
    same = (parents[:, :, None] == parents[:, None, :]) & hit[:, :, None] & hit[:, None, :]
    hit &= ~torch.tril(same, diagonal=-1).any(-1)
    hit[:, 0] = True
    kept = ~(_ancestors(parents) & ~hit[:, None, :]).any(-1)
    n = kept.sum(-1)
    nodes = torch.arange(t, device=tokens.device)
    path = torch.sort(torch.where(kept, nodes, t), dim=-1)[0]
    last = torch.where(kept, nodes, 0).amax(-1, keepdim=True)
    return [torch.where(path < t, path, -1).int(), n.int(), torch.gather(samples, 1, last)[:, 0]]


def _plain_commit(st):
    path, n, lengths = st["path"], st["n_keep"], st["lengths"]
    b, t = path.shape
    base = (lengths - t).long()[:, None]
    to = torch.arange(t, device=path.device)
    request = torch.arange(b, device=path.device)[:, None].expand(b, t)
    live = to < n[:, None]
    request, source, target = request[live], (base + path)[live], (base + to)[live]
    moved = [x for k, v in st["layers"] for x in (*k, *v)]
    rows = [x[request, :, source] for x in moved]
    [x.index_put_((request[:, None], torch.arange(x.shape[1], device=x.device), target[:, None]), r) for x, r in zip(moved, rows)]
    return [lengths - t + n, [[k, v] for k, v in st["layers"]]]


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "sample": _plain_sample, "accept": _plain_accept, "commit": _plain_commit}[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

_ROW_BYTES = {"bf16": 2 * D, "mlx8": D + D // 64 * 4, "int8": D + 4}


def work(case):
    op = case["op"]
    if op == "attn":
        b, t, hq, hkv, n = (case[k] for k in ("batch", "nodes", "hq", "hkv", "prefix"))
        mean = (t + case["own"]) / 2  # lengths lie evenly between the tree's and the capacity
        rows = b * hq * t
        return {"bytes": 2 * _ROW_BYTES[case["fmt"]] * hkv * (n + b * mean) + 2 * 2 * D * rows + (4 * rows if case["stats"] else 0),
                "flops": 4 * D * rows * (n + mean)}
    if op == "sample":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 28), "flops": 4 * case["rows"] * case["vocab"]}
    if op == "accept":
        return {"bytes": case["batch"] * (16 * case["nodes"] + 8), "flops": case["batch"] * case["nodes"]}
    kept = min(4, case["nodes"])  # nodes on an ordinary path
    return {"bytes": 2 * 2 * case["layers"] * case["batch"] * case["hkv"] * kept * _ROW_BYTES[case["fmt"]] + case["batch"] * (4 * kept + 12), "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_values(planes):
    if len(planes) == 3:
        codes = torch.stack([(planes[0] >> s) & 255 for s in (0, 8, 16, 24)], -1).flatten(-2).double()
        s, b = (x.double().repeat_interleave(64, -1) for x in planes[1:])
        return (codes * s + b).float().bfloat16().double()
    return planes[0].double() * (planes[1].double().unsqueeze(-1) if len(planes) == 2 else 1)


def _exact_attn(st):
    case = st["case"]
    b, t, hq, hkv, n = (case[k] for k in ("batch", "nodes", "hq", "hkv", "prefix"))
    g = hq // hkv
    parents, lengths = st["parents"].tolist(), st["lengths"].tolist()
    prefix_k, prefix_v = _exact_values(st["pk"])[0], _exact_values(st["pv"])[0]
    out = torch.empty((b, hq, t, D), dtype=torch.float64, device="cuda")
    lse = torch.empty((b, hq, t), dtype=torch.float64, device="cuda")
    for i in range(b):
        m = lengths[i]
        see = torch.zeros((t, n + m), dtype=torch.bool)
        see[:, :n + m - t] = True
        for node in range(t):
            up = node
            while up >= 0:
                see[node, n + m - t + up] = True
                up = parents[i][up]
        see = see.cuda()
        k = torch.cat([prefix_k, _exact_values([x[i, :, :m] for x in st["ok"]])], 1)
        v = torch.cat([prefix_v, _exact_values([x[i, :, :m] for x in st["ov"]])], 1)
        for h in range(hq):
            s = (st["q"][i, h].double() @ k[h // g].T / math.sqrt(D)).masked_fill(~see, -math.inf)
            lse[i, h] = torch.logsumexp(s, -1)
            out[i, h] = torch.softmax(s, -1) @ v[h // g]
    return [out, lse] if case["stats"] else [out]


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    rows, vocab = x.shape
    u = st["u"].double().cpu().numpy()
    column = [np.broadcast_to(v.double().cpu().numpy() if isinstance(v, torch.Tensor) else float(v), rows) for v in (st[n] for n in ("temperature", "top_k", "top_p", "min_p"))]
    tokens, logprobs = np.zeros(rows, np.int64), np.zeros(rows)
    for r in range(rows):
        temperature, k, p, floor = (float(v[r]) for v in column)
        order = np.argsort(-x[r], kind="stable")
        order = order[:1] if temperature <= 0 else order[:int(k)] if k > 0 else order
        w = np.exp((x[r][order] - x[r][order[0]]) / (temperature if temperature > 0 else 1.0))
        if p < 1:
            order = order[:int(np.searchsorted(np.cumsum(w), p * math.fsum(w), side="left")) + 1]
            w = w[:len(order)]
        order, w = order[w >= floor], w[w >= floor]
        mass = np.cumsum(w)
        at = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(order) - 1)
        tokens[r], logprobs[r] = order[at], math.log(w[at] / math.fsum(w))
    return [torch.from_numpy(tokens).int(), torch.from_numpy(logprobs)]


def _exact_accept(st):
    tokens, parents, samples = (st[n].tolist() for n in ("tokens", "parents", "samples"))
    paths, kept, then = [], [], []
    for token, parent, sample in zip(tokens, parents, samples):
        up = [0]
        while True:
            below = [i for i in range(up[-1] + 1, len(token)) if parent[i] == up[-1] and token[i] == sample[up[-1]]]
            if not below:
                break
            up.append(below[0])
        paths.append(up + [-1] * (len(token) - len(up)))
        kept.append(len(up))
        then.append(sample[up[-1]])
    return [torch.tensor(v, dtype=torch.int32) for v in (paths, kept, then)]


def _exact_commit(st):
    path, n, lengths = st["path"].tolist(), st["n_keep"].tolist(), st["lengths"].tolist()
    t = len(path[0])
    after = []
    for k, v in st["layers"]:
        pair = []
        for planes in (k, v):
            new = [x.clone() for x in planes]
            for i, (nodes, count, length) in enumerate(zip(path, n, lengths)):
                for x, y in zip(planes, new):
                    y[i, :, length - t:length - t + count] = x[i][:, [length - t + node for node in nodes[:count]]]
            pair.append([y.double() if y.is_floating_point() else y for y in new])
        after.append(pair)
    return [torch.tensor([length - t + count for length, count in zip(lengths, n)], dtype=torch.int32), after]


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "sample": _exact_sample, "accept": _exact_accept, "commit": _exact_commit}[case["op"]](st)
