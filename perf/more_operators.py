"""Cases of the operators of a speculative decoding step, for measuring them.

Four operators, each as ``run`` calls it when ``own`` is true, and in elementary torch operations
when it is false:

  sample   tokens drawn from logits with temperature, top-k, top-p and min-p and given random
           numbers (``ops.sample_tokens``)
  attend   attention of a tree of drafted tokens over a cache (``ops.tree_attention``)
  append   RoPE + append of a drafted tree to a cache (``ops.rope_kv_append_tree``)
  accept   the drafted branch that the samples agree with, and its rows moved together in the
           caches of every layer (``ops.tree_accept``)

A tree of T nodes has its root at node 0 and every parent before its children.  Of a sequence with
n keys in its cache, node t stands at row n + t and at rotary position n + depth(t); it sees the n
keys, its ancestors and itself.

Sampling: the weight of a logit is exp((logit - largest) / temperature).  Logits are ordered from
the largest down, equal ones by index.  The first top_k stay (0: all); of these the ones that have
at most top_p of these' sum before them; of these the ones that weigh at least min_p.  The token is
the lowest index at which the running sum of the weights that stay, in the order of the indices, is
above (random number) * (their sum); at temperature 0 the first of the order.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # -- sampling --------------------------------------------------------
        # one chat, vocabulary of the 7B shape, the generator's own top-k and top-p: latency
        {"name": "sample 1 x 32000 top-k 50 top-p 0.9", "op": "sample", "rows": 1, "vocab": 32000,
         "temperature": 0.8, "top_k": 50, "top_p": 0.9, "min_p": 0.0, "per_row": False,
         "type": "bf16"},
        # a small odd vocabulary, every row with its own settings, greedy rows among them
        {"name": "sample 37 x 1003 fp32", "op": "sample", "rows": 37, "vocab": 1003,
         "temperature": 0.9, "top_k": 40, "top_p": 0.8, "min_p": 0.05, "per_row": True,
         "type": "fp32"},
        # the nodes of 32 trees of 16, by nucleus, without top-k
        {"name": "sample 512 x 32000 top-p 0.95", "op": "sample", "rows": 512, "vocab": 32000,
         "temperature": 0.7, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "per_row": False,
         "type": "bf16"},
        # the largest: 256 sequences, the 128,256-row vocabulary, temperature alone
        {"name": "sample 256 x 128256", "op": "sample", "rows": 256, "vocab": 128256,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "per_row": False,
         "type": "bf16"},
        # -- attention of drafted trees --------------------------------------
        # one chat of about a thousand tokens, 7B heads, a tree of 16: latency
        {"name": "tree of 16 1 sequence 1000 keys", "op": "attend", "batch": 1, "nodes": 16,
         "heads": 32, "kv_heads": 32, "dim": 128, "cap": 1064, "shortest": 1000, "longest": 1000,
         "layout": "dense", "type": "bf16"},
        # a serving batch of mixed lengths, 32 heads on 8
        {"name": "tree of 24 32 sequences up to 4096 32:8", "op": "attend", "batch": 32,
         "nodes": 24, "heads": 32, "kv_heads": 8, "dim": 128, "cap": 4120, "shortest": 1,
         "longest": 4096, "layout": "dense", "type": "bf16"},
        # few long documents, 64 heads on 8 as in 70B, the widest tree: 512 rows a KV head
        {"name": "tree of 64 3 sequences of 60000 64:8", "op": "attend", "batch": 3, "nodes": 64,
         "heads": 64, "kv_heads": 8, "dim": 128, "cap": 60081, "shortest": 59000, "longest": 60017,
         "layout": "dense", "type": "bf16"},
        # packed cache of odd capacities, small heads, an empty sequence among them
        {"name": "tree of 13 ragged 17 sequences D=64", "op": "attend", "batch": 17, "nodes": 13,
         "heads": 12, "kv_heads": 6, "dim": 64, "cap": 1514, "shortest": 0, "longest": 1501,
         "layout": "ragged", "type": "fp16"},
        # -- append of drafted trees -----------------------------------------
        # one tree, 7B heads: latency
        {"name": "append a tree of 16", "op": "append", "batch": 1, "nodes": 16, "heads": 32,
         "kv_heads": 32, "dim": 128, "cap": 1064, "layout": "dense", "type": "bf16"},
        # 64 wide trees, 32 heads on 8, packed cache
        {"name": "append 64 trees of 64 ragged", "op": "append", "batch": 64, "nodes": 64,
         "heads": 32, "kv_heads": 8, "dim": 128, "cap": 400, "layout": "ragged", "type": "bf16"},
        # -- acceptance ------------------------------------------------------
        # one tree, the 32 layers of the 7B shape: latency
        {"name": "accept 1 of 16 32 layers", "op": "accept", "batch": 1, "nodes": 16, "layers": 32,
         "kv_heads": 32, "dim": 128, "cap": 300, "layout": "dense", "type": "bf16"},
        # 64 wide trees with long agreed branches, 32 layers of 8 KV heads, packed cache
        {"name": "accept 64 of 64 32 layers ragged", "op": "accept", "batch": 64, "nodes": 64,
         "layers": 32, "kv_heads": 8, "dim": 128, "cap": 200, "layout": "ragged", "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "attend", "attend", "append", "accept"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op == "sample":
        vocab = _log(rng, 2, 151936)
        return {"op": op, "rows": _log(rng, 1, max(1, min(1024, 16_000_000 // vocab))), "vocab": vocab,
                "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.6]),
                "top_k": rng.choice([0, 0, 1, 20, 50, 200, _log(rng, 2, 20000)]),
                "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                "min_p": rng.choice([0.0, 0.0, 0.02, 0.2]), "per_row": rng.random() < 0.4,
                "type": rng.choice(["bf16", "fp16", "fp32"])}
    kv_heads = rng.choice([1, 2, 5, 8, 16, 32])
    shared = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 128, 128])
    layout = rng.choice(["dense", "ragged"])
    nodes = _log(rng, 1, 64)
    if op == "attend":
        longest = _log(rng, 1, min(65536, 2 ** 20 // kv_heads))
        nodes = min(nodes, 2 ** 29 // (longest * kv_heads * shared))
        most = 2 ** 27 // (longest * kv_heads * shared * nodes)
        batch = _log(rng, 1, max(1, min(64, most, 2 ** 20 // (longest * kv_heads))))
        return {"op": op, "batch": batch, "nodes": nodes, "heads": kv_heads * shared,
                "kv_heads": kv_heads, "dim": dim, "cap": longest + nodes + rng.randint(0, 50),
                "shortest": rng.randint(0, longest), "longest": longest, "layout": layout,
                "type": kind}
    cap = nodes + rng.randint(0, 300)
    if op == "append":
        batch = _log(rng, 1, min(64, 196608 // (nodes * kv_heads * (shared + 2))))
        return {"op": op, "batch": batch, "nodes": nodes, "heads": kv_heads * shared,
                "kv_heads": kv_heads, "dim": dim, "cap": cap, "layout": layout, "type": kind}
    layers = rng.choice([1, 2, 16, 32])
    batch = _log(rng, 1, max(1, min(64, 2 ** 19 // (layers * kv_heads * cap))))
    return {"op": op, "batch": batch, "nodes": nodes, "layers": layers, "kv_heads": kv_heads,
            "dim": dim, "cap": cap, "layout": layout, "type": kind}


def _lengths(case):
    """Keys of each sequence before its tree.  For attention spread over [shortest, longest], both
    ends among them; else different places of the cache."""
    if case["op"] != "attend":
        return [(37 * b) % (case["cap"] - case["nodes"] + 1) for b in range(case["batch"])]
    r = random.Random(case["batch"] * 7919 + case["longest"])
    got = [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    got[0] = case["longest"]
    if case["batch"] > 1:
        got[-1] = case["shortest"]
    return got


def _capacities(case):
    """Rows that each sequence of a packed cache owns: odd numbers of them, at most `cap`."""
    r = random.Random(case["cap"])
    return [min(case["cap"], n + case["nodes"] + r.randint(0, 9)) for n in _lengths(case)]


def _parents(case, seed):
    """Random trees, [batch][nodes]: a node hangs on one of the few before it, so that branches are
    deep and siblings there.  Node 0, the root, has none."""
    r = random.Random(seed * 31 + case["nodes"])
    return [[-1] + [r.randint(max(0, t - 4), t - 1) for t in range(1, case["nodes"])]
            for _ in range(case["batch"])]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["type"] == "fp32" else 2) + 12 * case["rows"], "flops": 4 * n}
    kv, dim, nodes, batch = case["kv_heads"], case["dim"], case["nodes"], case["batch"]
    if case["op"] == "attend":
        keys = sum(_lengths(case)) + batch * nodes
        return {"bytes": 4 * keys * kv * dim + 4 * batch * nodes * case["heads"] * dim,
                "flops": 4 * keys * case["heads"] * nodes * dim}
    if case["op"] == "append":
        tokens, heads = batch * nodes, case["heads"]
        return {"bytes": 4 * tokens * (heads + 2 * kv) * dim + 4 * tokens * dim + 4 * tokens,
                "flops": 3 * tokens * (heads + kv) * dim}
    # about a fifth of the nodes are on the branch that is kept
    rows = batch * max(1, nodes // 5) * kv * case["layers"] * 2
    return {"bytes": 2 * 2 * rows * dim + 40 * batch * nodes, "flops": 3 * batch * nodes}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _settings(case, gen):
    """temperature, top_k, top_p, min_p: one for all rows, or one for each, around the case's."""
    rows = case["rows"]
    t, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
    if not case["per_row"]:
        return t, k, p, m

    def some(share):
        return torch.rand(rows, device=DEV, generator=gen) < share

    spread = torch.rand(rows, device=DEV, generator=gen)
    ts = torch.where(some(0.2), torch.zeros_like(spread), t * (0.5 + spread))
    ks = torch.where(some(0.3), 0, torch.randint(1, max(2 * k, 100), (rows,), device=DEV, generator=gen))
    ps = torch.where(some(0.3), torch.ones_like(spread), p * (0.6 + 0.4 * spread))
    return ts, ks.to(torch.int32), ps, m * spread


def _logits(case, gen, kind):
    """What a model's last layer gives: a wide bell, a few dozen tokens well above it; in every
    fourth row most of the vocabulary ruled out, as by a grammar."""
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, device=DEV, generator=gen)
    x *= 1 + 1.5 * torch.rand(rows, 1, device=DEV, generator=gen)
    lift = torch.rand(rows, vocab, device=DEV, generator=gen) < 48 / vocab
    x += lift * (6 + 3 * torch.randn(rows, vocab, device=DEV, generator=gen))
    out = torch.rand(rows, vocab, device=DEV, generator=gen) < 0.9
    out[torch.arange(rows, device=DEV) % 4 != 3] = False
    out[:, :1] = False
    return x.masked_fill_(out, -math.inf).to(kind)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] == "sample":
        st = {"logits": _logits(case, gen, kind), "settings": _settings(case, gen),
              "u": torch.rand(case["rows"], device=DEV, generator=gen)}
        return {"case": case, **st}
    kv, dim, batch, nodes = case["kv_heads"], case["dim"], case["batch"], case["nodes"]
    lens = _lengths(case)
    st = {"base": None, "caps": None, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV)}
    if case["layout"] == "ragged":
        caps = _capacities(case)
        bases = [sum(caps[:b]) for b in range(batch)]
        st["base"] = torch.tensor(bases, dtype=torch.int64, device=DEV)
        st["caps"] = torch.tensor(caps, dtype=torch.int32, device=DEV)
        shape = (kv, sum(caps), dim)
    else:
        shape = (batch, kv, case["cap"], dim)
    if case["op"] == "accept":
        shape = (case["layers"], *shape)
    # keys carry the rotation and spread wider than values
    st["k"] = torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16).to(kind)
    st["v"] = (torch.randn(shape, device=DEV, generator=gen, dtype=torch.bfloat16) * 0.8).to(kind)
    parents = _parents(case, seed)
    depth = [[0] * nodes for _ in range(batch)]
    seen = [[1] * nodes for _ in range(batch)]
    for b in range(batch):
        for t in range(1, nodes):
            depth[b][t] = depth[b][parents[b][t]] + 1
            seen[b][t] = seen[b][parents[b][t]] | (1 << t)
    st["depths"] = torch.tensor(depth, dtype=torch.int32, device=DEV)
    signed = [[m - (1 << 64) if m >> 63 else m for m in row] for row in seen]
    st["masks"] = torch.tensor(signed, dtype=torch.int64, device=DEV)
    st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
    if case["op"] == "attend":
        st["q"] = torch.randn(batch, case["heads"], nodes, dim, device=DEV, generator=gen).to(kind)
        if own:
            from llama_pure_compute_b200 import ops
            st["workspace"] = ops.tree_attention_workspace(st["q"], st["k"])
    elif case["op"] == "append":
        width = (case["heads"] + 2 * kv) * dim
        st["qkv"] = torch.randn(batch, nodes, width, device=DEV, generator=gen).to(kind)
        # the model's rotation tables, [positions, dim] in the data's type
        turn = 10000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
        angle = torch.arange(case["cap"], device=DEV, dtype=torch.float64)[:, None] * turn
        st["cos"] = angle.cos().repeat(1, 2).to(kind)
        st["sin"] = angle.sin().repeat(1, 2).to(kind)
    else:
        # few different tokens, so that siblings may repeat one; samples agree with a child of most
        # nodes
        st["drafted"] = torch.randint(0, 50, (batch, nodes), device=DEV, generator=gen)
        child = torch.zeros(batch, nodes, dtype=torch.int64, device=DEV)
        child.scatter_reduce_(1, st["parents"].clamp(min=0).long(),
                              torch.arange(nodes, device=DEV).expand(batch, -1), "amax")
        agreed = torch.rand(batch, nodes, device=DEV, generator=gen) < 0.95
        st["sampled"] = torch.where(agreed, st["drafted"].gather(1, child),
                                    torch.randint(50, 32000, (batch, nodes), device=DEV,
                                                  generator=gen))
        if own:
            from llama_pure_compute_b200 import ops
            st["kv"] = ops.LayerCaches(st["k"].unbind(0), st["v"].unbind(0), st["base"], st["caps"])
    return {"case": case, **st}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(st):
    from llama_pure_compute_b200 import ops
    case = st["case"]
    if case["op"] == "sample":
        t, k, p, m = st["settings"]
        return ops.sample_tokens(st["logits"], st["u"], temperature=t, top_k=k, top_p=p, min_p=m)
    if case["op"] == "attend":
        return ops.tree_attention(st["q"], st["k"], st["v"], st["lens"], st["masks"],
                                  seq_base=st["base"], seq_cap=st["caps"],
                                  workspace=st["workspace"])
    if case["op"] == "append":
        q = ops.rope_kv_append_tree(st["qkv"], st["lens"], st["depths"], st["cos"], st["sin"],
                                    st["k"], st["v"], case["heads"], case["kv_heads"],
                                    seq_base=st["base"], seq_cap=st["caps"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    accepted, tokens, path = ops.tree_accept(st["drafted"], st["parents"], st["sampled"], st["lens"],
                                             st["kv"])
    return {"accepted": accepted, "tokens": tokens, "path": path, "k": st["k"], "v": st["v"]}


def _plain(st):
    return {"sample": _plain_sample, "attend": _plain_attend, "append": _plain_append,
            "accept": _plain_accept}[st["case"]["op"]](st, st["case"])


def _plain_sample(st, case):
    """In 64 bits: a running sum of a hundred thousand weights is compared with a random number."""
    rows, vocab = st["logits"].shape
    t, k, p, m = (torch.as_tensor(x, device=DEV).double().expand(rows)[:, None]
                  for x in st["settings"])
    # settings are 32-bit numbers
    t, p, m = t.float().double(), p.float().double(), m.float().double()
    value, at = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    top = value[:, :1]
    x = (value - torch.where(top == -math.inf, torch.zeros_like(top), top)) / torch.where(t == 0, t + 1, t)
    w = torch.exp(x)
    rank = torch.arange(vocab, device=DEV)
    w = torch.where((k == 0) | (rank < k), w, torch.zeros_like(w))
    run_sum = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(top), run_sum[:, :-1]], 1)
    stay = ((p == 1) | (before <= p * run_sum[:, -1:])) & (w >= m)
    w = torch.zeros_like(w).scatter_(1, at, torch.where(stay, w, torch.zeros_like(w)))
    run_sum = torch.cumsum(w, 1)
    token = (run_sum <= st["u"].double()[:, None] * run_sum[:, -1:]).sum(1)
    token = torch.where(t[:, 0] == 0, at[:, 0], token)
    return torch.where(top[:, 0] == -math.inf, torch.full_like(token, -1), token)


def _plain_attend(st, case):
    batch, kv, dim, nodes = case["batch"], case["kv_heads"], case["dim"], case["nodes"]
    longest = case["longest"] + nodes
    if st["base"] is not None:
        # rows past a sequence's end belong to others: they are masked, and kept inside the tensor
        at = st["base"][:, None] + torch.arange(longest, device=DEV)
        at = at.clamp(max=st["k"].shape[1] - 1)
        k, v = (t[:, at].transpose(0, 1) for t in (st["k"], st["v"]))
    else:
        k, v = (t[:, :, :longest] for t in (st["k"], st["v"]))
    q = st["q"].float().view(batch, kv, -1, dim)
    score = torch.matmul(q, k.float().transpose(2, 3)) * dim ** -0.5
    at = torch.arange(longest, device=DEV) - st["lens"][:, None]  # [B, keys], nodes from 0 up
    bit = (st["masks"][:, :, None] >> at.clamp(0, 63)[:, None]) & 1
    seen = (at < 0)[:, None] | ((at < nodes)[:, None] & (bit == 1))  # [B, T, keys]
    seen = seen[:, None, None].expand(-1, kv, case["heads"] // kv, -1, -1).reshape(score.shape)
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    out = torch.matmul(p, v.float()) / p.sum(-1, keepdim=True)
    return out.view(batch, case["heads"], nodes, dim).to(st["q"].dtype)


def _plain_append(st, case):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    batch, nodes = case["batch"], case["nodes"]
    x = st["qkv"].float().view(batch, nodes, heads + 2 * kv, dim)
    turned, v = x[:, :, :heads + kv], x[:, :, heads + kv:]
    pos = st["lens"][:, None].long() + st["depths"].long()
    cos, sin = st["cos"][pos].float()[:, :, None], st["sin"][pos].float()[:, :, None]
    low, high = turned[..., :dim // 2], turned[..., dim // 2:]
    turned = (turned * cos + torch.cat([-high, low], -1) * sin).to(st["qkv"].dtype)
    row = st["lens"][:, None].long() + torch.arange(nodes, device=DEV)
    for cache, new in ((st["k"], turned[:, :, heads:]), (st["v"], v.to(st["qkv"].dtype))):
        if st["base"] is not None:
            cache[:, st["base"][:, None] + row] = new.permute(2, 0, 1, 3)
        else:
            cache[torch.arange(batch, device=DEV)[:, None], :, row] = new
    return {"q": turned[:, :, :heads].transpose(1, 2).contiguous(), "k": st["k"], "v": st["v"]}


def _plain_accept(st, case):
    batch, nodes = case["batch"], case["nodes"]
    # agreed[b, t, c]: c is a child of t and holds t's sample; `after` is the lowest such child
    agreed = (st["parents"][:, None, :] == torch.arange(nodes, device=DEV)[:, None])
    agreed &= st["drafted"][:, None, :] == st["sampled"][:, :, None]
    index = torch.arange(nodes, device=DEV)
    after = torch.where(agreed, index, torch.full_like(index, nodes)).amin(-1)  # nodes: none
    after = torch.cat([after, torch.full_like(after[:, :1], nodes)], 1)
    path = torch.full((batch, nodes), nodes, device=DEV)
    here = torch.zeros(batch, dtype=torch.int64, device=DEV)
    for i in range(nodes):
        path[:, i] = here
        here = after.gather(1, here[:, None])[:, 0]
    on = path < nodes
    tokens = torch.where(on, st["sampled"].gather(1, path.clamp(max=nodes - 1)), -1)
    # rows off the path are written with themselves
    source = torch.where(on, path, index) + st["lens"][:, None].long()
    target = index + st["lens"][:, None].long()
    for cache in (st["k"], st["v"]):
        if st["base"] is not None:
            cache[:, :, st["base"][:, None] + target] = cache[:, :, st["base"][:, None] + source]
        else:
            b = torch.arange(batch, device=DEV)[:, None]
            cache[:, b, :, target] = cache[:, b, :, source]
    return {"accepted": on.sum(1).to(torch.int32), "tokens": tokens,
            "path": torch.where(on, path, -1).to(torch.int32), "k": st["k"], "v": st["v"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"sample": _exact_sample, "attend": _exact_attend, "append": _exact_append,
            "accept": _exact_accept}[case["op"]](st, case)


def _exact_sample(st, case):
    """Row by row, by successive shortening of the ordered list."""
    rows = case["rows"]
    ts, ks, ps, ms = (torch.as_tensor(x).expand(rows).tolist() for x in st["settings"])
    ts, ps, ms = (torch.tensor(x, dtype=torch.float32).tolist() for x in (ts, ps, ms))
    us, got = st["u"].tolist(), []
    for r in range(rows):
        x = st["logits"][r].double()
        order = torch.argsort(-x, stable=True)
        best = float(x[order[0]])
        if best == -math.inf or ts[r] == 0:
            got.append(-1 if best == -math.inf else int(order[0]))
            continue
        order = order[:int(ks[r])] if ks[r] else order
        w = ((x[order] - best) / ts[r]).exp()
        if ps[r] < 1:
            upto = w.cumsum(0)
            n = int(torch.searchsorted(upto, (upto[-1] * ps[r])[None], right=True))
            order, w = order[:n + 1], w[:n + 1]
        order, w = order[w >= ms[r]], w[w >= ms[r]]
        order, by = order.sort()
        upto = w[by].cumsum(0)
        n = int(torch.searchsorted(upto, (upto[-1] * us[r])[None], right=True))
        got.append(int(order[min(n, order.numel() - 1)]))
    return torch.tensor(got, device=DEV)


def _exact_attend(st, case):
    kv, dim, nodes = case["kv_heads"], case["dim"], case["nodes"]
    group = case["heads"] // kv
    out = torch.zeros(case["batch"], case["heads"], nodes, dim, dtype=torch.float64, device=DEV)
    parents = st["parents"].tolist()
    for b, n in enumerate(st["lens"].tolist()):
        sees = [[False] * nodes for _ in range(nodes)]
        for t in range(nodes):
            a = t
            while a >= 0:
                sees[t][a] = True
                a = parents[b][a]
        hidden = torch.zeros(nodes, n + nodes, dtype=torch.float64, device=DEV)
        hidden[:, n:][~torch.tensor(sees, device=DEV)] = -math.inf
        for h in range(kv):
            if case["layout"] == "ragged":
                at = int(st["base"][b])
                k, v = (t[h, at:at + n + nodes].double() for t in (st["k"], st["v"]))
            else:
                k, v = (t[b, h, :n + nodes].double() for t in (st["k"], st["v"]))
            for g in range(h * group, (h + 1) * group):
                s = st["q"][b, g].double() @ k.mT / math.sqrt(dim) + hidden
                out[b, g] = torch.softmax(s, -1) @ v
    return out


def _exact_append(st, case):
    heads, kv, half = case["heads"], case["kv_heads"], case["dim"] // 2
    x = st["qkv"].double().view(case["batch"], case["nodes"], -1, case["dim"]).transpose(1, 2)
    pos = (st["lens"][:, None] + st["depths"]).long()
    a, b = x[:, :heads + kv, :, :half], x[:, :heads + kv, :, half:]
    cos, sin = (st[n][pos].double()[:, None] for n in ("cos", "sin"))
    turned = torch.empty_like(x[:, :heads + kv])
    turned[..., :half] = a * cos[..., :half] - b * sin[..., :half]
    turned[..., half:] = b * cos[..., half:] + a * sin[..., half:]
    k, v = st["k"].double(), st["v"].double()
    for i, n in enumerate(st["lens"].tolist()):
        if case["layout"] == "ragged":
            at = int(st["base"][i]) + n
            k[:, at:at + case["nodes"]] = turned[i, heads:]
            v[:, at:at + case["nodes"]] = x[i, heads + kv:]
        else:
            k[i, :, n:n + case["nodes"]] = turned[i, heads:]
            v[i, :, n:n + case["nodes"]] = x[i, heads + kv:]
    return {"q": turned[:, :heads], "k": k, "v": v}


def _exact_accept(st, case):
    """Whole numbers; rows of the caches are moved, not computed, and a later pass moves them on."""
    nodes, accepted, tokens, paths = case["nodes"], [], [], []
    for parent, held, said in zip(st["parents"].tolist(), st["drafted"].tolist(),
                                  st["sampled"].tolist()):
        path = [0]
        while True:
            nxt = [c for c in range(nodes) if parent[c] == path[-1] and held[c] == said[path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        accepted.append(len(path))
        tokens.append([said[t] for t in path] + [-1] * (nodes - len(path)))
        paths.append(path + [-1] * (nodes - len(path)))
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(tokens),
            "path": torch.tensor(paths, dtype=torch.int32), "k": None, "v": None}
