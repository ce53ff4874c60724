"""Append and acceptance of drafted trees against their definitions."""
import random

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from oracle.tree_ref import accept_ref, tree_masks_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def trees(batch, nodes, seed=0, back=4):
    """parents [batch][nodes], random, deep and branching."""
    r = random.Random(seed)
    return [[-1] + [r.randint(max(0, t - back), t - 1) for t in range(1, nodes)] for _ in range(batch)]


def layout(ragged, lens, nodes, spare=3):
    """(shape of a cache without its dims, seq_base, seq_cap, row of (sequence, place))."""
    if not ragged:
        cap = max(lens) + nodes + spare
        return (len(lens), None, cap), None, None
    caps = [n + nodes + (i % 2) for i, n in enumerate(lens)]
    bases = [sum(caps[:i]) for i in range(len(caps))]
    return ((None, sum(caps)), torch.tensor(bases, device=DEV),
            torch.tensor(caps, dtype=torch.int32, device=DEV))


def new_cache(lead, kv, dim, kind, gen):
    shape = [kv if n is None else n for n in lead] + [dim]
    return torch.randn(shape, device=DEV, generator=gen).to(kind)


def rows_of(cache, base, b, lo, hi):
    """[kv heads, hi - lo, dim] of sequence b, a view."""
    if base is None:
        return cache[b, :, lo:hi]
    return cache[:, int(base[b]) + lo:int(base[b]) + hi]


# -- append ------------------------------------------------------------------
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("table", ["same", "fp32"])
@pytest.mark.parametrize("nodes,heads,kv,dim", [(1, 4, 4, 128), (13, 6, 2, 64), (64, 8, 1, 32), (5, 3, 3, 16),
                                                (7, 40, 8, 128)])
def test_append(nodes, heads, kv, dim, table, kind, ragged):
    gen = torch.Generator(device=DEV).manual_seed(nodes)
    kind = TYPES[kind]
    lens = [0, 17, 3]
    lead, base, cap = layout(ragged, lens, nodes)
    kc, vc = (new_cache(lead, kv, dim, kind, gen) for _ in range(2))
    qkv = torch.randn(3, nodes, (heads + 2 * kv) * dim, device=DEV, generator=gen).to(kind)
    depths = torch.tensor([tree_masks_ref(p)[1] for p in trees(3, nodes, nodes)], dtype=torch.int32,
                          device=DEV)
    angle = torch.rand(200, dim, device=DEV, generator=gen) * 6
    tk = torch.float32 if table == "fp32" else kind
    cos, sin = angle.cos().to(tk), angle.sin().to(tk)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want_k, want_v = kc.clone(), vc.clone()
    q = ops.rope_kv_append_tree(qkv, seq, depths, cos, sin, kc, vc, heads, kv, base, cap)
    # every product and the sum rounded to fp32, once more to the type: as lpc_rope_kv_append
    x = qkv.float().view(3, nodes, heads + 2 * kv, dim)
    pos = seq[:, None].long() + depths.long()
    c, s = cos[pos].float()[:, :, None], sin[pos].float()[:, :, None]
    lo, hi = x[:, :, :heads + kv, :dim // 2], x[:, :, :heads + kv, dim // 2:]
    turned = torch.cat([lo * c[..., :dim // 2] - hi * s[..., :dim // 2],
                        hi * c[..., dim // 2:] + lo * s[..., dim // 2:]], -1).to(kind)
    assert torch.equal(q, turned[:, :, :heads].transpose(1, 2))
    for b, n in enumerate(lens):
        rows_of(want_k, base, b, n, n + nodes).copy_(turned[b, :, heads:].transpose(0, 1))
        rows_of(want_v, base, b, n, n + nodes).copy_(x[b, :, heads + kv:].to(kind).transpose(0, 1))
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)  # the other rows as they were
    assert _lib.device_status() == 0


def test_append_of_a_chain_is_the_append_of_a_prompt():
    gen = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(2, 9, (8 + 4) * 64, device=DEV, generator=gen).bfloat16()
    cos, sin = torch.randn(2, 50, 64, device=DEV, generator=gen).bfloat16()
    caches = [torch.zeros(2, 2, 40, 64, device=DEV).bfloat16() for _ in range(4)]
    lens = torch.tensor([5, 11], dtype=torch.int32, device=DEV)
    pos = lens[:, None].long() + torch.arange(9, device=DEV)
    a = ops.rope_kv_append(qkv, pos, cos, sin, caches[0], caches[1], 8, 2)
    b = ops.rope_kv_append_tree(qkv, lens, torch.arange(9, dtype=torch.int32, device=DEV), cos, sin,
                                caches[2], caches[3], 8, 2)
    assert torch.equal(a, b) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("ragged", [False, True])
def test_append_skips_and_flags(ragged):
    gen = torch.Generator(device=DEV).manual_seed(2)
    lead, base, cap = layout(ragged, [4, 4, 4], 4, spare=0)
    kc, vc = (new_cache(lead, 2, 32, torch.float16, gen) for _ in range(2))
    qkv = torch.randn(3, 4, 6 * 32, device=DEV, generator=gen).half()
    cos, sin = torch.randn(2, 8, 32, device=DEV, generator=gen).half()
    k0, v0 = kc.clone(), vc.clone()
    depths = torch.tensor([0, -1, 1, -5], dtype=torch.int32, device=DEV)
    lens = torch.tensor([4, 4, 4], dtype=torch.int32, device=DEV)
    q = ops.rope_kv_append_tree(qkv, lens, depths, cos, sin, kc, vc, 2, 2, base, cap)
    assert _lib.device_status() == 0
    for b in range(3):
        for t in (1, 3):
            assert (q[b, :, t] == 0).all()
            for now, was in ((kc, k0), (vc, v0)):
                assert torch.equal(rows_of(now, base, b, 4 + t, 5 + t), rows_of(was, base, b, 4 + t, 5 + t))
        assert (q[b, :, 0] != 0).any()
    # rows past the sequence's, before it, and positions past the tables
    for lens_bad, d in (([4, 30, 4], 0), ([4, -1, 4], 0), ([4, 2 ** 31 - 1, 4], 0), ([4, 4, 4], 7)):
        kc.copy_(k0)
        vc.copy_(v0)
        d = torch.tensor([d] * 4, dtype=torch.int32, device=DEV)
        q = ops.rope_kv_append_tree(qkv, torch.tensor(lens_bad, dtype=torch.int32, device=DEV), d, cos,
                                    sin, kc, vc, 2, 2, base, cap)
        assert (q[1] == 0).all() and torch.equal(rows_of(kc, base, 1, 0, 8), rows_of(k0, base, 1, 0, 8))
        assert _lib.device_status() == 2


# -- acceptance --------------------------------------------------------------
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("nodes,layers,kv,dim,kind", [(1, 1, 2, 64, torch.bfloat16), (2, 2, 1, 32, torch.float16),
                                                      (33, 3, 5, 128, torch.bfloat16), (64, 130, 1, 16, torch.float16),
                                                      (64, 2, 2, 8, torch.float32), (40, 1, 3, 40, torch.bfloat16)])
def test_accept(nodes, layers, kv, dim, kind, ragged):
    gen = torch.Generator(device=DEV).manual_seed(nodes)
    r = random.Random(nodes + ragged)
    lens = [0, 9, 30, 2, 5]
    B = len(lens)
    lead, base, cap = layout(ragged, lens, nodes)
    ks, vs = ([new_cache(lead, kv, dim, kind, gen) for _ in range(layers)] for _ in range(2))
    parents = trees(B, nodes, nodes, back=3)
    drafted = [[r.randint(0, 5) + 2 ** 40 * r.randint(0, 1) for _ in range(nodes)] for _ in range(B)]
    sampled = [[0] * nodes for _ in range(B)]
    for b in range(B):  # most nodes go on to a child of theirs, b = 0 never
        for t in range(nodes):
            kids = [c for c in range(nodes) if parents[b][c] == t]
            go = kids and b and r.random() < 0.97
            sampled[b][t] = drafted[b][r.choice(kids)] if go else 99
    as64 = lambda x: torch.tensor(x, dtype=torch.int64, device=DEV)  # noqa: E731
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want_k, want_v = [t.clone() for t in ks], [t.clone() for t in vs]
    acc, tok, path = ops.tree_accept(as64(drafted), torch.tensor(parents, dtype=torch.int32, device=DEV),
                                     as64(sampled), seq, ops.LayerCaches(ks, vs, base, cap))
    for b, n in enumerate(lens):
        p, t = accept_ref(drafted[b], parents[b], sampled[b])
        assert acc[b] == len(p) and (b or len(p) == 1)
        assert path[b].tolist() == p + [-1] * (nodes - len(p))
        assert tok[b].tolist() == t + [-1] * (nodes - len(p))
        for cache in want_k + want_v:
            rows = rows_of(cache, base, b, n, n + nodes)
            rows[:, :len(p)] = rows[:, p]
    for got, want in zip(ks + vs, want_k + want_v):
        assert torch.equal(got, want)
    assert seq.tolist() == lens and _lib.device_status() == 0


def test_accept_without_caches_and_with_one_tree():
    parents = torch.tensor([-1, 0, 0, 1, 1, 2], dtype=torch.int32, device=DEV)
    drafted = torch.tensor([[9, 5, 7, 1, 1, 2], [9, 5, 5, 1, 1, 2]], device=DEV)
    sampled = torch.tensor([[7, 0, 2, 0, 0, 4], [5, 1, 0, 8, 9, 0]], device=DEV)
    acc, tok, path = ops.tree_accept(drafted, parents, sampled)
    assert acc.tolist() == [3, 3]
    assert tok.tolist() == [[7, 2, 4, -1, -1, -1], [5, 1, 8, -1, -1, -1]]  # equal children: the lowest
    assert path.tolist() == [[0, 2, 5, -1, -1, -1], [0, 1, 3, -1, -1, -1]]
    assert _lib.device_status() == 0


def test_accept_of_trees_and_rows_that_are_not_sound():
    drafted = torch.zeros(1, 4, dtype=torch.int64, device=DEV)
    for parents in ([-1, 1, 1, 1], [3, 0, 2, 2], [-1, 2, 1, 2 ** 31 - 1], [0, 0, 0, 3]):
        acc, tok, path = ops.tree_accept(drafted, torch.tensor([parents], dtype=torch.int32, device=DEV), drafted)
        assert path[0].tolist()[:acc[0]] == accept_ref([0] * 4, parents, [0] * 4)[0]
        assert _lib.device_status() == 2
    # a branch past the sequence's rows stays where it is; the others move
    k, v = (torch.randn(2, 1, 10, 8, device=DEV) for _ in range(2))
    k0 = k.clone()
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32, device=DEV)
    drafted = torch.tensor([[0, 1, 2, 3]] * 2, device=DEV)
    sampled = torch.tensor([[2, 0, 3, 0]] * 2, device=DEV)
    for lens in ([7, 3], [-1, 3], [2 ** 31 - 1, 3]):
        k.copy_(k0)
        acc, _, _ = ops.tree_accept(drafted, parents, sampled, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                    ops.LayerCaches([k], [v]))
        assert acc.tolist() == [3, 3] and torch.equal(k[0], k0[0])
        assert torch.equal(k[1, :, 4:6], k0[1, :, 5:7])
        assert _lib.device_status() == 2


def test_refusals():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    kc = torch.zeros(2, 2, 16, 32, device=DEV).half()
    tab = torch.zeros(16, 32, device=DEV).half()
    qkv = torch.zeros(2, 3, 6 * 32, device=DEV).half()

    def append(qkv=qkv, lens=i32(2), depths=i32(2, 3), cos=tab, sin=tab, k=kc, v=kc, h=2, kv=2, **kw):
        return ops.rope_kv_append_tree(qkv, lens, depths, cos, sin, k, v, h, kv, **kw)
    append()
    for bad in (dict(qkv=qkv.cpu()), dict(qkv=qkv[0]), dict(qkv=qkv[..., :-1]), dict(lens=i32(1)),
                dict(depths=i32(3, 2)), dict(depths=i32(2, 3).cpu()), dict(cos=tab[:, :16]), dict(sin=tab[:8]),
                dict(k=kc[:, :, ::2], v=kc[:, :, ::2]), dict(v=kc[:, :, :8]), dict(k=kc[:1], v=kc[:1]),
                dict(k=kc[0], v=kc[0]), dict(seq_base=torch.zeros(2, dtype=torch.int64, device=DEV)),
                dict(h=3), dict(kv=4), dict(q_out=qkv.new_empty(2, 2, 3, 16)), dict(q_out=qkv.view(-1)[:384].view(2, 2, 3, 32))):
        with pytest.raises(ValueError):
            append(**bad)
    for bad in (dict(lens=i32(2).long()), dict(depths=i32(2, 3).long()), dict(qkv=qkv.bfloat16()),
                dict(cos=tab.bfloat16(), sin=tab.bfloat16()),
                dict(qkv=qkv.float(), k=kc.float(), v=kc.float())):
        with pytest.raises(TypeError):
            append(**bad)
    tok = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    kv = ops.LayerCaches([kc], [kc.clone()])
    ops.tree_accept(tok, i32(2, 3), tok, i32(2), kv)
    for bad in ((tok.cpu(), i32(2, 3), tok), (tok[0], i32(2, 3), tok), (tok, i32(2, 2), tok), (tok, i32(2, 3), tok[:, :2]),
                (tok, i32(2, 3), tok, None, kv), (tok, i32(2, 3), tok, i32(1), kv),
                (tok.repeat(2, 1), i32(3), tok.repeat(2, 1), i32(4), kv), (tok[:, :0], i32(2, 0), tok[:, :0]),
                (tok.repeat(1, 22), i32(66), tok.repeat(1, 22))):
        with pytest.raises(ValueError):
            ops.tree_accept(*bad)
    for bad in ((tok.int(), i32(2, 3), tok), (tok, i32(2, 3).long(), tok), (tok, i32(2, 3), tok, i32(2).long(), kv)):
        with pytest.raises(TypeError):
            ops.tree_accept(*bad)
    for bad in (([], []), ([kc], []), ([kc, kc[:1]], [kc, kc[:1]]), ([kc.cpu()], [kc.cpu()]),
                ([kc], [kc.bfloat16()[:1]])):
        with pytest.raises(ValueError):
            ops.LayerCaches(*bad)
    with pytest.raises(TypeError):
        ops.LayerCaches([kc[..., :4].contiguous()], [kc[..., :4].contiguous()])
    torch.cuda.synchronize()
    _lib.device_status()


@pytest.mark.parametrize("base", [2 ** 63 - 1, 2 ** 63 - 3, -2 ** 63, 2 ** 32])
def test_places_that_no_sum_can_hold(base):
    """A ragged sequence whose rows would begin past every number: flagged, nothing is moved."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    kc, vc = (new_cache((None, 40), 2, 64, torch.bfloat16, gen) for _ in range(2))
    bases = torch.tensor([0, base], device=DEV)
    caps = torch.tensor([20, 20], dtype=torch.int32, device=DEV)
    lens = torch.tensor([3, 3], dtype=torch.int32, device=DEV)
    depths = torch.arange(3, dtype=torch.int32, device=DEV)
    qkv = torch.randn(2, 3, 6 * 64, device=DEV, generator=gen).to(torch.bfloat16)
    table = torch.randn(20, 64, device=DEV, generator=gen).to(torch.bfloat16)
    was = kc.clone(), vc.clone()
    q = ops.rope_kv_append_tree(qkv, lens, depths, table, table, kc, vc, 2, 2, bases, caps)
    assert _lib.device_status() == 2 and (q[1] == 0).all() and (q[0] != 0).any()
    for c, w in zip((kc, vc), was):
        assert torch.equal(c[:, :3], w[:, :3]) and torch.equal(c[:, 6:], w[:, 6:])
    masks = torch.tensor([1, 3, 7], device=DEV)
    out = ops.tree_attention(torch.ones_like(q), kc, vc, lens, masks, seq_base=bases, seq_cap=caps)
    assert _lib.device_status() == 2 and (out[1] == 0).all() and (out[0] != 0).any()
    was = kc.clone(), vc.clone()
    drafted = torch.tensor([[0, 1, 2]] * 2, device=DEV)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV)
    sampled = torch.tensor([[2, 0, 0]] * 2, device=DEV)  # node 2 moves to row 1
    got = ops.tree_accept(drafted, parents, sampled, lens, ops.LayerCaches([kc], [vc], bases, caps))
    assert _lib.device_status() == 2 and got[0].tolist() == [2, 2]
    for c, w in zip((kc, vc), was):
        assert torch.equal(c[:, 4], w[:, 5]) and torch.equal(c[:, 5:], w[:, 5:]) and torch.equal(c[:, :4], w[:, :4])
