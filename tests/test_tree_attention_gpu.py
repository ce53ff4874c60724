"""ops.tree_attention against its definition in 64 bits.

Tolerance, element by element: the weights are rounded to the data type (half a step h = eps / 2 of
them, so h * A with A = sum p |v|), and the result once more (h * |out|).  What fp32 does adds: a
score of D products is off by D 2^-24 (sum |q k|) at most, and ex2.approx by 2^-22, which enters
every weight as a relative error: (D 2^-24 S + 2^-22 + 2^-20) A, S = max |q| |k| scale log2 e, the last
for the sums over up to 2^17 keys in fp32 (tree-wise over tiles of 128)."""
import math
import random

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from oracle.tree_ref import tree_attention_ref, tree_masks_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def trees(batch, nodes, seed=0, back=4):
    r = random.Random(seed)
    return [[-1] + [r.randint(max(0, t - back), t - 1) for t in range(1, nodes)] for _ in range(batch)]


def masks_of(parents):
    return torch.tensor([tree_masks_ref(p)[0] for p in parents], dtype=torch.int64, device=DEV)


class Case:
    def __init__(self, lens, nodes, heads, kv, dim, kind, ragged, seed=0, spare=5, spread=1.0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        self.lens, self.nodes, self.dim = lens, nodes, dim
        B = len(lens)
        if ragged:
            caps = [n + nodes + (i * 3) % 7 for i, n in enumerate(lens)]
            self.bases = [2 + sum(caps[:i]) for i in range(B)]
            self.base = torch.tensor(self.bases, device=DEV)
            self.cap = torch.tensor(caps, dtype=torch.int32, device=DEV)
            shape = (kv, sum(caps) + 5, dim)
        else:
            self.bases = self.base = self.cap = None
            shape = (B + 1, kv, max(lens) + nodes + spare, dim)
        self.k = (torch.randn(shape, device=DEV, generator=gen) * spread).to(kind)
        self.v = torch.randn(shape, device=DEV, generator=gen).to(kind)
        self.q = torch.randn(B, heads, nodes, dim, device=DEV, generator=gen).to(kind)
        self.seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.masks = masks_of(trees(B, nodes, seed))

    def rows(self, t, b, lo=0, hi=None):
        hi = self.lens[b] + self.nodes if hi is None else hi
        if self.bases is None:
            return t[b, :, lo:hi]
        return t[:, self.bases[b] + lo:self.bases[b] + hi]

    def run(self, **kw):
        return ops.tree_attention(self.q, self.k, self.v, self.seq, self.masks, seq_base=self.base,
                                  seq_cap=self.cap, **kw)

    def check(self, got=None, status=0, scale=None, sequences=None):
        got = self.run(sm_scale=scale) if got is None else got
        scale = self.dim ** -0.5 if scale is None else scale
        masks = self.masks.expand(len(self.lens), -1) if self.masks.dim() == 1 else self.masks
        h = torch.finfo(got.dtype).eps / 2
        for b in range(len(self.lens)) if sequences is None else sequences:
            k = self.rows(self.k, b)
            want, spread = tree_attention_ref(self.q[b], k, self.rows(self.v, b), self.lens[b],
                                              masks[b].tolist(), scale)
            s = float(self.q[b].double().norm(dim=-1).max() * torch.nan_to_num(k.double(), 0, 0, 0).norm(dim=-1).max())
            fp32 = self.dim * 2.0 ** -24 * s * scale * math.log2(math.e) + 2.0 ** -22 + 2.0 ** -20
            # the result's smallest step, where it is subnormal
            bound = (h + fp32) * spread + h * want.abs() + torch.finfo(got.dtype).smallest_normal * 2 * h
            err = (got[b].double() - want).abs()
            same = (got[b].double() == want) | (got[b].isnan() & want.isnan())
            assert bool((same | (err <= bound)).all()), (b, (err / bound).nan_to_num(0).max().item())
        assert _lib.device_status() == status
        return got


SHAPES = [  # lens, nodes, heads, kv heads, dim
    ([0], 1, 1, 1, 128), ([1], 1, 4, 4, 64), ([5, 0, 130], 3, 6, 2, 32), ([127, 128, 129], 64, 2, 1, 128),
    ([100, 64, 63, 65], 64, 4, 2, 64), ([1000], 16, 32, 32, 128), ([300, 1, 2000, 77], 24, 32, 8, 128),
    ([900, 31], 33, 16, 2, 128), ([513, 2], 64, 64, 8, 128), ([260, 700], 40, 40, 4, 64), ([90], 50, 48, 1, 32),
    ([257], 64, 10, 2, 128), ([64] * 9, 5, 8, 8, 128),
    # many tiles a CTA: rings that go round, ends of sequences anywhere in a stretch
    ([20000, 3], 4, 16, 8, 128), ([18931, 40], 64, 16, 4, 128), ([9000, 12345], 20, 64, 32, 64),
    ([711 + 37 * i for i in range(40)], 7, 8, 8, 128), ([300 + 61 * i for i in range(40)], 50, 32, 8, 64),
    ([128 * (i % 5) for i in range(60)], 30, 32, 16, 32),
]


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("kind", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, kind, ragged):
    out = Case(*shape, kind, ragged).check()
    assert out.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("nodes,heads,kv", [(7, 4, 2), (64, 8, 2), (40, 3, 1)])
def test_any_masks(nodes, heads, kv, ragged):
    """Masks need not be a tree's: rows of nothing, of all, bits past the nodes, self left out."""
    c = Case([3, 0, 129], nodes, heads, kv, 64, BF, ragged)
    g = torch.Generator().manual_seed(nodes)
    m = torch.randint(-2 ** 63, 2 ** 63 - 1, (3, nodes), generator=g)
    m[:, 0], m[:, 1], m[:, 2] = 0, -1, 1 << (nodes - 1) if nodes < 64 else -2 ** 63
    if nodes < 64:
        m[1, 3] = -1 << nodes  # nothing but bits past the nodes
    c.masks = m.to(DEV)
    out = c.check()
    assert (out[1, :, 0] == 0).all()  # no context, no node
    c.masks = c.masks[2].contiguous()  # one tree for all sequences
    c.check()


@pytest.mark.parametrize("kind", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("shape", [([100, 0, 127], 9, 4, 2, 128), ([64, 250], 64, 8, 2, 64), ([1100], 6, 4, 4, 32),
                                   ([5, 700], 30, 6, 1, 128)], ids=str)
def test_what_is_not_seen_does_not_count(shape, ragged, kind):
    """NaN and infinities in rows behind the nodes, of nodes that nobody sees and of nodes that
    some see: only those that see them are touched."""
    c = Case(*shape, kind, ragged)
    nodes, clean = c.nodes, c.run().clone()
    r = random.Random(1)
    for b, n in enumerate(c.lens):
        if c.bases is None:  # behind the nodes, up to the end of the sequence's rows
            for t, x in ((c.k, math.nan), (c.v, math.inf)):
                t[b, :, n + nodes:] = x
    if c.bases is not None:  # rows of nobody, and those between the sequences
        own = torch.zeros(c.k.shape[1], dtype=torch.bool, device=DEV)
        for b in range(len(c.lens)):
            own[c.bases[b]:c.bases[b] + c.lens[b] + nodes] = True
        c.k[:, ~own] = math.nan
        c.v[:, ~own] = -math.inf
    assert torch.equal(c.check(), clean)
    lost = nodes // 2  # a node that nobody sees, as one that was skipped
    masks = c.masks & ~(1 << lost)
    c.masks = masks
    clean = c.check().clone()
    for b, n in enumerate(c.lens):
        c.rows(c.k, b)[:, n + lost] = math.nan
        c.rows(c.v, b)[:, n + lost] = math.nan
    assert torch.equal(c.check(), clean)
    for what in (math.nan, math.inf, -math.inf):
        for b, n in enumerate(c.lens):
            leaf = nodes - 1 - r.randint(0, 1)
            c.rows(c.v, b)[:, n + leaf, r.randint(0, c.dim - 1)] = what
        out = c.check()
        touched = out.isnan() | out.isinf()
        assert touched.any() and not touched[:, :, :nodes // 3].any()
    for b, n in enumerate(c.lens):  # NaN keys: whole rows of those who see them
        c.rows(c.k, b)[:, n + nodes - 1, 0] = math.nan
    out = c.check()
    sees = (c.masks >> (nodes - 1) & 1).bool()
    assert out.transpose(1, 2)[sees].isnan().all()
    # NaN in the context reaches all of the sequence, and no other
    c = Case(*shape, kind, ragged)
    b = max(range(len(c.lens)), key=lambda i: c.lens[i])
    c.rows(c.v, b)[:, c.lens[b] // 2] = math.nan
    out = c.check()
    assert out[b].isnan().all() and not any(out[i].isnan().any() for i in range(len(c.lens)) if i != b)


@pytest.mark.parametrize("heads,kv", [(4, 4), (16, 1)])
def test_maxima_that_grow(heads, kv):
    """Scores that rise along the sequence by far more than the reference may lag, and fall."""
    for sign in (1, -1):
        c = Case([1500, 640], 16, heads, kv, 64, BF, False, spread=0.1)
        ramp = torch.arange(c.k.shape[2], device=DEV)[:, None] / 10 * sign
        c.q[..., 0] = 3
        c.k[..., 0] = ramp[:, 0].to(BF)
        c.check()
        c.check(scale=2.0)


def test_rows_past_the_sequence():
    """Lengths that leave no room: cut to the rows, flagged; nodes past them are not read."""
    for ragged in (False, True):
        c = Case([60, 20, 33], 8, 4, 2, 64, FP, ragged, spare=0)
        room = [68, 68, 68] if not ragged else c.cap.tolist()
        c.lens = [room[0] - 3, 20, room[2]]
        c.seq = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
        out = c.run()
        assert _lib.device_status() == 2
        full = c.masks.clone()
        c.masks = full & torch.tensor([[0b111], [0xff], [0]], device=DEV)  # what those rows can hold
        assert torch.equal(c.run(), out) and _lib.device_status() == 0
        c.masks = full
        for bad in (-1, 2 ** 31 - 1, room[1] + 1):
            c.seq[1] = bad
            c.run()
            assert _lib.device_status() == 2
    c = Case([60, 20], 8, 4, 2, 64, FP, True)
    good = c.run().clone()
    for field, bad in (("base", -1), ("base", 2 ** 40), ("cap", -5), ("cap", 10 ** 6)):
        was = getattr(c, field).clone()
        getattr(c, field)[1] = bad
        out = c.run()
        assert _lib.device_status() == 2 and torch.equal(out[0], good[0]) and not out[1].isnan().any()
        getattr(c, field).copy_(was)


def test_empty_capacity():
    c = Case([4, 0, 9], 3, 2, 2, 32, BF, True)
    c.cap[1] = 0
    c.masks[1] = 0
    out = c.run()
    assert _lib.device_status() == 0 and (out[1] == 0).all()
    c.check(out, sequences=(0, 2))


def test_many_sequences():
    """More sequences than a CTA has threads, of all lengths."""
    r = random.Random(3)
    for ragged in (False, True):
        c = Case([r.choice([0, 1, 50, 200, 300]) for _ in range(900)], 3, 2, 1, 32, BF, ragged)
        c.check(sequences=[0, 1, 383, 384, 385, 767, 768, 899] + r.sample(range(900), 40))


def test_long_cache_past_32_bit_offsets():
    """The last sequence's rows lie past 2^31 elements (4 GB) of the cache."""
    free, _ = torch.cuda.mem_get_info()
    if free < 14 << 30:
        pytest.skip("needs 14 GB")
    n, cap, kv = 70000, 70100, 8
    c = Case([3], 10, 16, 8, 128, BF, False)
    shape = (31, kv, cap, 128)
    assert 30 * kv * cap * 128 > 2 ** 31
    k, v = (torch.empty(shape, dtype=BF, device=DEV) for _ in range(2))
    gen = torch.Generator(device=DEV).manual_seed(5)
    for t in (k, v):
        t[30] = torch.randn(shape[1:], device=DEV, generator=gen, dtype=BF)
    q = torch.randn(31, 16, 10, 128, device=DEV, generator=gen).to(BF)
    lens = torch.zeros(31, dtype=torch.int32, device=DEV)
    lens[30] = n
    k[:30, :, :10], v[:30, :, :10] = 0.5, 0.25
    masks = masks_of(trees(31, 10, 4))
    out = ops.tree_attention(q, k, v, lens, masks)
    assert (out[:30] == 0.25).all()
    c.q, c.k, c.v, c.lens, c.seq, c.masks = q[30:], k[30:], v[30:], [n], lens[30:], masks[30:]
    c.nodes, c.dim = 10, 128
    c.check(out[30:])
    # the same memory as a ragged cache: rows past 2^22, offsets past 2^31 within a head
    rk, rv = (t.view(1, -1, 128) for t in (k, v))
    base = torch.tensor([(30 * kv + h) * cap for h in range(2)], device=DEV)
    cap_t = torch.tensor([cap, cap], dtype=torch.int32, device=DEV)
    got = ops.tree_attention(q[30:, :4].expand(2, -1, -1, -1).contiguous(), rk, rv, lens[30:].expand(2).contiguous(),
                             masks[30:].expand(2, -1).contiguous(), seq_base=base, seq_cap=cap_t)
    c.q = q[30:, :4]
    for h in range(2):
        c.k, c.v = k[30:, h:h + 1], v[30:, h:h + 1]
        c.check(got[h:h + 1])


def test_a_chain_is_decode_attention_step_by_step():
    c = Case([77, 400], 4, 8, 2, 128, BF, False)
    c.masks = torch.tensor([1, 3, 7, 15], device=DEV)
    out = c.check()
    for t in range(4):
        one = ops.decode_attention(c.q[:, :, t].contiguous(), c.k, c.v, c.seq + t + 1)
        h = torch.finfo(BF).eps / 2
        # decode_attention keeps its weights in fp32: this one's half step, and a rounding each
        bound = h * c.v.abs().max() + 2 * h * one.abs() + 1e-5
        assert ((out[:, :, t].float() - one.float()).abs() <= bound).all()


def test_graphs_streams_and_workspaces():
    a = Case([900, 40, 300], 12, 16, 4, 128, BF, False, seed=1)
    b = Case([10, 1200, 600], 12, 16, 4, 128, BF, False, seed=2)
    want = [a.run().clone(), b.run().clone()]
    graphs, outs, spaces = [], [], []
    for c in (a, b):
        spaces.append(ops.tree_attention_workspace(c.q, c.k))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run(workspace=spaces[-1]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):  # two graphs at once, each with its own workspace
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    a.seq.copy_(torch.tensor([5, 600, 33]))  # lengths are read when the graph runs
    a.lens = [5, 600, 33]
    graphs[0].replay()
    torch.cuda.synchronize()
    a.check(outs[0])
    for _ in range(5):  # the same bits every time
        assert torch.equal(a.run(), outs[0])


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("dim,heads,kv,nodes", [(32, 8, 8, 16), (64, 16, 4, 64), (128, 16, 8, 20), (128, 32, 4, 64)])
@pytest.mark.parametrize("batch,most", [(70, 60), (40, 190), (300, 60)])
def test_many_short_items(batch, most, dim, heads, kv, nodes, ragged):
    """Many items of one or two tiles: stretches of whole items, with and without parts to join,
    and more CTAs than SMs."""
    r = random.Random(batch)
    c = Case([r.randint(0, most) for _ in range(batch)], nodes, heads, kv, dim, BF, ragged)
    c.check(sequences=[0, 1, batch - 1] + r.sample(range(batch), 12))


@pytest.mark.parametrize("heads,kv,dim", [(8, 4, 64), (16, 4, 128), (32, 2, 128)])
@pytest.mark.parametrize("most", [60, 300])
def test_values_that_are_not_finite_stay_with_their_sequence(most, heads, kv, dim):
    """Many short items after one another in a CTA, every third with an infinite value that some of
    its nodes see: what is kept about one item's values is not taken for the next one's."""
    r = random.Random(most)
    c = Case([r.randint(0, most) for _ in range(200)], 20, heads, kv, dim, BF, False)
    for b in range(0, 200, 3):
        c.rows(c.v, b)[:, c.lens[b] + r.randint(0, 19), r.randrange(dim)] = r.choice([math.inf, -math.inf, math.nan])
    for _ in range(3):
        out = c.run()
        clean = [b for b in range(200) if b % 3]
        assert not out[clean].isnan().any() and not out[clean].isinf().any()
        c.check(out, sequences=range(0, 200, 7))


def test_views_of_q_and_masks():
    c = Case([50, 7], 6, 4, 2, 64, BF, False)
    want = c.run().clone()
    q, m = c.q, c.masks
    c.q = q.transpose(1, 2).contiguous().transpose(1, 2)
    c.masks = torch.stack([m, m], -1)[..., 0]
    assert torch.equal(c.run(), want)
    big = torch.empty(q.numel() + 1, dtype=BF, device=DEV)
    c.q = big[1:].view(q.shape).copy_(q)  # not 16-byte aligned
    assert torch.equal(c.run(), want)
    empty = ops.tree_attention(q[:0], c.k, c.v, c.seq[:0], m[:0])
    assert empty.shape == (0, 4, 6, 64)


def test_refusals():
    c = Case([5, 9], 4, 4, 2, 64, BF, False)
    q, k, v, n, m = c.q, c.k, c.v, c.seq, c.masks
    base, cap = torch.zeros(2, dtype=torch.int64, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    rk = k[0].contiguous()
    for bad in ((q.cpu(), k, v, n, m), (q[0], k, v, n, m), (q, k.cpu(), v.cpu(), n, m), (q, k, v[:, :1], n, m),
                (q, k, v, n[:1], m), (q, k, v, n.cpu(), m), (q, k, v, n, m[:, :3]), (q, k, v, n, m.cpu()),
                (q[:, :3], k, v, n, m), (q[..., :32], k, v, n, m), (q, k[:1], v[:1], n, m),
                (q, k[:, :, ::2], v[:, :, ::2], n, m), (q, rk, rk, n, m), (q[:, :0], k, v, n, m),
                (q.repeat(1, 1, 17, 1), k, v, n, m.repeat(1, 17)), (q[:, :, :0], k, v, n, m[:, :0])):
        with pytest.raises(ValueError):
            ops.tree_attention(*bad)
    for kw in (dict(sm_scale=0.0), dict(sm_scale=-1.0), dict(sm_scale=math.nan), dict(sm_scale=math.inf),
               dict(workspace=torch.empty(16, dtype=torch.uint8, device=DEV)), dict(seq_base=base),
               dict(workspace=torch.empty(1 << 26, dtype=torch.uint8)), dict(seq_base=base, seq_cap=cap)):
        if "workspace" in kw:
            big = Case([40000], 4, 8, 8, 64, BF, False)  # cut into stretches
            with pytest.raises(ValueError):
                big.run(**kw)
            continue
        with pytest.raises(ValueError):
            ops.tree_attention(q, k, v, n, m, **kw)
    for bad in ((q.half(), k, v, n, m), (q.float(), k.float(), v.float(), n, m), (q, k, v, n.long(), m),
                (q, k, v, n, m.int()), (q, k, v.half(), n, m)):
        with pytest.raises(TypeError):
            ops.tree_attention(*bad)
    with pytest.raises(ValueError):
        ops.tree_attention(q[..., :16].contiguous(), k[..., :16].contiguous(), v[..., :16].contiguous(), n, m)
    for kw in (dict(seq_base=base[:1], seq_cap=cap), dict(seq_base=base.cpu(), seq_cap=cap.cpu())):
        with pytest.raises(ValueError):
            ops.tree_attention(q, rk, rk, n, m, **kw)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
