"""Edges of the operators over drafted trees."""
import math

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("batch,heads,kv", [(2, 2, 2), (2, 32, 2), (80, 8, 8)],
                         ids=["cluster", "wide", "stretches"])
@pytest.mark.parametrize("rows", [128, 256, 4096])
def test_nodes_past_rows_that_end_with_a_tile(rows, batch, heads, kv, ragged):
    """The first sequence fills its rows, a whole number of tiles: its nodes have none.  Visible ones
    are flagged, and the context alone is seen."""
    gen = torch.Generator(device=DEV).manual_seed(rows)
    nodes, dim = 5, 64
    lens = [rows] + [3 + i % 60 for i in range(batch - 1)]
    shape = (kv, batch * rows, dim) if ragged else (batch, kv, rows, dim)
    k, v = (torch.randn(shape, device=DEV, generator=gen).to(BF) for _ in range(2))
    q = torch.randn(batch, heads, nodes, dim, device=DEV, generator=gen).to(BF)
    masks = torch.tensor([[1, 3, 5, 7, 0]] * batch, device=DEV)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    index = {}
    if ragged:
        index = dict(seq_base=torch.arange(batch, device=DEV) * rows,
                     seq_cap=torch.full((batch,), rows, dtype=torch.int32, device=DEV))
    assert _lib.device_status() == 0
    got = ops.tree_attention(q, k, v, seq, masks, **index)
    assert _lib.device_status() == 2
    # bits past the nodes are not read: no flag
    masks[0] = torch.tensor([0, 1 << 5, -1 << 5, 1 << 40, 0], device=DEV)
    assert torch.equal(ops.tree_attention(q, k, v, seq, masks, **index), got)
    assert _lib.device_status() == 0
    k0, v0 = (t[:, :rows] if ragged else t[0] for t in (k, v))
    s = q[0].double().view(kv, -1, dim) @ k0.double().mT * dim ** -0.5
    p = torch.softmax(s, -1)
    want, spread = ((p @ x).view(heads, nodes, dim) for x in (v0.double(), v0.double().abs()))
    # P and the result: half a step each; fp32 scores, exponentials and sums far below
    h = torch.finfo(BF).eps / 2
    assert bool(((got[0].double() - want).abs() <= (h + 2 ** -13) * spread + h * want.abs()).all())


@pytest.mark.parametrize("heads,kv", [(160, 160), (160 * 64, 160), (8, 1)], ids=["narrow", "wide", "one"])
@pytest.mark.parametrize("gap", [14.0, 20.0, 25.5, 28.0])
@pytest.mark.parametrize("n", [3000, 20000])
def test_many_small_weights_in_fp16(n, gap, heads, kv):
    """One key far above all others, which weigh 2^-gap of it each: together they count, although
    fp16 would hold the single weight as a subnormal, or as nothing.

    The kernel holds a weight as fp16 at 2^7 times its size relative to the reference, which is at
    most the largest: it is off by half a step (2^-11 of it), or, where that is subnormal, by 2^-25
    * 2^-7 of the largest weight.  So the result by h * (sum p |v|) + keys * 2^-32 * max |v|, besides
    a score's and an exponential's fp32 errors and the result's own rounding."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    dim, nodes = 64, 3
    k = torch.zeros(1, kv, n + nodes, dim, device=DEV, dtype=FP)
    v = torch.empty_like(k).uniform_(0.5, 1.0, generator=gen)
    top = 1  # the tiles behind it meet its reference, where a CTA has them all
    k[:, :, top, 0] = 4.0
    v[:, :, top] = 0
    q = torch.zeros(1, heads, nodes, dim, device=DEV, dtype=FP)
    q[..., 0] = 4.0
    scale = gap / 16 / math.log2(math.e)  # scores of gap octaves and 0
    masks = torch.tensor([1, 3, 5], device=DEV)
    seq = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = ops.tree_attention(q, k, v, seq, masks, sm_scale=scale)[0].double()
    h = torch.finfo(FP).eps / 2
    for t in range(nodes):
        rows = list(range(n)) + [n + i for i in range(nodes) if int(masks[t]) >> i & 1]
        s = (k[0][:, rows].double() @ q[0, 0, t].double()) * scale  # the heads' queries are alike
        p = torch.softmax(s, -1)
        want = (p[:, None] @ v[0][:, rows].double())[:, 0].repeat_interleave(heads // kv, 0)
        # an exponent of up to `gap` from four roundings, times ln 2; 2^-20 for sums over the keys
        fp32 = 2.0 ** -24 * 4 * gap + 2.0 ** -22 + 2.0 ** -20
        bound = (2 * h + fp32) * want + len(rows) * 2.0 ** -32 + 2.0 ** -25
        err = (got[:, t] - want).abs()
        assert bool((err <= bound).all()), (err / bound).max().item()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("step", [0.25, 9.0, 16.0])
@pytest.mark.parametrize("sign", [1, -1])
def test_maxima_that_grow_in_fp16(step, sign):
    """Scores that rise or fall by `step` octaves a tile: weights stay in fp16's range before and
    after the reference moves."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    n, nodes, dim = 128 * 14, 4, 64
    k = torch.zeros(1, 2, n + nodes, dim, device=DEV, dtype=FP)
    tile = torch.arange(n + nodes, device=DEV) // 128
    k[..., 0] = (tile * sign).to(FP)
    k[..., 1] = torch.rand(n + nodes, device=DEV, generator=gen).to(FP)
    v = torch.randn(k.shape, device=DEV, generator=gen).to(FP)
    q = torch.zeros(1, 4, nodes, dim, device=DEV, dtype=FP)
    q[..., 0], q[..., 1] = 1.0, 0.5
    scale = step / math.log2(math.e)
    masks = torch.tensor([1, 3, 5, 9], device=DEV)
    got = ops.tree_attention(q, k, v, torch.tensor([n], dtype=torch.int32, device=DEV), masks, sm_scale=scale)[0]
    h = torch.finfo(FP).eps / 2
    for t in range(nodes):
        rows = list(range(n)) + [n + i for i in range(nodes) if int(masks[t]) >> i & 1]
        s = (k[0][:, rows].double() @ q[0, 0, t].double()) * scale
        p = torch.softmax(s, -1)
        want, spread = (torch.einsum("kr,krd->kd", p, x).repeat_interleave(2, 0)
                        for x in (v[0][:, rows].double(), v[0][:, rows].double().abs()))
        fp32 = 2.0 ** -24 * 4 * 15 * step + 2.0 ** -22 + 2.0 ** -20
        bound = (h + fp32) * spread + h * want.abs() + len(rows) * 2.0 ** -32 * v.abs().max().item() + 2.0 ** -25
        err = (got[:, t].double() - want).abs()
        assert bool((err <= bound).all()), (err / bound).max().item()


def test_a_cache_is_handed_over_once():
    """tree_accept moves every cache by itself: the same memory twice would be moved twice at once."""
    a, b, c = (torch.zeros(2, 2, 16, 32, device=DEV, dtype=BF) for _ in range(3))
    ops.LayerCaches([a, b], [c, a.clone()])
    both = torch.zeros(3, 2, 16, 32, device=DEV, dtype=BF)
    for keys, values in (([a], [a]), ([a, b], [c, b]), ([a, a], [b, c]), ([both[:2]], [both[1:]])):
        with pytest.raises(ValueError, match="memory"):
            ops.LayerCaches(keys, values)
    ops.LayerCaches([both[:1]], [both[1:2]])  # side by side


def test_nodes_that_only_fill_up_a_smaller_tree():
    """A negative parent: nobody's child, whatever the token, and no fault of the tree's."""
    parents = torch.tensor([[-1, 0, 1, -1], [-1, 0, -2 ** 31, -5]], dtype=torch.int32, device=DEV)
    drafted = torch.tensor([[3, 4, -1, -1], [3, 4, 5, -1]], device=DEV)
    sampled = torch.tensor([[4, -1, -1, -1], [4, 5, -1, 0]], device=DEV)
    accepted, tokens, path = ops.tree_accept(drafted, parents, sampled)
    assert accepted.tolist() == [3, 2] and path.tolist() == [[0, 1, 2, -1], [0, 1, -1, -1]]
    assert tokens.tolist() == [[4, -1, -1, -1], [4, 5, -1, -1]]
    assert _lib.device_status() == 0
