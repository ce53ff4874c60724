"""Edges of the operators over drafted trees."""
import pytest
import torch

from llama_pure_compute_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


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
