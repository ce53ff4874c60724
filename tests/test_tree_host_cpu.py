"""Operators of speculative decoding, host side: the C ABI's refusals (nothing is launched), the trees'
tensors, and refusals of CPU tensors."""
import ctypes
import math

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from llama_pure_compute_b200.tree_decode import DraftTree, TreeCache
from oracle.tree_ref import accept_ref, sample_ref, tree_masks_ref

OK, INVALID, UNSUPPORTED = _lib.LPC_OK, _lib.LPC_ERR_INVALID, _lib.LPC_ERR_UNSUPPORTED


def call(name, defaults, kw):
    args = dict(defaults, **kw)
    return getattr(_lib.load(), name)(*args.values())


# the addresses are never followed: every call below is refused first, or has no work
SAMPLE = dict(logits=16, stride=100, u=16, tt=None, kt=None, pt=None, mt=None, t=1.0, k=0, p=1.0, m=0.0, out=16,
              rows=4, vocab=100, dtype=0, stream=None)
ATTEND = dict(q=16, k=16, v=16, lens=16, masks=16, masks_stride=8, base=None, cap=None, out=16, ws=None, nbytes=0,
              batch=2, nodes=8, heads=8, kv=2, dim=128, max_batch=2, max_seq_len=256, total_rows=0, scale=0.1, dtype=2,
              stream=None)
APPEND = dict(qkv=16, lens=16, depths=16, depths_stride=8, cos=16, sin=16, rows=64, q=16, k=16, v=16, base=None,
              cap=None, batch=2, nodes=8, heads=8, kv=2, dim=128, max_batch=2, max_seq_len=64, total_rows=0, dtype=2,
              tdtype=2, stream=None)
ACCEPT = dict(drafted=16, parents=16, parents_stride=8, sampled=16, lens=16, ks=None, vs=None, layers=0, base=None,
              cap=None, accepted=16, tokens=16, path=16, batch=2, nodes=8, kv=2, dim=128, max_batch=2, max_seq_len=64,
              total_rows=0, elem=2, stream=None)
TWO = (ctypes.c_void_p * 2)(16, 32)
ODD = (ctypes.c_void_p * 2)(16, 40)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(stride=99), INVALID),
    (dict(t=-1.0), INVALID), (dict(t=math.nan), INVALID), (dict(t=math.inf), INVALID), (dict(p=0.0), INVALID),
    (dict(p=1.5), INVALID), (dict(m=-0.1), INVALID), (dict(m=1.1), INVALID), (dict(vocab=385025, stride=400000), UNSUPPORTED),
    (dict(vocab=770049, stride=800000, dtype=2), UNSUPPORTED), (dict(rows=2 ** 31), UNSUPPORTED),
    (dict(logits=None), INVALID), (dict(u=None), INVALID), (dict(out=None), INVALID), (dict(logits=18), INVALID),
    (dict(rows=0, logits=None), OK),
], ids=str)
def test_sample_refusals(kw, code):
    assert call("lpc_sample_tokens", SAMPLE, kw) == code
    assert code == OK or b"sample_tokens" in _lib.load().lpc_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), UNSUPPORTED), (dict(dim=96), UNSUPPORTED), (dict(base=16), INVALID), (dict(base=16, cap=16), INVALID),
    (dict(total_rows=64), INVALID), (dict(batch=-1), INVALID), (dict(batch=3), INVALID), (dict(nodes=0), INVALID),
    (dict(nodes=65, masks_stride=65), INVALID), (dict(masks_stride=7), INVALID), (dict(heads=7), INVALID),
    (dict(heads=0), INVALID), (dict(kv=0), INVALID), (dict(max_seq_len=0), INVALID), (dict(max_seq_len=2 ** 31), INVALID),
    (dict(batch=70000, max_batch=70000), INVALID), (dict(scale=0.0), INVALID), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(q=None), INVALID), (dict(masks=None), INVALID), (dict(out=24), INVALID),
    (dict(k=8), INVALID), (dict(batch=60000, max_batch=60000, max_seq_len=2 ** 30), UNSUPPORTED), (dict(batch=0), OK),
    (dict(batch=1, kv=8, max_seq_len=60000), INVALID),  # no workspace
], ids=str)
def test_attention_refusals(kw, code):
    assert call("lpc_tree_attention", ATTEND, kw) == code
    assert code == OK or b"tree_attention" in _lib.load().lpc_last_error()


def test_attention_workspace():
    ws = _lib.load().lpc_tree_attention_workspace_bytes
    assert ws(0, 8, 8, 2, 128, 256, 0) == 0 and ws(1, 8, 8, 2, 96, 256, 0) == 0 and ws(1, 65, 8, 2, 128, 256, 0) == 0
    assert ws(1, 8, 8, 2, 128, 2 ** 31, 0) == 0 and ws(60000, 8, 8, 2, 128, 2 ** 30, 0) == 0
    assert ws(1, 16, 32, 32, 128, 1064, 0) == 0                 # clusters join in shared memory
    narrow, wide = ws(32, 24, 32, 8, 128, 4120, 0), ws(3, 64, 64, 8, 128, 60081, 0)
    # two parts a CTA, of 128 or 256 rows of 128 columns, a maximum and a sum
    assert narrow % (2 * 128 * 130 * 4 + 16) == 0 and wide % (2 * 256 * 130 * 4 + 16) == 0 and narrow > 0 < wide


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), INVALID), (dict(batch=3), INVALID), (dict(heads=0), INVALID), (dict(dim=0), INVALID),
    (dict(depths_stride=7), INVALID), (dict(max_seq_len=0), INVALID), (dict(base=16), INVALID), (dict(rows=0), INVALID),
    (dict(base=16, cap=16), INVALID), (dict(dtype=0), UNSUPPORTED), (dict(dim=24), UNSUPPORTED), (dict(qkv=24), UNSUPPORTED),
    (dict(tdtype=1), UNSUPPORTED), (dict(lens=None), INVALID), (dict(depths=None), INVALID), (dict(q=None), INVALID),
    (dict(batch=0), OK), (dict(nodes=0), OK),
], ids=str)
def test_append_refusals(kw, code):
    assert call("lpc_rope_kv_append_tree", APPEND, kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), INVALID), (dict(nodes=0), INVALID), (dict(nodes=65, parents_stride=65), UNSUPPORTED),
    (dict(batch=70000), UNSUPPORTED), (dict(parents_stride=7), INVALID), (dict(layers=-1), INVALID),
    (dict(layers=2), INVALID), (dict(layers=2, ks=TWO, vs=ODD), INVALID), (dict(layers=2, ks=TWO, vs=TWO, lens=None), INVALID),
    (dict(layers=2, ks=TWO, vs=TWO, elem=1), INVALID), (dict(layers=2, ks=TWO, vs=TWO, dim=12), UNSUPPORTED),
    (dict(layers=2, ks=TWO, vs=TWO, batch=3), INVALID), (dict(layers=2, ks=TWO, vs=TWO, base=16), INVALID),
    (dict(layers=2, ks=TWO, vs=TWO, base=16, cap=16), INVALID), (dict(drafted=None), INVALID), (dict(path=None), INVALID),
    (dict(batch=0), OK),
], ids=str)
def test_accept_refusals(kw, code):
    assert call("lpc_tree_accept", ACCEPT, kw) == code
    assert code == OK or b"tree_accept" in _lib.load().lpc_last_error()


def test_draft_tree():
    t = DraftTree([-1, 0, 0, 1, 3], "cpu")
    assert t.nodes == 5 and t.max_depth == 3
    assert t.masks.tolist() == [1, 3, 5, 11, 27] and t.depths.tolist() == [0, 1, 1, 2, 3]
    assert t.parents.dtype == t.depths.dtype == torch.int32 and t.masks.dtype == torch.int64
    wide = DraftTree([-1] + list(range(63)), "cpu")
    assert wide.masks[63] == -1 and wide.masks.tolist() == tree_masks_ref([-1] + list(range(63)))[0]
    assert DraftTree.chain(64, "cpu").masks.tolist() == wide.masks.tolist()
    for bad in ([], [0], [-1, -1], [-1, 1], [-1, 0, 5], [-1] + [0] * 64):
        with pytest.raises(ValueError):
            DraftTree(bad, "cpu")
    with pytest.raises(TypeError):
        TreeCache(object(), 1, t)


def test_cpu_tensors_are_refused():
    x, i32, i64 = torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int64)
    c = torch.zeros(2, 2, 8, 32).half()
    for f in (lambda: ops.sample_tokens(x, x[:, 0]), lambda: ops.tree_accept(i64, i32, i64),
              lambda: ops.LayerCaches([c], [c]), lambda: ops.tree_attention(c, c, c, i32[:, 0], i64),
              lambda: ops.tree_attention_workspace(c, c),
              lambda: ops.rope_kv_append_tree(x[None].half(), i32[:, 0], i32, x, x, c, c, 2, 2)):
        with pytest.raises(ValueError, match="must be on CUDA device"):
            f()


def test_the_definitions():
    """The oracle on cases that can be worked out by hand."""
    logits = torch.tensor([0.125, 0.5, 0.125, 0.25]).log()
    assert [sample_ref(logits, u) for u in (0.0, 0.124, 0.126, 0.624, 0.626, 0.76)] == [0, 0, 1, 1, 2, 3]
    assert [sample_ref(logits, u, top_p=0.6) for u in (0.0, 0.66, 0.67)] == [1, 1, 3]
    assert sample_ref(logits, 0.99, top_k=1) == 1 and sample_ref(logits, 0.99, min_p=0.6) == 1
    assert sample_ref(torch.tensor([1.0, 3, 3]), 0.9, temperature=0) == 1
    assert sample_ref(torch.tensor([-math.inf, math.nan]), 0.5) == -1
    assert accept_ref([9, 5, 5, 7], [-1, 0, 0, 2], [5, 7, 7, 1]) == ([0, 1], [5, 7])
