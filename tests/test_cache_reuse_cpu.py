"""Caches, host side: selections and decode workspaces that are used again, arguments; the
bookkeeping on CPU tensors (no kernel runs)."""
import ctypes
import types
import weakref

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from llama_pure_compute_b200.int4_cache import Int4KVCache, Int4RaggedKVCache
from llama_pure_compute_b200.kv_manager import KVCacheManager, KVCacheSpec
from llama_pure_compute_b200.ragged_cache import RaggedKVCache


def workspaces():
    return getattr(ops, "StepWorkspaces", lambda: None)()


def ragged(caps=(5, 9, 4, 7)):
    """A RaggedKVCache's bookkeeping without its rows, on the CPU."""
    kv = RaggedKVCache.__new__(RaggedKVCache)
    kv.device = torch.device("cpu")
    kv.capacities = list(caps)
    kv.seq_base = torch.tensor([sum(caps[:i]) for i in range(len(caps))])
    kv.seq_cap = torch.tensor(caps, dtype=torch.int32)
    kv.seq_lens = torch.arange(len(caps), dtype=torch.int32)
    kv._captured, kv._ws = [], None
    kv._workspaces = workspaces()
    return kv


def test_a_sequence_is_selected_once():
    """Two rows of a batch on one sequence would append to the same cache rows."""
    kv = ragged()
    with pytest.raises(ValueError, match="twice"):
        kv.select([1, 2, 1])


def test_what_a_captured_step_uses_outlives_the_selection(monkeypatch):
    """A graph holds addresses: the selection that it was captured with must not be
    freed by the next one, nor be written over."""
    kv = ragged()
    kv.head_dim, kv.max_seq_len = 64, 9
    capturing = [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    kv.select(range(4))
    kv.prepare_forward(torch.tensor([[3], [1], [2], [0]]), types.SimpleNamespace(), 2)
    capturing[0] = False
    used = [kv._idx, kv.active_base, kv.active_cap, kv.active_lens]
    kept, values = [weakref.ref(t) for t in used], [t.clone() for t in used]
    assert kv.seq_lens.tolist() == [4, 2, 3, 1]
    del used
    for ids in ([2], [3, 1], range(4)):
        kv.select(ids)
        kv.prepare_forward(torch.zeros(len(ids), 1, dtype=torch.int64), types.SimpleNamespace(), 2)
    assert kv.seq_lens.tolist() == [1] * 4
    assert all(r() is not None and torch.equal(r(), v) for r, v in zip(kept, values))


def bare(kind):
    """A cache's decode_workspace on the CPU, without its rows."""
    kv = kind.__new__(kind)
    kv._ws, kv._workspaces = None, workspaces()
    kv.seq_lens = torch.zeros(4, dtype=torch.int32)
    if kind is KVCacheManager:
        kv.spec = KVCacheSpec(1, 4, 9000, 2, 128, torch.bfloat16, torch.device("cpu"))
    else:
        kv.device, kv.head_dim, kv.max_seq_len = torch.device("cpu"), 128, 9000
    held = _lib.Kv4(16, 16, 16, 16, None, None, 4, 9000, 0, 2, 128, 2, 0)
    kv.layers = [types.SimpleNamespace(ref=ctypes.addressof(held), held=held, index=-1, device="cpu")]
    return kv


@pytest.mark.parametrize("kind", [KVCacheManager, RaggedKVCache, Int4KVCache, Int4RaggedKVCache])
def test_a_captured_workspace_outlives_other_batch_sizes(monkeypatch, kind):
    kv = bare(kind)
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    eager = weakref.ref(kv.decode_workspace(2, 4))
    assert kv.decode_workspace(2, 4) is eager()
    capturing[0] = True
    graph = weakref.ref(kv.decode_workspace(4, 4))
    assert graph().nbytes > 16
    capturing[0] = False
    kv.decode_workspace(1, 4)
    kv.decode_workspace(3, 4)
    assert eager() is None  # no more than the last one is kept for eager steps
    assert graph() is not None and kv.decode_workspace(4, 4) is graph()


def test_int4_cache_read_of_negative_sizes():
    """-1 is no batch: expand() would take it for one row."""
    kv = Int4KVCache.__new__(Int4KVCache)
    kv.num_layers, kv.max_batch_size, kv.max_seq_len, kv.device = 1, 4, 10, torch.device("cpu")
    for batch, seq in ((-1, 3), (2, -3)):
        with pytest.raises(ValueError, match="negative"):
            kv.read(layer_idx=0, batch_size=batch, seq_len=seq)
