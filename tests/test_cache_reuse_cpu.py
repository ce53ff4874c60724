"""Ragged caches and decode workspaces that are used again, host side: the caches'
bookkeeping on CPU tensors (no kernel runs)."""
import types
import weakref

import pytest
import torch

from llama_pure_compute_b200.ragged_cache import RaggedKVCache


def ragged(caps=(5, 9, 4, 7)):
    """A RaggedKVCache's bookkeeping without its rows, on the CPU."""
    kv = RaggedKVCache.__new__(RaggedKVCache)
    kv.device = torch.device("cpu")
    kv.capacities = list(caps)
    kv.seq_base = torch.tensor([sum(caps[:i]) for i in range(len(caps))])
    kv.seq_cap = torch.tensor(caps, dtype=torch.int32)
    kv.seq_lens = torch.arange(len(caps), dtype=torch.int32)
    kv._captured, kv._ws = [], None
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
