"""Ragged caches and decode workspaces that are used again, host side: the caches'
bookkeeping on CPU tensors (no kernel runs)."""
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
    return kv


def test_a_sequence_is_selected_once():
    """Two rows of a batch on one sequence would append to the same cache rows."""
    kv = ragged()
    with pytest.raises(ValueError, match="twice"):
        kv.select([1, 2, 1])
