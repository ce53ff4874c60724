"""LlamaGenerator(kv_cache=): a cache that is not the model's is refused by what differs."""
import types

import pytest
import torch

from llama_pure_compute_b200.config import LlamaModelConfig
from llama_pure_compute_b200.generate import LlamaGenerator

CFG = LlamaModelConfig(vocab_size=64, dim=128, inter_dim=192, num_layers=3, num_heads=2, num_kv_heads=1,
                       max_seq_len=32)


def cache(**kw):
    f = dict(num_layers=3, n_kv_heads=1, head_dim=64, dtype=torch.bfloat16, max_seq_len=40,
             seq_lens=torch.zeros(1))
    return types.SimpleNamespace(**{**f, **kw})


@pytest.mark.parametrize("kw,text", [(dict(num_layers=2), "layers"), (dict(n_kv_heads=2), "KV heads"),
                                     (dict(head_dim=32), "head_dim"), (dict(dtype=torch.float16), "dtype"),
                                     (dict(max_seq_len=31), "shorter"),
                                     (dict(seq_lens=torch.zeros(1, device="meta")), "meta")])
def test_another_models_cache(kw, text):
    model = torch.nn.Linear(4, 4).to(torch.bfloat16)
    assert LlamaGenerator(model, CFG, cache()).kv_cache.max_seq_len == 40
    with pytest.raises(ValueError, match=text):
        LlamaGenerator(model, CFG, cache(**kw))
