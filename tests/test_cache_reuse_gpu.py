"""Decoders and caches that are used again after a capture: what a captured step
reads and writes stays where it is.  Tokens are compared with eager decoders on
fresh caches, exactly."""
import pytest
import torch

from llama_pure_compute_b200 import _lib
from llama_pure_compute_b200.config import LlamaModelConfig
from llama_pure_compute_b200.generate import BatchedGreedyDecoder
from llama_pure_compute_b200.int4_cache import Int4KVCache, Int4RaggedKVCache
from llama_pure_compute_b200.kv_manager import KVCacheManager
from llama_pure_compute_b200.model import LlamaForCausalLM
from llama_pure_compute_b200.ragged_cache import RaggedKVCache
from oracle.model_ref import make_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
SMALL = dict(vocab_size=256, dim=256, inter_dim=384, num_layers=2, num_heads=4, num_kv_heads=2,
             max_seq_len=96)


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0, "a kernel flagged a device-side error"


@pytest.fixture(scope="module")
def model():
    cfg = LlamaModelConfig(**SMALL)
    return cfg, LlamaForCausalLM.from_state_dict(cfg, make_state_dict(SMALL, 7), device=DEV, dtype=BF)


def ragged_cache(kind, cfg, caps):
    return kind(num_layers=cfg.num_layers, capacities=caps, n_kv_heads=cfg.num_kv_heads,
                head_dim=cfg.head_dim, dtype=BF, device=DEV)


def prompts(seed, lens):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]


def churn():
    """Other tensors in the allocator's free blocks."""
    keep = [torch.full((n,), 7, dtype=torch.uint8, device=DEV) for n in (8, 16, 32, 64, 512, 4096) * 20]
    torch.cuda.synchronize()
    return keep


@pytest.mark.parametrize("kind", [RaggedKVCache, Int4RaggedKVCache])
def test_a_captured_ragged_decoder_generates_again(model, kind):
    """The graph of the first generate() serves the next ones, whose prompts select
    the sequences group by group, and another decoder's use of the cache between."""
    cfg, net = model
    caps = [40, 30, 55, 20]
    kv = ragged_cache(kind, cfg, caps)
    dec = BatchedGreedyDecoder(net, kv, 4)
    for seed, lens in ((1, [7, 7, 40, 3]), (2, [30, 2, 2, 11]), (3, [5, 5, 5, 5])):
        p = prompts(seed, lens)
        got = dec.generate(p, 9)
        kept = churn()
        want = BatchedGreedyDecoder(net, ragged_cache(kind, cfg, caps), 4,
                                    use_cuda_graph=False).generate(p, 9)
        assert torch.equal(got, want), seed
        assert kv.seq_lens.tolist() == [n + 8 for n in lens] and len(kept) == 120
    # a selection that someone else left is not the decoder's, captured or eager
    want = BatchedGreedyDecoder(net, ragged_cache(kind, cfg, caps), 4, use_cuda_graph=False)
    for d in (dec, want):
        d.kv.select([3])
        d.prefill(p)
    for _ in range(3):
        dec.kv.select([2, 0])
        want.kv.select([1])
        assert torch.equal(dec.step(), want.step())
    dec.release()


@pytest.mark.parametrize("kind", [RaggedKVCache, Int4RaggedKVCache])
def test_one_token_prompts_between_the_replays(kind):
    """A prompt of one token runs as a decode step of its own batch size: it must not
    take the workspace of the captured step.  Long enough for split sums."""
    cfgd = {**SMALL, "max_seq_len": 3100}
    cfg = LlamaModelConfig(**cfgd)
    net = LlamaForCausalLM.from_state_dict(cfg, make_state_dict(cfgd, 8), device=DEV, dtype=BF)
    caps = [3000, 40, 3000, 50]
    kv = ragged_cache(kind, cfg, caps)
    dec = BatchedGreedyDecoder(net, kv, 4)
    for seed, lens in ((1, [2900, 1, 1, 9]), (2, [1, 2, 2800, 1]), (3, [2950, 1, 2700, 1])):
        p = prompts(seed, lens)
        got = dec.generate(p, 7)
        kept = churn()
        want = BatchedGreedyDecoder(net, ragged_cache(kind, cfg, caps), 4,
                                    use_cuda_graph=False).generate(p, 7)
        assert torch.equal(got, want) and len(kept) == 120, seed
    dec.release()


@pytest.mark.parametrize("kind", [KVCacheManager, Int4KVCache])
def test_decoders_of_two_batch_sizes_on_one_cache(kind):
    """Captured steps of 3 and 2 sequences on the same dense cache, in turns."""
    cfgd = {**SMALL, "max_seq_len": 3100}
    cfg = LlamaModelConfig(**cfgd)
    net = LlamaForCausalLM.from_state_dict(cfg, make_state_dict(cfgd, 9), device=DEV, dtype=BF)

    def cache():
        return kind(num_layers=cfg.num_layers, max_batch_size=3, max_seq_len=cfg.max_seq_len,
                    n_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, dtype=BF, device=DEV)
    kv = cache()
    decs = {b: BatchedGreedyDecoder(net, kv, b) for b in (3, 2)}
    for seed in range(4):
        b = 3 - seed % 2
        p = prompts(seed, [2900, 2850, 3000][:b])
        got = decs[b].generate(p, 6)
        kept = churn()
        want = BatchedGreedyDecoder(net, cache(), b, use_cuda_graph=False).generate(p, 6)
        assert torch.equal(got, want) and len(kept) == 120, seed
    for d in decs.values():
        d.release()
