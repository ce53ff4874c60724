"""The model on 4-bit caches and 4-bit weights.

Caches: every layer's append and attention of a forward is recorded and held to
64-bit attention over the rows that the cache then holds (the bars of the
operators' tests; prefill goes through the 16-bit kernel on rows rounded to
bf16, whose own bar against an oracle is 2e-2).  Weights: greedy tokens against
the fp32 oracle on the dequantised weights, with the tie tolerance that the
16-bit model is held to."""
import pytest
import torch

from llama_pure_compute_b200 import _lib, int4_cache, ops
from llama_pure_compute_b200.config import LlamaModelConfig
from llama_pure_compute_b200.generate import (BatchedGreedyDecoder, GenerationConfig,
                                              LlamaGenerator)
from llama_pure_compute_b200.int4_cache import Int4KVCache, Int4RaggedKVCache
from llama_pure_compute_b200.int4_linear import Int4Weight
from llama_pure_compute_b200.kv_manager import KVCacheManager
from llama_pure_compute_b200.model import LlamaForCausalLM
from oracle.int4_ref import attention_ref, rows_ref, weight_ref
from oracle.model_ref import OracleLlama, make_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
SMALL = dict(vocab_size=256, dim=256, inter_dim=384, num_layers=2, num_heads=4, num_kv_heads=2,
             max_seq_len=96)


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0


def build(cfgd, seed=0):
    cfg = LlamaModelConfig(**cfgd)
    sd = make_state_dict(cfgd, seed)
    return cfg, LlamaForCausalLM.from_state_dict(cfg, sd, device=DEV, dtype=BF), sd


def dense_cache(cfg, batch, kind=Int4KVCache):
    return kind(num_layers=cfg.num_layers, max_batch_size=batch, max_seq_len=cfg.max_seq_len,
                n_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, dtype=BF, device=DEV)


def held(kv, b, n):
    if kv.ragged:
        at = int(kv.seq_base[b])
        pick = lambda t: t[:, at:at + n]  # noqa: E731
    else:
        pick = lambda t: t[b, :, :n]  # noqa: E731
    return (rows_ref(pick(kv.key_codes), pick(kv.key_scales)),
            rows_ref(pick(kv.value_codes), pick(kv.value_scales)))


@pytest.fixture
def recorded(monkeypatch):
    """(cache handle, q, positions of the queries, output, decode step or not) of
    every attention call of the caches."""
    calls = []
    append = int4_cache.rope_kv_append_int4

    def spy(kv, context, qkv, positions, ctx, num_heads, scale):
        seen = {}

        def keep(*a):
            seen["q"] = append(*a)
            return seen["q"]
        monkeypatch.setattr(int4_cache, "rope_kv_append_int4", keep)
        out = plain(kv, context, qkv, positions, ctx, num_heads, scale)
        # the decoder advances its positions in place; cache rows are overwritten by no
        # later call and can be read afterwards
        calls.append((kv, seen["q"], positions.clone(), out, ctx.decode, scale))
        return out
    plain = int4_cache._attend
    monkeypatch.setattr(int4_cache, "_attend", spy)
    return calls


def check(calls):
    for kv, q, positions, out, decode, scale in calls:
        B, H, S, D = q.shape
        o = out.view(B, S, H, D)
        for b in range(B):
            for s in ({0, S // 2, S - 1}):
                n = int(positions[b, s]) + 1
                k, v = held(kv, b, n)
                want, size = attention_ref(q[b, :, s], k, v, scale)
                far = (o[b, s].double() - want).abs()
                bar = want.abs() * 2.0 ** -9 + size * 2.0 ** -7 if decode else \
                    torch.full_like(want, 2e-2)
                assert (far <= bar).all(), (b, s, n, decode, (far / bar).max().item())


def test_dense_cache_prompt_in_two_chunks_then_decode(recorded):
    cfg, model, _ = build(SMALL)
    kv = dense_cache(cfg, 3)
    kv.begin_request(3)
    ids = torch.randint(0, 256, (3, 50), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    whole = dense_cache(cfg, 3)
    with torch.inference_mode():
        for lo, hi in ((0, 33), (33, 50)):
            pos = torch.arange(lo, hi, device=DEV)[None].expand(3, -1)
            logits = model(ids[:, lo:hi], positions=pos, kv_cache=kv)
        pos = torch.arange(50, device=DEV)[None].expand(3, -1)
        other = model(ids, positions=pos, kv_cache=whole)
        for step in range(5):
            pos = torch.full((3, 1), 50 + step, device=DEV)
            logits = model(logits[:, -1:].argmax(-1), positions=pos, kv_cache=kv)
    assert kv.seq_lens.tolist() == [55] * 3 and kv.current_seq_len(1) == 55
    assert logits.isfinite().all() and other.isfinite().all()
    assert len(recorded) == (2 + 1 + 5) * cfg.num_layers
    check(recorded)
    # the first layer's rows depend on the tokens alone: one piece or two is the same
    a, b = kv.layers[0], whole.layers[0]
    assert torch.equal(a.key_codes[:, :, :50], b.key_codes[:, :, :50])
    assert torch.equal(a.value_scales[:, :, :50], b.value_scales[:, :, :50])
    k, v = kv.read(layer_idx=1, batch_size=2, seq_len=55)
    for r in range(2):
        rk, rv = held(kv.layers[1], r, 55)
        assert torch.equal(k[r], rk.float().to(BF)) and torch.equal(v[r], rv.float().to(BF))
    kv.reset()
    assert kv.seq_lens.tolist() == [0] * 3


def test_ragged_cache(recorded):
    cfg, model, _ = build(SMALL, 3)
    lens = [7, 40, 1, 23]
    kv = Int4RaggedKVCache(num_layers=cfg.num_layers, capacities=[n + 9 for n in lens],
                           n_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, dtype=BF, device=DEV)
    assert kv.memory_footprint_bytes() == 2 * 2 * 2 * sum(n + 9 for n in lens) * (32 + 8)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in lens]
    dec = BatchedGreedyDecoder(model, kv, 4, use_cuda_graph=False)
    toks = dec.generate(prompts, 6)
    check(recorded)
    del recorded[:]
    # the same sequences one by one in a dense cache
    for i, p in enumerate(prompts):
        one = BatchedGreedyDecoder(model, dense_cache(cfg, 1), 1, use_cuda_graph=False)
        assert one.generate([p], 6).shape == (1, 6)
    check(recorded)
    again = BatchedGreedyDecoder(model, kv, 4, use_cuda_graph=True)
    assert torch.equal(again.generate(prompts, 6), toks)
    again.release()
    with pytest.raises(ValueError, match="capacity"):
        kv.select([2])
        model(torch.zeros(1, 11, dtype=torch.long, device=DEV),
              positions=torch.arange(11, device=DEV)[None], kv_cache=kv)


@pytest.mark.parametrize("name", ["mha", "gqa"])
def test_graph_equals_eager_and_generator(golden, name):
    g = golden("model")[name]
    cfg, model, _ = build(g["cfg"], g["seed"])
    outs = []
    for graph in (True, False):
        dec = BatchedGreedyDecoder(model, dense_cache(cfg, 2), 2, use_cuda_graph=graph)
        outs.append(dec.generate(g["prompt"].to(DEV)[:2], 12).cpu())
        dec.release()
    assert torch.equal(outs[0], outs[1])
    gen = LlamaGenerator(model, cfg, dense_cache(cfg, 1))
    one = list(gen.generate(g["prompt"][0].tolist(), generation=GenerationConfig(max_new_tokens=12)))
    assert len(one) == 12 and one[0] == outs[0][0, 0]
    with pytest.raises(ValueError, match="shorter"):
        LlamaGenerator(model, cfg, Int4KVCache(num_layers=1, max_batch_size=1, max_seq_len=8,
                                               n_kv_heads=2, head_dim=64, dtype=BF))


def test_cache_refusals():
    cfg, model, _ = build(SMALL)
    for bad in (dict(num_layers=0), dict(max_batch_size=0), dict(max_seq_len=0), dict(n_kv_heads=0)):
        kw = dict(num_layers=1, max_batch_size=1, max_seq_len=8, n_kv_heads=2, head_dim=64, dtype=BF)
        with pytest.raises(ValueError):
            Int4KVCache(**{**kw, **bad})
    with pytest.raises(RuntimeError):
        Int4KVCache(num_layers=1, max_batch_size=1, max_seq_len=8, n_kv_heads=2, head_dim=64, device="cpu")
    kv = dense_cache(cfg, 1)
    with pytest.raises(ValueError):
        kv.begin_request(2)
    with pytest.raises(IndexError):
        kv.current_seq_len(1)
    with pytest.raises(IndexError):
        kv.read(layer_idx=9, batch_size=1, seq_len=1)
    with pytest.raises(ValueError):
        kv.read(layer_idx=0, batch_size=1, seq_len=97)
    ids = torch.zeros(1, 97, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="overflow"):
        model(ids, positions=torch.arange(97, device=DEV)[None], kv_cache=kv)
    with pytest.raises(ValueError, match="batch size"):
        model(ids[:, :4].expand(2, -1), positions=torch.arange(4, device=DEV)[None].expand(2, -1),
              kv_cache=kv)


# ---------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------
def dequantised(sd, group, lm_head=True):
    out = {}
    for n, w in sd.items():
        w = w.to(BF)
        if "proj" in n or (lm_head and n == "lm_head.weight"):
            out[n] = weight_ref(*Int4Weight.quantize(w, group)).float()
        else:
            out[n] = w.float()
    return out


@pytest.mark.parametrize("name,group,lm_head", [("mha", 32, True), ("gqa", 64, True),
                                                ("gqa", 64, False)])
def test_int4_weights_greedy_tokens_match_oracle(golden, name, group, lm_head):
    g = golden("model")[name]
    cfgd = g["cfg"]
    cfg, model, sd = build(cfgd, g["seed"])
    before = sum(p.numel() for p in model.parameters())
    model.quantize_weights_int4(group, lm_head=lm_head)
    assert sum(p.numel() for p in model.parameters()) < before / 2
    B, P = g["prompt"].shape
    kv = KVCacheManager(num_layers=cfg.num_layers, max_batch_size=B, max_seq_len=cfg.max_seq_len,
                        n_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, dtype=BF, device=DEV)
    dec = BatchedGreedyDecoder(model, kv, B, use_cuda_graph=True)
    toks = dec.generate(g["prompt"].to(DEV), g["tokens"].shape[1]).cpu()
    dec.release()
    orc = OracleLlama(cfgd, dequantised(sd, group, lm_head), cfgd["max_seq_len"], table_dtype=BF)
    mine, gap, _ = orc.greedy(g["prompt"].cpu(), toks.shape[1], forced=toks)
    bad = (mine != toks) & (gap > 5e-2)
    assert not bad.any(), (bad.nonzero().tolist(), gap.max().item())


def test_int4_weights_and_cache_together_short_and_long_steps():
    """Steps below and above the 4-bit kernels' token limit, with and without a
    cache, give the same logits up to the rounding that the 16-bit model's tokens
    are granted; graph and eager steps agree; a second quantisation is refused."""
    cfg, model, _ = build(SMALL, 5)
    model.quantize_weights_int4(64)
    ids = torch.randint(0, 256, (1, 90), device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    with torch.inference_mode():
        pos = torch.arange(90, device=DEV)[None]
        long = model(ids, positions=pos, kv_cache=dense_cache(cfg, 1, KVCacheManager))[:, :60]
        short = model(ids[:, :60], positions=pos[:, :60], kv_cache=dense_cache(cfg, 1, KVCacheManager))
        free = model(ids[:, :60], positions=pos[:, :60])
    assert (long - short).abs().max() <= 5e-2 and (free - short).abs().max() <= 5e-2
    dec = BatchedGreedyDecoder(model, dense_cache(cfg, 4), 4)
    a = dec.generate(ids[:, :40].view(4, 10), 8)
    dec.release()
    eager = BatchedGreedyDecoder(model, dense_cache(cfg, 4), 4, use_cuda_graph=False)
    assert torch.equal(eager.generate(ids[:, :40].view(4, 10), 8), a)
    with pytest.raises(RuntimeError, match="already"):
        model.quantize_weights_int4(64)
    cfg, model, _ = build({**SMALL, "inter_dim": 352})
    with pytest.raises(ValueError, match="must divide"):
        model.quantize_weights_int4(64)
    assert model.model.layers[0].int4_down is None
