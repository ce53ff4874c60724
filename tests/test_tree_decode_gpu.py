"""Speculative decoding over drafted trees: the model's forward over a tree, the decoder's tokens.

Greedy tokens are held to the fp32 oracle, teacher-forced on them: equal, or within the oracle's own
near-tie (as the greedy decoder's are).  Drawn tokens are held to the definition on the decoder's
own logits."""
import random

import pytest
import torch

from llama_pure_compute_b200 import (BatchedTreeDecoder, DraftTree, Int4KVCache, TreeCache, _lib, ops)
from llama_pure_compute_b200.config import LlamaModelConfig
from llama_pure_compute_b200.generate import (BatchedGreedyDecoder, GenerationConfig, LlamaGenerator,
                                              sample_next_token)
from llama_pure_compute_b200.kv_manager import KVCacheManager
from llama_pure_compute_b200.model import LlamaForCausalLM
from llama_pure_compute_b200.ragged_cache import RaggedKVCache
from oracle.model_ref import OracleLlama, make_state_dict
from oracle.tree_ref import accept_ref, sample_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TIE = 5e-2
SHAPE = dict(vocab_size=320, dim=256, inter_dim=512, num_layers=3, num_heads=4, num_kv_heads=2,
             max_seq_len=160, rms_norm_eps=1e-5, rope_theta=10000.0)
TREE = [-1, 0, 0, 0, 1, 1, 2, 4, 4, 7, 9]  # branches of up to five


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0


@pytest.fixture(scope="module")
def model():
    cfg = LlamaModelConfig(**SHAPE)
    sd = make_state_dict(SHAPE, 11)
    m = LlamaForCausalLM.from_state_dict(cfg, sd, device=DEV, dtype=torch.bfloat16)
    m.oracle = OracleLlama(SHAPE, {k: v.bfloat16().float() for k, v in sd.items()}, cfg.max_seq_len,
                           table_dtype=torch.bfloat16)
    return m


def cache_of(model, ragged, batch, rows=150):
    c = model.config
    if ragged:
        return RaggedKVCache(num_layers=c.num_layers, capacities=[rows - i for i in range(batch)],
                             n_kv_heads=c.num_kv_heads, head_dim=c.head_dim, dtype=torch.bfloat16, device=DEV)
    return KVCacheManager(num_layers=c.num_layers, max_batch_size=batch, max_seq_len=rows, n_kv_heads=c.num_kv_heads,
                          head_dim=c.head_dim, dtype=torch.bfloat16, device=DEV)


def prompts_of(lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, SHAPE["vocab_size"], (n,), generator=g).tolist() for n in lens]


class Guesses:
    """Drafts for the tree from texts that are known: along each branch the right continuation with
    probability `right`, else anything."""

    def __init__(self, tree_parents, texts, right, seed=0):
        self.parents, self.texts, self.right = tree_parents, texts, right
        self.r = random.Random(seed)
        self.at = [0] * len(texts)  # how much of each text the decoder has
        self.calls = 0

    def __call__(self, roots):
        self.calls += 1
        out = []
        for b, text in enumerate(self.texts):
            depth = [0]
            row = []
            for t in range(1, len(self.parents)):
                depth.append(depth[self.parents[t]] + 1)
                i = self.at[b] + depth[t] - 1
                hit = i < len(text) and self.r.random() < self.right
                row.append(text[i] if hit else self.r.randrange(SHAPE["vocab_size"]))
            out.append(row)
        return torch.tensor(out, device=DEV)


def run(dec, prompts, steps, guesses):
    """Prefill and steps; the tokens of each sequence."""
    first = dec.prefill(prompts).tolist()
    got = [[t] for t in first]
    for b in range(len(got)):
        guesses.at[b] = 1
    for _ in range(steps):
        tokens, accepted = dec.step()
        for b, (row, n) in enumerate(zip(tokens.tolist(), accepted.tolist())):
            got[b] += row[:n]
            assert row[n:] == [-1] * (len(row) - n)
            guesses.at[b] += n
    return got


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_greedy_is_greedy(model, ragged, graph):
    prompts = prompts_of([5, 17, 17, 40])
    kv = cache_of(model, ragged, 4)
    plain = BatchedGreedyDecoder(model, kv, 4, use_cuda_graph=False)
    texts = plain.generate(prompts, 30).tolist()
    guesses = Guesses(TREE, texts, 0.8)
    dec = BatchedTreeDecoder(model, cache_of(model, ragged, 4), 4, DraftTree(TREE), guesses, use_cuda_graph=graph)
    got = run(dec, prompts, 8, guesses)
    assert guesses.calls == 8 and max(map(len, got)) > 9  # drafts were accepted
    for p, tokens in zip(prompts, got):
        forced = torch.tensor([tokens])
        mine, gap, _ = model.oracle.greedy(torch.tensor([p]), len(tokens), forced=forced)
        assert ((mine == forced) | (gap <= TIE)).all()
    lens = dec.cache.lens.tolist()
    assert lens == [len(p) + len(g) - 1 for p, g in zip(prompts, got)]
    # what the cache holds is what a plain run over the same tokens holds, up to bf16's noise
    for b, (p, tokens) in enumerate(zip(prompts, got)):
        one = cache_of(model, False, 1)
        ids = torch.tensor([p + tokens[:-1]], device=DEV)
        model(ids, positions=torch.arange(ids.shape[1], device=DEV)[None], kv_cache=one)
        for layer in range(model.config.num_layers):
            for mine, theirs in ((dec.kv.k_cache, one.k_cache), (dec.kv.v_cache, one.v_cache)):
                if ragged:
                    at = dec.kv.bases[b]
                    x = mine[layer][:, at:at + lens[b]]
                else:
                    x = mine[layer][b, :, :lens[b]]
                y = theirs[layer][0, :, :lens[b]]
                assert (x.float() - y.float()).abs().max() <= 2 ** -5 * y.float().abs().max()
    dec.release()


def test_a_forward_over_a_tree_is_a_forward_over_each_branch(model):
    prompts = prompts_of([9, 30])
    tree = DraftTree(TREE)
    kv = cache_of(model, False, 2)
    BatchedGreedyDecoder(model, kv, 2, use_cuda_graph=False).prefill(prompts)
    ids = torch.randint(0, 320, (2, tree.nodes), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    cache = TreeCache(kv, 2, tree)
    logits = model(ids, positions=cache.lens[:, None].long() + tree.depths, kv_cache=cache)
    for t in range(tree.nodes):
        branch, a = [], t
        while a >= 0:
            branch.insert(0, a)
            a = TREE[a]
        for b, p in enumerate(prompts):
            full = model(torch.tensor([p + ids[b, branch].tolist()], device=DEV))
            assert (logits[b, t].float() - full[0, -1].float()).abs().max() < TIE


@pytest.mark.parametrize("settings", [dict(temperature=0.9, top_k=50, top_p=0.9), dict(temperature=1.2, min_p=0.02),
                                      dict(temperature=0.7, top_p=0.8)], ids=str)
def test_draws_are_the_definitions(model, settings):
    """Each step's draws from its own logits; the branch that they agree with; the same text again
    from the same random numbers, with and without a graph."""
    prompts = prompts_of([6, 25])
    texts = []
    for graph in (True, False):
        seen = []

        class Watched(torch.nn.Module):
            config = model.config

            def forward(self, ids, **kw):
                out = model(ids, **kw)
                if not graph:
                    seen.append((ids.clone(), kw["positions"].clone(), out.clone()))
                return out
        guesses = Guesses(TREE, texts[0] if texts else [[], []], 0.9)
        dec = BatchedTreeDecoder(Watched(), cache_of(model, False, 2), 2, DraftTree(TREE), guesses, use_cuda_graph=graph,
                                 generator=torch.Generator(device=DEV).manual_seed(8), **settings)
        got = run(dec, prompts, 6, guesses)
        texts.append(got)
        if graph:
            dec.release()
            continue
        u = dec.uniforms.cpu()
        steps = [s for s in seen if s[0].shape == (2, len(TREE))]
        at = [1, 1]
        for ids, positions, logits in steps:
            for b in range(2):
                draws = [sample_ref(logits[b, t], u[b, positions[b, t] + 1].item(),
                                    **{k: torch.tensor(v).item() for k, v in settings.items()})
                         for t in range(len(TREE))]
                path, tokens = accept_ref(ids[b].tolist(), TREE, draws)
                assert got[b][at[b]:at[b] + len(tokens)] == tokens
                at[b] += len(tokens)
        assert at == [len(g) for g in got] and max(at) > 7
    # a draw depends on its position alone, not on what was drafted (up to bf16's noise of the
    # logits, which moves few borders: the first tokens at least)
    assert all(a[:4] == b[:4] for a, b in zip(*texts))


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
def test_generate(model, ragged):
    prompts = prompts_of([4, 11, 30])
    plain = BatchedGreedyDecoder(model, cache_of(model, ragged, 3), 3, use_cuda_graph=False)
    texts = plain.generate(prompts, 25).tolist()
    tree = DraftTree.chain(6)
    guesses = Guesses([-1, 0, 1, 2, 3, 4], texts, 0.7)
    dec = BatchedTreeDecoder(model, cache_of(model, ragged, 3), 3, tree, guesses)
    for _ in range(2):  # the second run replays the first one's graph
        guesses.at = [1, 1, 1]
        got = dec.generate(prompts, 25)
        assert got.shape == (3, 25)
        for p, tokens in zip(prompts, got.cpu()):
            mine, gap, _ = model.oracle.greedy(torch.tensor([p]), 25, forced=tokens[None])
            assert ((mine[0] == tokens) | (gap[0] <= TIE)).all()
    with pytest.raises(ValueError, match="rows"):
        dec.generate(prompts_of([140, 4, 4]), 25)
    dec.release()


def test_root_alone_is_batched_sampling(model):
    """Trees of one node: plain sampling of a batch, without a drafter."""
    prompts = prompts_of([12, 12, 5])
    dec = BatchedTreeDecoder(model, cache_of(model, False, 3), 3, DraftTree([-1]), temperature=0.8, top_k=20,
                             generator=torch.Generator(device=DEV).manual_seed(1))
    a = dec.generate(prompts, 10)
    dec.generator.manual_seed(1)
    assert torch.equal(dec.generate(prompts, 10), a)
    dec.generator.manual_seed(2)
    assert not torch.equal(dec.generate(prompts, 10), a)
    dec.release()


def test_generator_with_min_p(model):
    gen = LlamaGenerator(model, model.config)
    torch.manual_seed(0)
    g = GenerationConfig(max_new_tokens=6, temperature=1.0, top_k=0, top_p=1.0, min_p=1.0)
    out = list(gen.generate(prompts_of([7])[0], generation=g))  # min_p 1: the likeliest alone
    greedy = list(gen.generate(prompts_of([7])[0], generation=GenerationConfig(max_new_tokens=6)))
    assert out == greedy
    x = torch.randn(4, 100, device=DEV)
    u = torch.rand(4, device=DEV)
    got = sample_next_token(x, temperature=0.7, top_k=5, top_p=0.9, uniforms=u)
    assert got.shape == (4, 1)
    assert torch.equal(got[:, 0], ops.sample_tokens(x, u, temperature=0.7, top_k=5, top_p=0.9))


def test_refusals(model):
    c = model.config
    kv = cache_of(model, False, 2)
    four = Int4KVCache(num_layers=1, max_batch_size=2, max_seq_len=64, n_kv_heads=2, head_dim=64,
                       dtype=torch.bfloat16, device=DEV)
    tree = DraftTree(TREE)
    with pytest.raises(TypeError, match="KVCacheManager"):
        TreeCache(four, 2, tree)
    with pytest.raises(TypeError, match="KVCacheManager"):
        BatchedTreeDecoder(model, four, 2, tree, lambda r: r)
    with pytest.raises(ValueError, match="drafter"):
        BatchedTreeDecoder(model, kv, 2, tree)
    with pytest.raises(ValueError, match="capacity"):
        TreeCache(kv, 3, tree)
    with pytest.raises(ValueError, match="device"):
        TreeCache(kv, 2, DraftTree(TREE, "cpu"))
    cache = TreeCache(kv, 2, tree)
    with pytest.raises(ValueError, match="forward of"):
        model(torch.zeros(2, 3, dtype=torch.long, device=DEV),
              positions=torch.zeros(2, 3, dtype=torch.long, device=DEV), kv_cache=cache)
    dec = BatchedTreeDecoder(model, kv, 2, tree, lambda r: r)
    with pytest.raises(RuntimeError, match="prefill"):
        dec.step()
    assert c.num_layers == 3


def test_steps_go_on_from_a_prefill_only(model):
    """generate leaves its sequences at different places: step() would take them on wrongly."""
    prompts = prompts_of([6, 9])
    dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, DraftTree([-1]))
    dec.generate(prompts, 5)
    with pytest.raises(RuntimeError, match="prefill"):
        dec.step()
    dec.prefill(prompts)
    dec.step()
    dec.release()


def test_guesses_that_are_no_tokens(model):
    """A drafter without a guess: nothing outside the embedding is read, tokens stay the greedy ones."""
    prompts = prompts_of([6, 9])
    tree = DraftTree(TREE)
    want = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, DraftTree([-1])).generate(prompts, 8)
    for guess in (-1, -2 ** 63, 2 ** 63 - 1, SHAPE["vocab_size"]):
        dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, tree,
                                 lambda r: torch.full((2, tree.nodes - 1), guess, device=DEV), use_cuda_graph=False)
        got = dec.generate(prompts, 8)
        for p, tokens in zip(prompts, got.cpu()):
            mine, gap, _ = model.oracle.greedy(torch.tensor([p]), 8, forced=tokens[None])
            assert ((mine[0] == tokens) | (gap[0] <= TIE)).all()
        assert (got[:, 0] == want[:, 0]).all()
    for bad in (torch.zeros(2, 1, dtype=torch.long, device=DEV), torch.zeros(2, tree.nodes - 1, device=DEV),
                torch.zeros(tree.nodes - 1, dtype=torch.long, device=DEV)):
        dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, tree, lambda r: bad)
        dec.prefill(prompts)
        with pytest.raises(ValueError, match="drafter"):
            dec.step()


def test_logits_that_leave_nothing(model):
    """A model whose logits are NaN gives -1 and does not read embeddings out of range."""
    weight = model.lm_head.weight
    was = weight.detach().clone()
    try:
        with torch.no_grad():
            weight.fill_(float("nan"))
        dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, DraftTree([-1]), use_cuda_graph=False,
                                 temperature=1.0)
        assert (dec.generate(prompts_of([6, 9]), 4) == -1).all()
        x = torch.full((2, 9), float("nan"), device=DEV)
        assert (sample_next_token(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.5) == 0).all()
    finally:
        with torch.no_grad():
            weight.copy_(was)


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
@pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])
def test_root_alone_is_a_decode_step(model, ragged, graph):
    """Trees of one node take the decode step's kernels: its tokens, bit by bit; sequences that
    are done wait for the others."""
    prompts = prompts_of([5, 17, 17, 40])
    want = BatchedGreedyDecoder(model, cache_of(model, ragged, 4), 4, use_cuda_graph=graph).generate(prompts, 20)
    kv = cache_of(model, ragged, 4)
    dec = BatchedTreeDecoder(model, kv, 4, DraftTree([-1]), use_cuda_graph=graph)
    for _ in range(2):
        assert torch.equal(dec.generate(prompts, 20), want)
        assert kv.seq_lens[:4].tolist() == [len(p) + 19 for p in prompts]
    dec.prefill(prompts)
    dec.active[1] = 0  # stays where it is
    for _ in range(3):
        dec.step()
    assert kv.seq_lens[:4].tolist() == [8, 17, 20, 43]
    dec.release()


@pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
def test_root_alone_with_the_fused_projection(ragged):
    """head_dim 128: the decode step projects, rotates and appends in one kernel."""
    shape = dict(SHAPE, num_heads=2, num_kv_heads=1)
    cfg = LlamaModelConfig(**shape)
    m = LlamaForCausalLM.from_state_dict(cfg, make_state_dict(shape, 5), device=DEV, dtype=torch.bfloat16)
    prompts = prompts_of([7, 30, 12])
    want = BatchedGreedyDecoder(m, cache_of(m, ragged, 3), 3).generate(prompts, 15)
    dec = BatchedTreeDecoder(m, cache_of(m, ragged, 3), 3, DraftTree([-1]))
    assert torch.equal(dec.generate(prompts, 15), want)
    dec.release()
