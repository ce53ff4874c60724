"""What a BatchedTreeDecoder and its caches hold between steps."""
import pytest
import torch

from llama_pure_compute_b200 import BatchedTreeDecoder, DraftTree, TreeCache, _lib
from oracle.tree_ref import accept_ref, sample_ref
from test_tree_decode_gpu import DEV, TIE, TREE, Guesses, cache_of, model, prompts_of  # noqa: F401

pytestmark = pytest.mark.gpu
LAYOUTS = pytest.mark.parametrize("ragged", [False, True], ids=["dense", "ragged"])
GRAPHS = pytest.mark.parametrize("graph", [True, False], ids=["graph", "eager"])


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0


def greedy_by_the_oracle(model, prompts, texts):  # noqa: F811
    for p, tokens in zip(prompts, texts):
        forced = torch.tensor([tokens])
        mine, gap, _ = model.oracle.greedy(torch.tensor([p]), len(tokens), forced=forced)
        assert ((mine == forced) | (gap <= TIE)).all()


def steps(dec, got, n, guesses=None):
    """n steps; the new tokens go behind `got`."""
    for _ in range(n):
        tokens, accepted = dec.step()
        for b, (row, count) in enumerate(zip(tokens.tolist(), accepted.tolist())):
            assert row[count:] == [-1] * (len(row) - count)
            got[b] += row[:count]
            if guesses is not None:
                guesses.at[b] += count


@LAYOUTS
@GRAPHS
@pytest.mark.parametrize("temperature", [0.0, 1.2])
@pytest.mark.parametrize("parents", [[-1], TREE], ids=["root", "tree"])
def test_a_sequence_that_waits_goes_on_where_it_was(model, ragged, graph, parents, temperature):  # noqa: F811
    """active 0: no tokens, the same length and the same root; afterwards the text goes on, and the
    cache holds what a plain run over that text holds."""
    prompts = prompts_of([5, 17, 9])
    texts = [model.oracle.greedy(torch.tensor([p]), 40)[0][0].tolist() for p in prompts]
    guesses = Guesses(parents, texts, 0.7)
    dec = BatchedTreeDecoder(model, cache_of(model, ragged, 3), 3, DraftTree(parents),
                             guesses if len(parents) > 1 else None, use_cuda_graph=graph, temperature=temperature,
                             generator=torch.Generator(device=DEV).manual_seed(2))
    got = [[t] for t in dec.prefill(prompts).tolist()]
    guesses.at = [1, 1, 1]
    for active, n in (([1, 1, 1], 2), ([1, 0, 1], 3), ([0, 1, 0], 3), ([1, 1, 1], 2)):
        dec.active.copy_(torch.tensor(active))
        had = [list(g) for g in got]
        for _ in range(n):
            steps(dec, got, 1, guesses)
            assert dec.tokens[:, 0].tolist() == [g[-1] for g in got]
        for b in range(3):
            assert len(got[b]) >= len(had[b]) + n if active[b] else got[b] == had[b]
    lens = [len(p) + len(g) - 1 for p, g in zip(prompts, got)]
    assert dec.kv.seq_lens[:3].tolist() == lens
    if temperature == 0:
        greedy_by_the_oracle(model, prompts, got)
    for b, (p, tokens) in enumerate(zip(prompts, got)):
        one = cache_of(model, False, 1)
        ids = torch.tensor([p + tokens[:-1]], device=DEV)
        model(ids, positions=torch.arange(ids.shape[1], device=DEV)[None], kv_cache=one)
        for mine, theirs in ((dec.kv.k_cache, one.k_cache), (dec.kv.v_cache, one.v_cache)):
            for x, y in zip(mine, theirs):
                x = x[:, dec.kv.bases[b]:][:, :lens[b]] if ragged else x[b, :, :lens[b]]
                y = y[0, :, :lens[b]]
                assert (x.float() - y.float()).abs().max() <= 2 ** -5 * y.float().abs().max()
    dec.release()


def test_no_steps_after_a_run_that_was_broken_off(model):  # noqa: F811
    """A drafter that raises, a prompt that does not fit: sequences stand anywhere, a prefill comes first."""
    prompts = prompts_of([6, 9])
    tree = DraftTree.chain(3)
    calls = []

    def drafter(roots):
        calls.append(1)
        if len(calls) == 3:
            raise KeyError("no more")
        return torch.zeros(2, 2, dtype=torch.long, device=DEV)
    dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, tree, drafter)
    with pytest.raises(KeyError):
        dec.generate(prompts, 12)
    with pytest.raises(RuntimeError, match="prefill"):
        dec.step()
    dec.prefill(prompts)
    dec.step()
    with pytest.raises(ValueError):
        dec.prefill(prompts_of([6, 400]))
    with pytest.raises(RuntimeError, match="prefill"):
        dec.step()
    with pytest.raises(RuntimeError, match="prefill"):
        dec.capture()
    dec.release()
    fresh = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, tree, drafter)
    with pytest.raises(RuntimeError, match="prefill"):
        fresh.capture()


@GRAPHS
def test_lengths_that_other_caches_read(model, graph):  # noqa: F811
    """Steps of a second run, a selection in between, trees of another shape over the same
    sequences: every TreeCache goes on from the lengths that the ragged cache has."""
    prompts = prompts_of([5, 17])
    kv = cache_of(model, True, 2)
    texts = [model.oracle.greedy(torch.tensor([p]), 40)[0][0].tolist() for p in prompts]
    guesses = Guesses(TREE, texts, 0.8)
    dec = BatchedTreeDecoder(model, kv, 2, DraftTree(TREE), guesses, use_cuda_graph=graph)
    for _ in range(2):  # the second run replays the first one's graph
        got = [[t] for t in dec.prefill(prompts).tolist()]
        guesses.at = [1, 1]
        steps(dec, got, 3, guesses)
        lens = [len(p) + len(g) - 1 for p, g in zip(prompts, got)]
        assert kv.seq_lens.tolist() == kv.active_lens.tolist() == lens
        assert TreeCache(kv, 2, DraftTree.chain(2)).lens.tolist() == lens
    with torch.inference_mode():
        early = TreeCache(kv, 2, DraftTree.chain(3))
        kv.select([1, 0])
        turned = TreeCache(kv, 2, DraftTree([-1]))
        steps(dec, got, 2, guesses)
        for cache, order in ((turned, [1, 0]), (early, [0, 1])):
            T = cache.tree.nodes
            roots = torch.tensor([[got[b][-1]] + [0] * (T - 1) for b in order], device=DEV)
            logits = model(roots, positions=torch.zeros(2, T, dtype=torch.long, device=DEV), kv_cache=cache)
            for i, b in enumerate(order):
                full = model(torch.tensor([prompts[b] + got[b]], device=DEV))
                assert (logits[i, 0].float() - full[0, -1].float()).abs().max() < TIE
            accepted, tokens, _ = cache.accept(roots, logits.argmax(-1))
            for i, b in enumerate(order):
                got[b] += tokens[i, :accepted[i]].tolist()
            assert kv.seq_lens.tolist() == [len(p) + len(g) - 1 for p, g in zip(prompts, got)]
    greedy_by_the_oracle(model, prompts, got)
    dec.release()


@LAYOUTS
def test_capture_leaves_the_lengths(model, ragged):  # noqa: F811
    prompts = prompts_of([5, 17])
    kv = cache_of(model, ragged, 2)
    dec = BatchedTreeDecoder(model, kv, 2, DraftTree.chain(3),
                             lambda r: torch.zeros(2, 2, dtype=torch.long, device=DEV))
    got = [[t] for t in dec.prefill(prompts).tolist()]
    dec.capture()
    assert kv.seq_lens[:2].tolist() == dec.cache.lens.tolist() == [5, 17]
    steps(dec, got, 4)
    greedy_by_the_oracle(model, prompts, got)
    dec.release()


PER_SEQUENCE = [
    dict(temperature=torch.tensor([0.0, 0.8, 1.1])),
    dict(temperature=0.9, top_k=torch.tensor([1, 4, 0])),
    dict(temperature=torch.tensor([0.7, 1.0, 0.0], dtype=torch.float64), top_p=torch.tensor([0.5, 1.0, 0.9]),
         min_p=torch.tensor([0.0, 0.2, 0.0]), top_k=torch.tensor([[30], [0], [2]], dtype=torch.int32)),
]


@LAYOUTS
@pytest.mark.parametrize("parents", [[-1], TREE], ids=["root", "tree"])
@pytest.mark.parametrize("settings", PER_SEQUENCE, ids=["temperature", "top-k", "all"])
def test_settings_of_each_sequence(model, settings, parents, ragged):  # noqa: F811
    """Entries of B sequences hold for all of a sequence's draws: the first token's, by prefill
    groups, and its nodes'."""
    prompts = prompts_of([6, 25, 25])
    T = len(parents)
    seen = []

    class Watched(torch.nn.Module):
        config = model.config

        def forward(self, ids, **kw):
            out = model(ids, **kw)
            seen.append((ids.clone(), kw["positions"].clone(), out.clone()))
            return out
    mine = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    guesses = Guesses(parents, [[], [], []], 0.9)
    made = dict(use_cuda_graph=False, generator=torch.Generator(device=DEV).manual_seed(4), **mine)
    dec = BatchedTreeDecoder(Watched(), cache_of(model, ragged, 3), 3, DraftTree(parents),
                             guesses if T > 1 else None, **made)
    got = [[t] for t in dec.prefill(prompts).tolist()]
    guesses.texts = got
    steps(dec, got, 5, guesses)

    def one(b):  # settings are 32-bit numbers
        return {k: torch.as_tensor(v).reshape(-1).expand(3)[b].to(torch.int32 if k == "top_k" else torch.float32).item()
                for k, v in settings.items()}
    u = dec.uniforms.cpu()
    rows = [(0, seen[0][2][0]), (1, seen[1][2][0]), (2, seen[1][2][1])]  # two groups of prompts
    for b, logits in rows:
        assert got[b][0] == sample_ref(logits[-1], u[b, len(prompts[b])].item(), **one(b))
    at = [1, 1, 1]
    for ids, positions, logits in seen[2:]:
        for b in range(3):
            draws = [sample_ref(logits[b, t], u[b, positions[b, t] + 1].item(), **one(b)) for t in range(T)]
            _, tokens = accept_ref(ids[b].tolist(), parents, draws)
            assert got[b][at[b]:at[b] + len(tokens)] == tokens
            at[b] += len(tokens)
    assert at == [len(g) for g in got]


def test_settings_in_a_captured_step(model):  # noqa: F811
    """The captured step reads the entries when it runs: what a server changes between requests holds."""
    prompts = prompts_of([6, 25])
    t = torch.zeros(2, device=DEV)
    dec = BatchedTreeDecoder(model, cache_of(model, False, 2), 2, DraftTree([-1]), temperature=t, top_k=50)
    greedy = dec.generate(prompts, 12)
    greedy_by_the_oracle(model, prompts, greedy.tolist())
    t[1] = 5.0
    hot = dec.generate(prompts, 12)
    greedy_by_the_oracle(model, prompts[:1], hot[:1].tolist())
    assert not torch.equal(hot[1], greedy[1])
    dec.release()


def test_settings_that_fit_no_sequence(model):  # noqa: F811
    kv = cache_of(model, False, 3)
    for kw in (dict(temperature=torch.ones(2, device=DEV)), dict(top_p=torch.ones(6, device=DEV)),
               dict(min_p=torch.zeros(3)), dict(top_k=torch.zeros((), dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError, match=next(iter(kw))):
            BatchedTreeDecoder(model, kv, 3, DraftTree([-1]), **kw)


@LAYOUTS
def test_a_cache_made_in_inference_mode_is_read_outside(model, ragged):  # noqa: F811
    prompts = prompts_of([9, 30])
    kv = cache_of(model, ragged, 2)
    tree = DraftTree(TREE)
    with torch.inference_mode():
        if ragged:
            kv.select([0, 1])
        cache = TreeCache(kv, 2, tree)
        ids = torch.zeros(2, tree.nodes, dtype=torch.long, device=DEV)
    for b, p in enumerate(prompts):
        if ragged:
            kv.select([b])
        one = kv if ragged else cache_of(model, False, 1)
        model(torch.tensor([p], device=DEV), positions=torch.arange(len(p), device=DEV)[None], kv_cache=one)
        if not ragged:
            for mine, theirs in zip(kv.k_cache + kv.v_cache, one.k_cache + one.v_cache):
                mine[b].copy_(theirs[0])
            kv.seq_lens[b] = len(p)
    with torch.no_grad():
        logits = model(ids, positions=torch.zeros_like(ids), kv_cache=cache)
    for b, p in enumerate(prompts):
        full = model(torch.tensor([p + [0]], device=DEV))
        assert (logits[b, 0].float() - full[0, -1].float()).abs().max() < TIE
