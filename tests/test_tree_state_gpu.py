"""What a BatchedTreeDecoder and its caches hold between steps."""
import pytest
import torch

from llama_pure_compute_b200 import BatchedTreeDecoder, DraftTree, TreeCache, _lib
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
