"""ops.sample_tokens against its definition in 64 bits.  Tokens have to be equal: weights are held
to 2^-44 of the largest, so that a random number would have to fall within ~1e-9 of a border."""
import math

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from oracle.tree_ref import sample_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def check(logits, u, **kw):
    got = ops.sample_tokens(logits, u, **kw)
    flat, us = logits.reshape(-1, logits.shape[-1]).cpu(), u.reshape(-1).tolist()

    def row(name, r):
        v = kw.get(name)
        return {} if v is None else {name: v.reshape(-1)[r].item() if torch.is_tensor(v) else v}
    want = []
    for r in range(flat.shape[0]):
        s = {}
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s.update(row(name, r))
        # settings reach the kernel as 32-bit numbers
        s = {n: torch.tensor(v, dtype=torch.float32).item() if n != "top_k" else v for n, v in s.items()}
        want.append(sample_ref(flat[r], us[r], **s))
    assert got.reshape(-1).tolist() == want
    assert _lib.device_status() == 0
    return got


def rows(n, vocab, kind, seed, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(n, vocab, device=DEV, generator=g) * spread).to(TYPES[kind])
    return x, torch.rand(n, device=DEV, generator=g)


FILTERS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(top_k=50, top_p=0.9),
           dict(top_k=700), dict(temperature=1.5, top_p=0.95), dict(top_p=0.3), dict(min_p=0.05),
           dict(temperature=0.9, top_k=40, top_p=0.8, min_p=0.1), dict(min_p=1.0), dict(top_p=1e-9)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("kw", FILTERS, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()) or "none")
@pytest.mark.parametrize("vocab", [1, 2, 31, 1003, 32000])
def test_filters(vocab, kw, kind):
    x, u = rows(3, vocab, kind, vocab)
    check(x, u, **kw)


@pytest.mark.parametrize("n,vocab,kind", [(1, 128256, "bf16"), (2, 128257, "fp32"), (300, 515, "fp16"),
                                          (1, 385024, "fp32"), (1, 770048, "bf16"), (1, 4097, "bf16")])
def test_sizes(n, vocab, kind):
    x, u = rows(n, vocab, kind, 7)
    check(x, u, top_p=0.9)
    check(x, u, top_k=100, min_p=0.01)
    check(x, u)


@pytest.mark.parametrize("kind", list(TYPES))
def test_settings_of_each_row(kind):
    n = 64
    x, u = rows(n, 777, kind, 3)
    g = torch.Generator(device=DEV).manual_seed(1)
    t = torch.rand(n, device=DEV, generator=g) + 0.3
    t[::5] = 0
    k = torch.randint(-3, 900, (n,), device=DEV, generator=g, dtype=torch.int32)
    p = 1 - torch.rand(n, device=DEV, generator=g)
    p[::3] = 1
    m = torch.rand(n, device=DEV, generator=g) * 0.2
    check(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    check(x, u, top_k=k.long(), top_p=0.9)


@pytest.mark.parametrize("kind", list(TYPES))
def test_equal_logits_go_by_index(kind):
    """Ties at the border of each filter, to the lowest index; sums of equal weights are exact."""
    for vocab in (5, 1000, 40001):
        x = torch.zeros(4, vocab, device=DEV, dtype=TYPES[kind])
        u = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24], device=DEV)
        for kw in (dict(), dict(top_k=3), dict(top_p=0.5), dict(top_p=0.25, top_k=4),
                   dict(temperature=0.0), dict(min_p=1.0), dict(top_k=vocab - 1, top_p=0.75)):
            check(x, u, **kw)
    x = torch.tensor([[1.0, 2, 2, 1, 2, -0.0, 0.0, 0.0]], device=DEV, dtype=TYPES[kind]).repeat(8, 1)
    u = torch.arange(8, device=DEV) / 8
    for kw in (dict(top_k=2), dict(top_k=4), dict(top_p=0.6), dict(top_k=7), dict(top_p=0.2)):
        check(x, u, **kw)


@pytest.mark.parametrize("kind", list(TYPES))
def test_ruled_out_logits(kind):
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, nan, -inf, -inf], [-inf, nan, 1.0, -inf], [inf, 0.0, inf, -inf],
                      [nan, 3.0, 3.0, inf], [-inf, -5.0, nan, -5.0], [-inf, -inf, -inf, -inf]],
                     device=DEV).to(TYPES[kind])
    for step in range(5):
        u = torch.full((6,), step / 5, device=DEV)
        for kw in (dict(), dict(temperature=0.0), dict(top_k=1), dict(top_p=0.5), dict(top_k=3, top_p=0.9)):
            check(x, u, **kw)
    big = torch.full((2, 50000), -inf, device=DEV, dtype=TYPES[kind])
    big[0, 49999] = -3
    assert ops.sample_tokens(big, torch.zeros(2, device=DEV), top_p=0.5).tolist() == [49999, -1]


def test_extremes_of_temperature_and_range():
    x = torch.tensor([[3e38, -3e38, 2.9e38, 0.0], [1e-38, 0.0, -1e-38, 1e-45]], device=DEV)
    u = torch.tensor([0.7, 0.7], device=DEV)
    for t in (1e-38, 1e-3, 1.0, 1e30, 3e38):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.6)):
            check(x, u, temperature=t, **kw)


def test_known_shares():
    """Probabilities 1/2, 1/4, 1/8, 1/8: the draws have those shares, top-p cuts where it should."""
    p = torch.tensor([0.125, 0.5, 0.125, 0.25], device=DEV, dtype=torch.float64)
    n = 4000
    x = p.log().float().repeat(n, 1)
    u = (torch.arange(n, device=DEV) + 0.5) / n
    got = ops.sample_tokens(x, u)
    assert torch.bincount(got, minlength=4).tolist() == [500, 2000, 500, 1000]
    got = ops.sample_tokens(x, u, top_p=0.7)  # 1/2 and 1/4 stay
    share = torch.bincount(got, minlength=4).tolist()
    assert share[0] == share[2] == 0 and abs(share[1] - 2 * n / 3) <= 1


def test_strides_shapes_and_out():
    big = torch.randn(6, 5, 1001, device=DEV)
    u = torch.rand(6, device=DEV)
    check(big[:, -1, :], u, top_k=20)         # a view with its own row stride
    check(big[:, :, ::2], torch.rand(6, 5, device=DEV), top_p=0.8)
    assert check(big[0, 0, 3:], torch.rand((), device=DEV)).shape == ()
    check(big.view(-1)[1:29030].view(29, 1001), torch.rand(29, device=DEV))  # rows off 16 bytes
    out = torch.empty(6, dtype=torch.int64, device=DEV)
    assert ops.sample_tokens(big[:, 0], u, out=out) is out
    assert out.tolist() == ops.sample_tokens(big[:, 0], u).tolist()
    assert ops.sample_tokens(big[:0, 0], u[:0]).shape == (0,)


def test_rows_outside_the_settings():
    x, u = rows(8, 100, "fp32", 1)
    u[0], u[1] = 1.0, math.nan
    t = torch.ones(8, device=DEV)
    t[2], t[3] = -1.0, math.nan
    p = torch.ones(8, device=DEV)
    p[4], p[5] = 0.0, 1.5
    m = torch.zeros(8, device=DEV)
    m[6] = -0.1
    got = ops.sample_tokens(x, u, temperature=t, top_p=p, min_p=m).tolist()
    assert got[:7] == [-1] * 7 and got[7] == sample_ref(x[7], u[7].item())
    assert _lib.device_status() == 2


def test_same_answer_every_time_and_in_a_graph():
    x, u = rows(64, 32000, "bf16", 9, spread=0.5)
    kw = dict(temperature=1.3, top_k=9000, top_p=0.9)
    want = ops.sample_tokens(x, u, **kw)
    for _ in range(20):
        assert torch.equal(ops.sample_tokens(x, u, **kw), want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.sample_tokens(x, u, **kw)
    for seed in (1, 2):
        nx, nu = rows(64, 32000, "bf16", seed, spread=0.5)
        x.copy_(nx)
        u.copy_(nu)
        g.replay()
        assert torch.equal(out, ops.sample_tokens(nx, nu, **kw))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.sample_tokens(x, u, **kw)
    s.synchronize()
    assert torch.equal(out, other)


def test_refusals():
    x, u = rows(4, 10, "fp32", 1)
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_p=0.0), dict(top_p=1.1),
               dict(min_p=-0.1), dict(min_p=2.0), dict(temperature=math.inf)):
        with pytest.raises(ValueError, match="temperature must be"):
            ops.sample_tokens(x, u, **kw)
    for kw in (dict(temperature=u[:3]), dict(top_k=torch.ones(3, dtype=torch.int32, device=DEV)),
               dict(temperature=u.cpu())):
        with pytest.raises(ValueError):
            ops.sample_tokens(x, u, **kw)
    with pytest.raises(TypeError):
        ops.sample_tokens(x, u, top_k=u)
    with pytest.raises(TypeError):
        ops.sample_tokens(x.double(), u)
    with pytest.raises(TypeError):
        ops.sample_tokens(x, u.double())
    with pytest.raises(ValueError):
        ops.sample_tokens(x, u[:3])
    with pytest.raises(ValueError):
        ops.sample_tokens(x[:, :0], u)
    with pytest.raises(TypeError, match="at most"):
        ops.sample_tokens(torch.zeros(1, 385025, device=DEV), u[:1])
    with pytest.raises(ValueError, match="share memory"):
        both = torch.zeros(8, device=DEV)
        ops.sample_tokens(x, both[:4], out=both.view(torch.int64))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [1, 9, 10, 18, 19, 37])
def test_few_long_rows(n, kind):
    """Rows of eight, four and one CTA, of lengths that those do not divide, flat and peaked."""
    for vocab in (24000, 24001, 40007):
        x, u = rows(n, vocab, kind, n + vocab, spread=0.5 if vocab == 24001 else 2.0)
        check(x, u, temperature=0.9, top_p=0.95)
        check(x, u, top_k=60, top_p=0.9)
        check(x, u, min_p=0.02)
        check(x, u, temperature=0.0)


@pytest.mark.parametrize("top_p", [1e-6, 4e-5, 0.5, 0.99, 0.9999, 1 - 2.0 ** -24])
def test_window_of_top_p(top_p):
    """Shares that end at, and next to, the histogram's own error; weights that all lie in a few
    bins, and ones that mostly lie below all of them."""
    for spread in (0.01, 1.0, 30.0):
        x, u = rows(4, 20011, "fp32", 3, spread)
        check(x, u, top_p=top_p)
        check(x, u, top_p=top_p, temperature=0.05)
