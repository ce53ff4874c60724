"""4-bit attention and products where sizes differ widely within one call, against
64-bit results.

Attention's bar is that of test_int4_gpu.py: half a step of the output's type and 2^-10
of sum p (s c + |m|), of which P s in fp16 takes 2^-11 and the fp32 scores and
exponentials 2^-12."""
import math

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from oracle.int4_ref import rows_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0, "a kernel flagged a device-side error"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def held_rows(g, lead, D, dtype):
    """Codes and numbers [..., 4] of rows of about unit spread."""
    codes = torch.randint(0, 256, (*lead, D // 2), dtype=torch.uint8, device=DEV, generator=g)
    s = torch.rand(*lead, 2, device=DEV, generator=g) * 0.2 + 0.2
    m = -7.5 * s * (torch.rand(*lead, 2, device=DEV, generator=g) * 0.4 + 0.8)
    return codes, torch.stack([s[..., 0], m[..., 0], s[..., 1], m[..., 1]], -1).to(dtype)


def check(q, kv, n, dims=slice(None)):
    B, H, D = q.shape
    out = ops.decode_attention_int4(q, kv, torch.full((B,), n, dtype=torch.int32, device=DEV))
    for b in range(B):
        G = H // kv.kv_heads
        k = rows_ref(kv.key_codes[b, :, :n], kv.key_scales[b, :, :n]).repeat_interleave(G, 0)
        v = rows_ref(kv.value_codes[b, :, :n], kv.value_scales[b, :, :n]).repeat_interleave(G, 0)
        a = rows_ref(kv.value_codes[b, :, :n], kv.value_scales[b, :, :n].abs()).repeat_interleave(G, 0)
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[b].double(), k) / math.sqrt(D), -1)
        want, size = (torch.einsum("hn,hnd->hd", p, t)[:, dims] for t in (v, a))
        far = (out[b].double()[:, dims] - want).abs()
        bar = want.abs() * (torch.finfo(q.dtype).eps / 2) + size * 2.0 ** -10 \
            + torch.finfo(q.dtype).tiny * 2.0 ** -8
        assert (far <= bar).all(), (b, (far / bar).max().item())


@pytest.mark.parametrize("G", [1, 4, 8])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype,grow", [(BF, 2.0 ** 20), (BF, 2.0 ** 26), (BF, 2.0 ** 34), (HF, 2.0 ** 10),
                                        (HF, 2.0 ** 24)])
def test_large_values_on_keys_without_weight(dtype, grow, D, G):
    """One key of each tile has much larger values and a score that leaves it nothing:
    the others keep all their bits."""
    g = gen(D + G)
    n, Hkv = 300, 2
    kc, ks = held_rows(g, (2, Hkv, n), D, dtype)
    vc, vs = held_rows(g, (2, Hkv, n), D, dtype)
    low = torch.arange(5, n, 29, device=DEV)
    # q's sum times a constant key: a score of -60, a weight of 1e-26
    q = torch.randn(2, Hkv * G, D, device=DEV, generator=g).abs().to(dtype)
    ks[:, :, low] = 0
    ks[:, :, low, 1::2] = -60.0 * math.sqrt(D) / float(q.double().sum(-1).min())
    if dtype == HF:  # the others' scales small, so that the ratio fits the type
        vs *= 2.0 ** -12
    vs[:, :, low] *= grow
    check(q, ops.Int4KV(kc, ks, vc, vs), n)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("spread", [1.0, 12.0])
def test_values_of_all_sizes_in_any_order(dtype, spread):
    """V rows from 2^-40 to 2^20 (fp16: 2^-14 to 2^4) side by side, scores near and far
    apart."""
    g = gen(3)
    n, D, Hkv, G = 1500, 128, 2, 4
    kc, ks = held_rows(g, (1, Hkv, n), D, dtype)
    vc, vs = held_rows(g, (1, Hkv, n), D, torch.float32)
    lo, hi = (-40, 20) if dtype == BF else (-12, 4)
    size = 2.0 ** (torch.rand(1, Hkv, n, 1, device=DEV, generator=g) * (hi - lo) + lo)
    q = (torch.randn(1, Hkv * G, D, device=DEV, generator=g) * spread).to(dtype)
    check(q, ops.Int4KV(kc, ks, vc, (vs * size).to(dtype)), n)


@pytest.mark.parametrize("value", [1e-30, 1.0, 1e18, -3e25, 2e38])
@pytest.mark.parametrize("n", [1, 33, 700])
def test_constant_values(value, n):
    """Rows whose halves are constants (scale 0): the output is the constant, however
    large."""
    g = gen(4)
    D = 64
    kc, ks = held_rows(g, (1, 1, n), D, BF)
    vc = torch.zeros(1, 1, n, D // 2, dtype=torch.uint8, device=DEV)
    vs = torch.zeros(1, 1, n, 4, dtype=BF, device=DEV)
    vs[..., 1::2] = value
    q = torch.randn(1, 4, D, device=DEV, generator=g).to(BF)
    check(q, ops.Int4KV(kc, ks, vc, vs), n)


@pytest.mark.parametrize("n", [1, 40, 900])
@pytest.mark.parametrize("score", [-3e29, -3e31, -2e36])
def test_scores_far_below_zero(score, n):
    """However low the scores are, the highest keys have all the weight: equal ones the
    mean of their values."""
    g = gen(5)
    D = 64
    kc, ks = held_rows(g, (1, 1, n), D, BF)
    vc, vs = held_rows(g, (1, 1, n), D, BF)
    q = torch.full((1, 2, D), 2.0 ** 50, dtype=BF, device=DEV)
    ks[..., 0::2] = 0
    ks[..., 1::2] = score / (2.0 ** 50 * math.sqrt(D))
    check(q, ops.Int4KV(kc, ks, vc, vs), n)


@pytest.mark.parametrize("dtype,n,Hkv,G,D", [(HF, 131072, 4, 2, 128), (HF, 60000, 2, 8, 64), (HF, 9000, 8, 1, 128),
                                             (BF, 3000000, 1, 2, 64), (BF, 600000, 1, 8, 32)])
def test_sums_over_long_sequences(dtype, n, Hkv, G, D):
    """Many keys average to little: errors of the sums that all lean one way would show.
    In the mean square, over all heads and dims: a rounding to e bits is off by
    2^-e / sqrt(3) of the value at the lower end of a binade, 0.736 of that over
    significands of equal weight in the logarithm (E 1/m^2 = 0.75 / (2 ln 2)); the output
    has one, and P s (11 bits) one that counts times c (bf16) or c - 8 (fp16, whose
    products take 8 of them out again).  A tenth more for the number of outputs."""
    g = gen(6)
    kc, ks = held_rows(g, (1, Hkv, n), D, dtype)
    vc, vs = held_rows(g, (1, Hkv, n), D, dtype)
    q = torch.randn(1, Hkv * G, D, device=DEV, generator=g).to(dtype)
    out = ops.decode_attention_int4(q, ops.Int4KV(kc, ks, vc, vs),
                                    torch.tensor([n], dtype=torch.int32, device=DEV)).double()
    half = torch.finfo(dtype).eps / 2 / math.sqrt(3)
    off, bar = 0.0, 0.0
    for h in range(Hkv):
        p = torch.softmax(q[0, h * G:(h + 1) * G].double() @ rows_ref(kc[0, h], ks[0, h]).T / math.sqrt(D), -1)
        v = rows_ref(vc[0, h], vs[0, h])
        want = p @ v
        taken = vs[0, h].clone()  # s (c - 8), or s c
        taken[:, 1::2] = -8 * taken[:, 0::2] if dtype == HF else 0
        rounded = p.square() @ rows_ref(vc[0, h], taken).square()
        off += (out[0, h * G:(h + 1) * G] - want).square().sum().item()
        bar += (want.square() * half ** 2 + rounded * (2.0 ** -11 / math.sqrt(3)) ** 2).sum().item()
    assert off <= (1.1 * 0.736) ** 2 * bar, math.sqrt(off / bar)
