"""4-bit KV cache and weights on the GPU against 64-bit oracles.

Bars, from arithmetic:
  append, read   bit-exact: the definition names every rounding;
  attention      half a step of the output's type, plus 2^-10 of sum p|v~| with
                 |v~| <= s c + |m|: P s enters the products in fp16 (2^-11), and
                 the fp32 scores and exponentials move p by less than 2^-12;
  linear         half a step of the output's type, plus the fp32 accumulation:
                 a group of 128 is 8 products that each round the accumulator
                 once (2^-23), of magnitude 143 s sum|x| for bf16 (codes enter as
                 128 + c) and as much again for the sum of x that takes the 128
                 out: 2 * 8 * 2^-23 * 143 < 2^-11 of s sum|x|; and 2^-19 of
                 |m| sum|x|.  Fewer than that for the operands without the 128.
                 Where the kernel for more tokens takes over (9 on weights above 72 *
                 2^20 values, 17 where blocks of 16 cost more), a weight enters as fp16,
                 off by 2^-11 |w| and 2^-15 of its row's largest s at most: `rounded`
                 adds that in full.  Without it (normal x and w, |w| about 4.6 s):
                 the roundings are independent, 2.7 s |x| 2^-11 sqrt(k) in the mean
                 square, and 5 of those are below the above from k = 384 on."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from llama_pure_compute_b200 import _lib, ops
from llama_pure_compute_b200.int4_linear import Int4Weight, int4_linear
from llama_pure_compute_b200.model import precompute_freqs_cis
from oracle.int4_ref import attention_ref, quantize_rows_ref, rows_ref, weight_ref
from oracle.ops_ref import rope_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    assert _lib.device_status() == 0, "a kernel flagged a device-side error"


def flagged():
    """Reads and clears the device status; true when a bounds check failed."""
    return _lib.device_status() == 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ragged_index(caps):
    base = [sum(caps[:i]) for i in range(len(caps))]
    return (torch.tensor(base, dtype=torch.int64, device=DEV),
            torch.tensor(caps, dtype=torch.int32, device=DEV), base)


def tables(D, n, dtype):
    cos, sin = precompute_freqs_cis(D, n, device=DEV)
    return cos.to(dtype), sin.to(dtype)


def filled(g, lead, D, dtype, scale=1.0):
    """Codes and numbers of quantised normal rows."""
    return [t.contiguous() for t in quantize_rows_ref(
        (torch.randn(*lead, D, device=DEV, generator=g) * scale).to(dtype))]


def make_cache(g, B, Hkv, cap, D, dtype, caps=None, v_scale=1.0):
    if caps is None:
        lead, idx = (B, Hkv, cap), ()
    else:
        base, c, _ = ragged_index(caps)
        lead, idx = (Hkv, sum(caps)), (base, c, cap)
    return ops.Int4KV(*filled(g, lead, D, dtype), *filled(g, lead, D, dtype, v_scale), *idx)


def held(kv, b, n, start=0):
    """K, V values [Hkv, n, D] of sequence b in 64 bits."""
    if kv.ragged:
        at = int(kv.seq_base[b]) + start
        pick = lambda t: t[:, at:at + n]  # noqa: E731
    else:
        pick = lambda t: t[b, :, start:start + n]  # noqa: E731
    return (rows_ref(pick(kv.key_codes), pick(kv.key_scales)),
            rows_ref(pick(kv.value_codes), pick(kv.value_scales)))


def check_attention(out, q, kv, lens, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q = q.reshape(out.shape[0], out.shape[1], -1)
    o = out.reshape(q.shape)
    half = torch.finfo(out.dtype).eps / 2
    for b, n in enumerate(lens):
        k, v = held(kv, b, n)
        want, size = attention_ref(q[b], k, v, scale)
        if n:
            # |v~|: minimum and code part do not cancel in the bound
            pick = (lambda t: t[:, int(kv.seq_base[b]):int(kv.seq_base[b]) + n]) if kv.ragged \
                else (lambda t: t[b, :, :n])
            _, size = attention_ref(q[b], k, rows_ref(pick(kv.value_codes),
                                                      pick(kv.value_scales).abs()), scale)
        far = (o[b].double() - want).abs()
        bar = want.abs() * half + size * 2.0 ** -10 + torch.finfo(out.dtype).tiny * 2.0 ** -8
        assert (far <= bar).all(), (b, n, (far / bar).max().item())


# ---------------------------------------------------------------------------
# append, read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 128), (8, 2, 128), (6, 3, 64), (5, 5, 32), (1, 1, 64),
                                     (40, 40, 128)])
@pytest.mark.parametrize("layout", ["dense", "ragged"])
def test_append_is_bit_exact(dtype, H, Hkv, D, layout):
    g = gen(H * 100 + D)
    B, S, caps = 3, 5, [40, 7, 33]
    kv = make_cache(g, B, Hkv, 40, D, dtype, caps if layout == "ragged" else None)
    before = [t.clone() for t in (kv.key_codes, kv.key_scales, kv.value_codes, kv.value_scales)]
    qkv = torch.randn(B, S, (H + 2 * Hkv) * D, device=DEV, generator=g).to(dtype)
    pos = torch.tensor([[0, 1, 2, 3, 4], [6, 5, 2, 0, 1], [30, 31, -1, 32, 7]], device=DEV)
    for wide in (False, True):
        cos, sin = tables(D, 64, torch.float32 if wide else dtype)
        q = ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, H)
        x = qkv.view(B, S, H + 2 * Hkv, D).cpu()
        at = pos.clamp(min=0).cpu()
        qr, kr = rope_ref(x[:, :, :H], x[:, :, H:H + Hkv], cos.cpu()[at][:, :, None],
                          sin.cpu()[at][:, :, None], table_mode=1)
        live = pos.cpu() >= 0
        want_q = torch.where(live[..., None, None], qr, torch.zeros_like(qr))
        assert torch.equal(q.cpu(), want_q.transpose(1, 2))
        want = [t.cpu().clone() for t in before]
        for i, rows in ((0, kr), (2, x[:, :, H + Hkv:])):
            c, n = quantize_rows_ref(rows)
            for b in range(B):
                for s in range(S):
                    p = int(pos[b, s])
                    if p < 0:
                        continue
                    row = sum(caps[:b]) + p
                    where = (slice(None), row) if layout == "ragged" else (b, slice(None), p)
                    want[i][where], want[i + 1][where] = c[b, s], n[b, s]
        for got, ref in zip((kv.key_codes, kv.key_scales, kv.value_codes, kv.value_scales), want):
            assert torch.equal(got.cpu(), ref)  # rows that no token names included


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_of_special_values(dtype):
    """Constant and zero halves, NaN and infinities, halves whose scale is
    subnormal, zero after rounding, or overflows: as the oracle defines them."""
    D, top = 64, torch.finfo(dtype).max
    g = gen(5)
    rows = torch.randn(12, D, device=DEV, generator=g).to(dtype)
    rows[0] = 0
    rows[1] = 3.25
    rows[2, 5] = float("nan")
    rows[3, 40] = float("inf")
    rows[4, 3] = -float("inf")
    rows[5, 2], rows[5, 3] = top, -top
    rows[6] = (torch.randn(D, device=DEV, generator=g) * torch.finfo(dtype).tiny).to(dtype)
    rows[7] = (torch.randn(D, device=DEV, generator=g) * torch.finfo(dtype).tiny * 2.0 ** -7).to(dtype)
    rows[8] = (torch.randn(D, device=DEV, generator=g) * 1e4).to(dtype)
    rows[9, 1:32] = 1.0
    qkv = torch.zeros(1, 12, 3 * D, dtype=dtype, device=DEV)
    qkv[0, :, 2 * D:] = rows
    kv = make_cache(g, 1, 1, 12, D, dtype)
    cos, sin = tables(D, 12, dtype)
    pos = torch.arange(12, device=DEV)[None]
    ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, 1)
    c, n = quantize_rows_ref(rows.cpu())
    assert torch.equal(kv.value_codes[0, 0].cpu(), c)
    assert torch.equal(torch.nan_to_num(kv.value_scales[0, 0].cpu(), nan=-77.0),
                       torch.nan_to_num(n, nan=-77.0))
    _, v = ops.kv_read_int4(kv, pos)
    want = (rows_ref(c, n)).float().to(dtype)
    assert torch.equal(torch.nan_to_num(v[0, 0].cpu(), nan=-77.0, posinf=-78.0, neginf=-79.0),
                       torch.nan_to_num(want, nan=-77.0, posinf=-78.0, neginf=-79.0))
    for bad in (2, 4):
        assert v[0, 0, bad, :32].isnan().all() and not v[0, 0, bad, 32:].isnan().any()


@pytest.mark.parametrize("layout", ["dense", "ragged"])
def test_positions_outside_are_skipped_and_flagged(layout):
    g = gen(6)
    H, D, caps = 2, 64, [9, 4]
    kv = make_cache(g, 2, 2, 9, D, BF, caps if layout == "ragged" else None)
    before = [t.clone() for t in (kv.key_codes, kv.key_scales, kv.value_codes, kv.value_scales)]
    qkv = torch.randn(2, 1, 6 * D, device=DEV, generator=g).to(BF)
    cos, sin = tables(D, 9, BF)
    past = 4 if layout == "ragged" else 9
    q = ops.rope_kv_append_int4(qkv, torch.tensor([[-1], [past]], device=DEV), cos, sin, kv, H)
    assert flagged() and (q == 0).all()
    for t, b in zip((kv.key_codes, kv.key_scales, kv.value_codes, kv.value_scales), before):
        assert torch.equal(t, b)
    # tables shorter than the cache
    q = ops.rope_kv_append_int4(qkv, torch.tensor([[3], [3]], device=DEV), cos[:3], sin[:3], kv, H)
    assert flagged() and (q == 0).all() and torch.equal(kv.key_codes, before[0])
    k, v = ops.kv_read_int4(kv, torch.tensor([[-1, 2], [past, 0]], device=DEV))
    assert flagged()
    assert (k[:, :, 0] == 0).all() and (v[:, :, 0] == 0).all()
    assert (k[0, :, 1] != 0).any() and (k[1, :, 1] != 0).any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("layout,S", [("dense", 1), ("dense", 77), ("ragged", 300)])
def test_read_is_bit_exact(dtype, D, layout, S):
    g = gen(D + S)
    Hkv, caps = 3, [S + 3, S, S + 11]
    kv = make_cache(g, 3, Hkv, max(caps), D, dtype, caps if layout == "ragged" else None)
    pos = torch.stack([torch.randperm(S, device=DEV, generator=g) for _ in range(3)])
    k, v = ops.kv_read_int4(kv, pos)
    for b in range(3):
        rk, rv = held(kv, b, S)
        # c * s is exact in fp32, so fp32 then T is what one fp32 FMA then T gives
        assert torch.equal(k[b], rk.float().to(dtype)[:, pos[b]])
        assert torch.equal(v[b], rv.float().to(dtype)[:, pos[b]])


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("G", [1, 2, 3, 8, 12, 16])
def test_attention_heads_types_and_lengths(dtype, D, G):
    g = gen(D * G)
    Hkv, cap = 2, 700
    lens = [0, 1, 2, 15, 16, 31, 32, 33, 127, 128, 129, 255, 257, 640, 699, 700]
    kv = make_cache(g, len(lens), Hkv, cap, D, dtype)
    q = torch.randn(len(lens), Hkv * G, D, device=DEV, generator=g).to(dtype)
    out = ops.decode_attention_int4(q, kv, torch.tensor(lens, dtype=torch.int32, device=DEV))
    check_attention(out, q, kv, lens)


@pytest.mark.parametrize("dtype,D,G", [(BF, 128, 1), (HF, 64, 4), (BF, 32, 8)])
def test_attention_ragged_bit_identical_to_dense(dtype, D, G):
    g = gen(D + G)
    Hkv, caps = 3, [301, 1, 1030, 64, 513]
    lens = [257, 1, 1030, 0, 500]
    cap = max(caps)
    dense = make_cache(g, 5, Hkv, cap, D, dtype)
    base, c, at = ragged_index(caps)
    flat = [torch.cat([t[b, :, :n] for b, n in enumerate(caps)], 1).contiguous()
            for t in (dense.key_codes, dense.key_scales, dense.value_codes, dense.value_scales)]
    rag = ops.Int4KV(*flat, base, c, cap)
    q = torch.randn(5, Hkv * G, D, device=DEV, generator=g).to(dtype)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    a, b = ops.decode_attention_int4(q, dense, ln), ops.decode_attention_int4(q, rag, ln)
    assert torch.equal(a, b)
    check_attention(b, q, rag, lens)


@pytest.mark.parametrize("B,Hkv,G,cap,lens", [
    (1, 8, 4, 20000, [19999]), (1, 32, 1, 1064, [1000]), (2, 1, 8, 40000, [40000, 1]),
    (64, 8, 1, 300, [5 * i for i in range(60)] + [300] * 4), (33, 32, 1, 1500, [1500 - 40 * i for i in range(33)])])
def test_attention_split_lengths(B, Hkv, G, cap, lens):
    """Sizes on each side of the split rule."""
    g = gen(cap)
    kv = make_cache(g, B, Hkv, cap, 128, BF)
    q = torch.randn(B, Hkv * G, 128, device=DEV, generator=g).to(BF)
    out = ops.decode_attention_int4(q, kv, torch.tensor(lens, dtype=torch.int32, device=DEV))
    check_attention(out, q, kv, lens)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("v_scale", [1e-4, 3e3])
@pytest.mark.parametrize("q_scale", [1e-5, 1.0, 30.0])
def test_attention_magnitudes(dtype, v_scale, q_scale):
    """Values and queries far from 1, and scores that leave one key all the
    weight: the running reference and q's power of two follow."""
    g = gen(9)
    lens = [513, 40]
    kv = make_cache(g, 2, 2, 600, 128, dtype, v_scale=v_scale)
    q = (torch.randn(2, 4, 128, device=DEV, generator=g) * q_scale).to(dtype)
    out = ops.decode_attention_int4(q, kv, torch.tensor(lens, dtype=torch.int32, device=DEV))
    check_attention(out, q, kv, lens)


def test_attention_values_that_grow_along_the_sequence():
    """V scales from 2^-40 to 2^20 in one sequence, the heaviest keys among the
    smallest and among the largest values."""
    g = gen(10)
    n, D = 2000, 64
    x = torch.randn(1, 1, n, D, device=DEV, generator=g)
    grow = 2.0 ** torch.linspace(-40, 20, n, device=DEV)[None, None, :, None]
    q = torch.randn(1, 1, D, device=DEV, generator=g).to(BF)
    for order in (grow, grow.flip(2)):
        kv = ops.Int4KV(*filled(g, (1, 1, n), D, BF),
                        *[t.contiguous() for t in quantize_rows_ref((x * order).to(BF))])
        out = ops.decode_attention_int4(q, kv, torch.tensor([n], dtype=torch.int32, device=DEV))
        check_attention(out, q, kv, [n])


def test_attention_ignores_what_lies_past_the_end():
    """NaN and infinite scales in rows past a sequence's end do not reach it;
    a NaN row inside reaches exactly the heads and dims that it should."""
    g = gen(11)
    lens = [37, 130, 0]
    kv = make_cache(g, 3, 2, 160, 128, BF)
    clean = ops.decode_attention_int4(q := torch.randn(3, 4, 128, device=DEV, generator=g).to(BF), kv,
                                      ln := torch.tensor(lens, dtype=torch.int32, device=DEV))
    for b, n in enumerate(lens):
        kv.key_scales[b, :, n:] = float("nan")
        kv.value_scales[b, :, n:] = float("inf")
        kv.key_codes[b, :, n:] = 255
        kv.value_codes[b, :, n:] = 255
    assert torch.equal(ops.decode_attention_int4(q, kv, ln), clean)
    assert (clean[2] == 0).all()
    kv.value_scales[1, 1, 100, 2:] = float("nan")  # upper half of the dims, KV head 1
    out = ops.decode_attention_int4(q, kv, ln)
    assert out[1, 2:, 64:].isnan().all()
    assert torch.equal(out[1, :2], clean[1, :2]) and torch.equal(out[0], clean[0])
    want, size = attention_ref(q[1], held(kv, 1, 130)[0], torch.nan_to_num(held(kv, 1, 130)[1]), 128 ** -0.5)
    far = (out[1, 2:, :64].double() - want[2:, :64]).abs()
    assert (far <= want[2:, :64].abs() * 2.0 ** -9 + size[2:, :64] * 2.0 ** -8).all()
    kv.key_scales[0, 0, 3, :2] = float("nan")
    out = ops.decode_attention_int4(q, kv, ln)
    assert out[0, :2].isnan().all() and torch.equal(out[0, 2:], clean[0, 2:])


@pytest.mark.parametrize("layout", ["dense", "ragged"])
def test_attention_length_beyond_the_rows_is_cut_and_flagged(layout):
    g = gen(12)
    caps = [50, 20]
    kv = make_cache(g, 2, 2, 50, 64, BF, caps if layout == "ragged" else None)
    q = torch.randn(2, 2, 64, device=DEV, generator=g).to(BF)
    cut = [50, 20] if layout == "ragged" else [50, 50]
    long = torch.tensor([51, 60], dtype=torch.int32, device=DEV)
    out = ops.decode_attention_int4(q, kv, long)
    assert flagged()
    check_attention(out, q, kv, cut)
    out = ops.decode_attention_int4(q, kv, torch.tensor([-3, 7], dtype=torch.int32, device=DEV))
    check_attention(out, q, kv, [0, 7])


def test_ragged_rows_outside_the_buffer_are_flagged():
    g = gen(13)
    kv = make_cache(g, 2, 1, 30, 64, BF, [30, 20])
    q = torch.randn(2, 1, 64, device=DEV, generator=g).to(BF)
    ln = torch.tensor([10, 10], dtype=torch.int32, device=DEV)
    one = ops.decode_attention_int4(q, kv, ln)
    for base, cap in (([0, 31], [30, 20]), ([0, -1], [30, 20]), ([0, 30], [30, 31]), ([0, 30], [30, -4])):
        bad = kv.select(torch.tensor(base, dtype=torch.int64, device=DEV),
                        torch.tensor(cap, dtype=torch.int32, device=DEV))
        out = ops.decode_attention_int4(q, bad, ln)
        assert flagged() and torch.equal(out[0], one[0]) and (out[1] == 0).all()
        k, _ = ops.kv_read_int4(bad, torch.zeros(2, 1, dtype=torch.int64, device=DEV))
        assert flagged() and (k[1] == 0).all()


def test_offsets_past_32_bits():
    """Caches whose code bytes, rows times heads, pass 2^32."""
    g = gen(14)
    cap, Hkv, D = 65535 * 128, 9, 128
    kv = ops.Int4KV.empty(1, Hkv, cap, D, BF, DEV)
    assert kv.key_codes.numel() > 2 ** 32
    S = 300
    qkv = torch.randn(1, S, 3 * Hkv * D, device=DEV, generator=g).to(BF)
    cos, sin = tables(D, S, BF)
    pos = torch.arange(S, device=DEV)[None]
    ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, Hkv)
    c, n = quantize_rows_ref(qkv.view(1, S, 3 * Hkv, D)[:, :, 2 * Hkv:])
    assert torch.equal(kv.value_codes[0, :, :S], c[0].transpose(0, 1))
    assert torch.equal(kv.value_scales[0, :, :S], n[0].transpose(0, 1))
    q = torch.randn(1, Hkv, D, device=DEV, generator=g).to(BF)
    out = ops.decode_attention_int4(q, kv, torch.tensor([S], dtype=torch.int32, device=DEV))
    check_attention(out, q, kv, [S])
    far = torch.tensor([[cap - 1]], device=DEV)
    for t in (kv.key_codes, kv.key_scales, kv.value_codes, kv.value_scales):
        t[:, :, cap - 1] = t[:, :, 5]
    k5, v5 = ops.kv_read_int4(kv, torch.tensor([[5]], device=DEV))
    k, v = ops.kv_read_int4(kv, far)
    assert torch.equal(k, k5) and torch.equal(v, v5)


def test_attention_layouts_streams_and_repeats():
    """A strided query, a 4-D one, given outputs, another stream; the same call
    twice gives the same bits."""
    g = gen(15)
    lens = [900, 33, 512]
    kv = make_cache(g, 3, 4, 900, 128, BF)
    wide = torch.randn(3, 8, 256, device=DEV, generator=g).to(BF)
    q = wide[..., 64:192]
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = ops.decode_attention_int4(q, kv, ln, sm_scale=0.2)
    check_attention(out, q.contiguous(), kv, lens, 0.2)
    q4 = q.contiguous().view(3, 8, 1, 128)
    given = torch.full_like(q4, float("nan"))
    ws = ops.decode_attention_int4_workspace(kv, 3, 8)
    assert ops.decode_attention_int4(q4, kv, ln, 0.2, out=given, workspace=ws) is given
    assert torch.equal(given.view_as(out), out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.decode_attention_int4(q, kv, ln, sm_scale=0.2)
    s.synchronize()
    assert torch.equal(other, out)


@pytest.mark.parametrize("B,Hkv,G,cap,lens", [
    (1, 8, 4, 20000, [19999]), (1, 32, 1, 1064, [1000]), (3, 2, 8, 5000, [5000, 1, 0]),
    (64, 8, 1, 300, [5 * i for i in range(60)] + [300] * 4)])
def test_attention_into_its_query(B, Hkv, G, cap, lens):
    """out may be q: every split has read its queries when the first output is written."""
    g = gen(cap + 1)
    kv = make_cache(g, B, Hkv, cap, 128, BF)
    q = torch.randn(B, Hkv * G, 128, device=DEV, generator=g).to(BF)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = ops.decode_attention_int4(q, kv, ln)
    ops.decode_attention_int4(q, kv, ln, out=q)
    assert torch.equal(q, want)


def test_two_graphs_with_workspaces_of_their_own():
    g = gen(16)
    kv = make_cache(g, 2, 4, 1500, 128, BF)
    qs = [torch.randn(2, 4, 128, device=DEV, generator=g).to(BF) for _ in range(2)]
    lens = [torch.tensor(n, dtype=torch.int32, device=DEV) for n in ([1500, 700], [3, 1400])]
    eager = [ops.decode_attention_int4(q, kv, n) for q, n in zip(qs, lens)]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for q, n in zip(qs, lens):
        ws = ops.decode_attention_int4_workspace(kv, 2, 4)
        out = torch.empty_like(q)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.decode_attention_int4(q, kv, n, out=out, workspace=ws)
        graphs.append((gr, ws))
        outs.append(out)
    for _ in range(5):
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, eager):
        assert torch.equal(a, b)
    # the graph reads lengths on the device
    lens[0].copy_(lens[1])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    check_attention(outs[0], qs[0], kv, [3, 1400])


def test_prefill_decode_and_read_together():
    """A prompt in two chunks, then decode steps, as a model drives them: every
    step's attention against 64-bit attention over what the cache then holds."""
    g = gen(17)
    B, H, Hkv, D, cap = 2, 8, 2, 64, 90
    kv = ops.Int4KV.empty(B, Hkv, cap, D, BF, DEV)
    cos, sin = tables(D, cap, BF)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    done = 0
    for n in (40, 30):
        qkv = torch.randn(B, n, (H + 2 * Hkv) * D, device=DEV, generator=g).to(BF)
        pos = torch.arange(done, done + n, device=DEV)[None].expand(B, -1)
        ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, H)
        done += n
    k, v = ops.kv_read_int4(kv, torch.arange(done, device=DEV)[None].expand(B, -1))
    for b in range(B):
        rk, rv = held(kv, b, done)
        assert torch.equal(k[b].double(), rk.to(BF).double()) and torch.equal(v[b].double(), rv.to(BF).double())
    for step in range(12):
        qkv = torch.randn(B, 1, (H + 2 * Hkv) * D, device=DEV, generator=g).to(BF)
        pos = torch.full((B, 1), done, device=DEV)
        q = ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, H)
        done += 1
        lens.fill_(done)
        out = ops.decode_attention_int4(q.view(B, H, D), kv, lens)
        check_attention(out, q.view(B, H, D), kv, [done] * B)


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------
def random_weight(g, rows, k, group, dtype):
    return Int4Weight.quantize((torch.randn(rows, k, device=DEV, generator=g) * 0.02).to(dtype), group)


def linear_bar(x, codes, s, m, y):
    group = x.shape[1] // s.shape[1]
    ax = x.double().abs().view(x.shape[0], -1, group).sum(-1)
    return ax @ s.double().mT * 2.0 ** -11 + ax @ m.double().abs().mT * 2.0 ** -19


def check_linear(y, x, codes, s, m, epilogue="store", resid=None, rounded=False):
    z = x.double() @ weight_ref(codes, s, m).mT
    e = linear_bar(x, codes, s, m, z)
    if rounded:
        ax = x.double().abs()
        e = e + ax @ weight_ref(codes, s, m).abs().mT * 2.0 ** -11 \
            + ax.sum(-1, keepdim=True) * s.double().abs().amax(-1) * 2.0 ** -15
    if epilogue == "residual":
        z = z + resid.double()
    if epilogue == "swiglu":
        n = z.shape[1] // 2
        gt, up, eg, eu = z[:, :n], z[:, n:], e[:, :n], e[:, n:]
        silu = gt * torch.sigmoid(gt)
        z = silu * up
        # silu' <= 1.1; the exponential and the division are good to 2^-20
        e = 1.1 * eg * (up.abs() + eu) + (silu.abs() + 1.1 * eg) * eu + z.abs() * 2.0 ** -20
    bar = z.abs() * (torch.finfo(y.dtype).eps / 2) + e + torch.finfo(y.dtype).tiny
    far = (y.double() - z).abs()
    assert (far <= bar).all(), (far / bar).max().item()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,n,k", [(1, 1, 128), (1, 17, 1024), (3, 1000, 256), (8, 33, 2176),
                                        (9, 64, 128), (16, 15, 640), (17, 48, 4096), (33, 130, 384),
                                        (64, 1003, 1152)])
def test_linear(dtype, group, tokens, n, k):
    g = gen(tokens * n + k)
    codes, s, m = random_weight(g, n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    check_linear(int4_linear(x, w), x, codes, s, m)
    r = torch.randn(tokens, n, device=DEV, generator=g).to(dtype)
    y = int4_linear(x, w, "residual", resid=r)
    check_linear(y, x, codes, s, m, "residual", r)
    assert torch.equal(int4_linear(x, w, "residual", resid=r, out=r), y) and torch.equal(r, y)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,n,k", [(1, 16, 128), (4, 1001, 512), (12, 40, 256), (25, 7, 1024),
                                        (64, 33, 384)])
def test_linear_swiglu(dtype, group, tokens, n, k):
    g = gen(tokens + n + k)
    codes, s, m = random_weight(g, 2 * n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group, layout="swiglu")
    x = (torch.randn(tokens, k, device=DEV, generator=g) * 3).to(dtype)
    check_linear(int4_linear(x, w, "swiglu"), x, codes, s, m, "swiglu")


@pytest.mark.parametrize("k,group", [(64, 64), (64, 32), (192, 64), (448, 32), (11008, 128)])
def test_linear_short_and_uneven_k(k, group):
    """Fewer column groups than warps, and a count that does not divide by them."""
    g = gen(k)
    codes, s, m = random_weight(g, 100, k, group, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=group)
    for tokens in (1, 11, 30):
        x = torch.randn(tokens, k, device=DEV, generator=g).to(BF)
        check_linear(int4_linear(x, w), x, codes, s, m)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_many_rows(dtype):
    """More tile rows than CTAs run at once."""
    g = gen(3)
    codes, s, m = random_weight(g, 20011, 512, 128, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    for tokens in (1, 10, 20):
        x = torch.randn(tokens, 512, device=DEV, generator=g).to(dtype)
        check_linear(int4_linear(x, w), x, codes, s, m)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n", [48, 37008])
def test_linear_code_by_code(dtype, n):
    """One-hot x reads single weights: every code of every column in its place."""
    g = gen(4)
    k = 128
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    s = torch.ones(n, 1, dtype=dtype, device=DEV)
    m = torch.zeros(n, 1, dtype=dtype, device=DEV)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    want = weight_ref(codes, s, m).to(dtype)
    assert torch.equal(w.dequantize(), want)
    eye = torch.eye(k, dtype=dtype, device=DEV)
    for at in (0, 64):
        assert torch.equal(int4_linear(eye[at:at + 64], w), want.t()[at:at + 64])


@pytest.mark.parametrize("n", [65, 27000])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_values(dtype, n):
    """Offset activations (large sums of x), large and small ones; a non-finite
    token stays in its row."""
    g = gen(7)
    codes, s, m = random_weight(g, n, 1024, 128, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    x = torch.randn(6, 1024, device=DEV, generator=g)
    x[1] += 4.0
    x[2] *= 100
    x[3] *= 1e-4
    x[4, 7] = 900.0
    x[5] = 0
    x = x.to(dtype)
    y = int4_linear(x, w)
    check_linear(y, x, codes, s, m)
    assert (y[5] == 0).all()
    x[1, 3], x[4, 1000] = float("nan"), float("inf")
    z = int4_linear(x, w)
    keep = [0, 2, 3, 5]
    assert torch.equal(z[keep], y[keep])
    assert not z[1].isfinite().any() and not z[4].isfinite().any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 8])
def test_linear_items_that_share_their_sums(dtype, group, tokens):
    """Few tokens on larger weights add up several items' sums at once: full and
    broken batches, the last item past the rows; twice the same."""
    g = gen(tokens)
    for n, k, epilogue in ((20011, 1792, "store"), (9999, 1792, "swiglu"), (8209, 4096, "residual")):
        codes, s, m = random_weight(g, 2 * n if epilogue == "swiglu" else n, k, group, dtype)
        w = Int4Weight.from_codes(codes, s, m, group_size=group,
                                  layout="swiglu" if epilogue == "swiglu" else "linear")
        x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
        r = torch.randn(tokens, n, device=DEV, generator=g).to(dtype) if epilogue == "residual" else None
        y = int4_linear(x, w, epilogue, resid=r)
        check_linear(y, x, codes, s, m, epilogue, r)
        assert torch.equal(int4_linear(x, w, epilogue, resid=r), y)
        if r is not None:
            assert torch.equal(int4_linear(x, w, epilogue, resid=r, out=r), y)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,k,group", [
    (1, 4160, 64), (8, 4096, 128), (3, 5504, 128), (4, 11008, 128), (1, 17408, 128), (2, 18432, 128),
    # as much of x as fits beside the weight ring, and the next width
    (2, 26624, 64), (2, 24576, 64), (1, 49152, 32), (1, 47104, 32), (8, 5120, 128), (7, 5120, 128)])
def test_linear_widths_of_x(dtype, tokens, k, group):
    """x of 256, 1024 and more columns a warp, up to where it fits no longer."""
    g = gen(k + tokens)
    n = ((8 + 3 * tokens) << 20) // k + 17  # the least weight whose x is kept
    codes, s, m = random_weight(g, n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    check_linear(int4_linear(x, w), x, codes, s, m)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,n,k,group,epilogue", [
    (8, 200, 16384, 128, "store"), (5, 40, 32768, 64, "residual"), (8, 2400, 11008, 128, "store"),
    (9, 5000, 640, 32, "store"), (16, 5000, 640, 64, "residual"), (13, 2500, 512, 128, "swiglu"),
    (16, 100, 16384, 32, "swiglu"), (16, 4800, 8192, 32, "store"),
    # blocks of 16 tokens
    (17, 1, 64, 32, "store"), (32, 129, 192, 64, "residual"), (33, 63, 256, 128, "swiglu"),
    (64, 65, 4096, 128, "swiglu"), (48, 3000, 128, 32, "residual"), (20, 5000, 320, 32, "swiglu"),
    (64, 4096, 1024, 128, "store")])
def test_linear_x_from_the_caches(dtype, tokens, n, k, group, epilogue):
    """x not kept in shared memory: with and without kept sums of x, 8 and 16 warps,
    one and two tile rows, one to four blocks of tokens."""
    g = gen(tokens + n)
    codes, s, m = random_weight(g, 2 * n if epilogue == "swiglu" else n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group,
                              layout="swiglu" if epilogue == "swiglu" else "linear")
    assert w.workspace_bytes(tokens) == 0
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    r = torch.randn(tokens, n, device=DEV, generator=g).to(dtype) if epilogue == "residual" else None
    y = int4_linear(x, w, epilogue, resid=r)
    check_linear(y, x, codes, s, m, epilogue, r)
    if r is not None:
        assert torch.equal(int4_linear(x, w, epilogue, resid=r, out=r), y) and torch.equal(r, y)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,n,k,group,epilogue", [
    (17, 1225, 16384, 128, "store"), (32, 301, 65536, 64, "residual"), (33, 601, 8192, 128, "swiglu"),
    (64, 65, 65536, 128, "swiglu"), (48, 3000, 4096, 32, "residual"), (64, 40000, 128, 128, "store"),
    (20, 12000, 1088, 32, "swiglu")])
def test_linear_many_tokens(dtype, tokens, n, k, group, epilogue):
    """17 to 64 tokens, larger weights: columns split over clusters or not, ragged
    last tiles."""
    g = gen(tokens + n)
    codes, s, m = random_weight(g, 2 * n if epilogue == "swiglu" else n, k, group, dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=group,
                              layout="swiglu" if epilogue == "swiglu" else "linear")
    assert (w.workspace_bytes(tokens) > 0) == (dtype == BF)
    x = torch.randn(tokens, k, device=DEV, generator=g).to(dtype)
    r = torch.randn(tokens, n, device=DEV, generator=g).to(dtype) if epilogue == "residual" else None
    y = int4_linear(x, w, epilogue, resid=r)
    check_linear(y, x, codes, s, m, epilogue, r, rounded=True)
    if r is not None:
        assert torch.equal(int4_linear(x, w, epilogue, resid=r, out=r), y) and torch.equal(r, y)


@pytest.mark.parametrize("tokens", [9, 16])
def test_linear_of_a_large_weight(tokens):
    """The same from 9 tokens on where the weight has more than 72 * 2^20 values."""
    g = gen(tokens)
    codes, s, m = random_weight(g, 19000, 4096, 128, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    assert w.workspace_bytes(tokens) > 0
    x = torch.randn(tokens, 4096, device=DEV, generator=g).to(BF)
    check_linear(int4_linear(x, w), x, codes, s, m, rounded=True)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_many_tokens_values(dtype):
    """Groups of very different scale in a row, negative scales, rows of zeros, x of
    very different sizes; a non-finite token stays in its row."""
    g = gen(21)
    n, k = 16403, 512
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV, generator=g)
    s = (torch.rand(n, 4, device=DEV, generator=g) + 0.5) * torch.tensor([1e-2, 1e-4, -3e-3, 1.0], device=DEV)
    m = torch.randn(n, 4, device=DEV, generator=g) * torch.tensor([0.1, 1e-3, 1e-2, 8.0], device=DEV)
    s[5], m[5] = 0, 0
    s[6] = 0
    s, m = s.to(dtype), m.to(dtype)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    x = torch.randn(40, k, device=DEV, generator=g)
    x[1] *= 30
    x[2] *= 1e-4
    x[3] = 0
    x[4, 7] = 900.0
    x = x.to(dtype)
    y = int4_linear(x, w)
    z = x.double() @ weight_ref(codes, s, m).mT
    ax = x.double().abs()
    e = linear_bar(x, codes, s.abs(), m, z) + ax @ weight_ref(codes, s, m).abs().mT * 2.0 ** -11 \
        + ax.sum(-1, keepdim=True) * s.double().abs().amax(-1) * 2.0 ** -15
    far = (y.double() - z).abs()
    bar = z.abs() * (torch.finfo(dtype).eps / 2) + e + torch.finfo(dtype).tiny
    assert (far <= bar).all(), (far / bar).max().item()
    assert (y[3] == 0).all() and (y[:, 5] == 0).all()
    x[1, 3], x[39, 500] = float("nan"), float("inf")
    z = int4_linear(x, w)
    keep = [i for i in range(40) if i not in (1, 39)]
    assert torch.equal(z[keep], y[keep])
    assert not z[1].isfinite().any() and not z[39].isfinite().any()


def test_linear_many_tokens_in_graphs_and_streams():
    """Two graphs and two streams at once, each call with scratch of its own."""
    g = gen(22)
    codes, s, m = random_weight(g, 5120, 5120, 128, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    assert w.workspace_bytes(24) > 0
    xs = [torch.randn(t, 5120, device=DEV, generator=g).to(BF) for t in (24, 64)]
    nw = torch.ones(5120, dtype=BF, device=DEV)
    want = [int4_linear(int4_linear(ops.rmsnorm_forward(x, nw), w), w) for x in xs]
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(int4_linear(int4_linear(ops.rmsnorm_forward(x, nw), w), w))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    eager = []
    for _ in range(10):
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                eager.append(int4_linear(int4_linear(ops.rmsnorm_forward(x, nw), w), w))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(eager))


FIRST_CALLS_IN_A_GRAPH = """
import torch
from llama_pure_compute_b200 import _lib, ops
from llama_pure_compute_b200.int4_linear import Int4Weight, int4_linear
g = torch.Generator(device="cuda").manual_seed(1)
def rnd(*s):
    return torch.randn(*s, device="cuda", generator=g).bfloat16()
ws = [Int4Weight(rnd(n, 4096)) for n in (8192, 1024)]
xs = [rnd(t, 4096) for t in (1, 2, 8, 16, 33, 64)]
kv = ops.Int4KV.empty(4, 8, 700, 128)
for t in (kv.key_codes, kv.value_codes):
    t.random_(0, 255)
for t in (kv.key_scales, kv.value_scales):
    t.normal_()
q, qkv = rnd(4, 32, 128), rnd(4, 1, 48 * 128)
lens = torch.tensor([700, 1, 0, 350], dtype=torch.int32, device="cuda")
pos = torch.tensor([[699], [0], [5], [349]], device="cuda")
cos, sin = torch.ones(700, 128, device="cuda").bfloat16(), torch.zeros(700, 128, device="cuda").bfloat16()
def all_of_them():
    y = [int4_linear(x, w) for w in ws for x in xs]
    y.append(ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, 32))
    y.append(ops.decode_attention_int4(q, kv, lens))
    return y + list(ops.kv_read_int4(kv, pos))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = all_of_them()
for _ in range(3):
    graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, all_of_them())) and _lib.device_status() == 0
"""


def test_first_calls_of_a_process_are_captured():
    """No entry point needs a call outside a graph before one inside."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_GRAPH], cwd=Path(__file__).parents[1],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_from_several_threads():
    """Each thread on a stream of its own, sizes in another order."""
    g = gen(24)
    weights = []
    for n in (8192, 1024):
        codes, s, m = random_weight(g, n, 4096, 128, BF)
        weights.append(Int4Weight.from_codes(codes, s, m, group_size=128))
    xs = [torch.randn(t, 4096, device=DEV, generator=g).to(BF) for t in (1, 2, 8, 16, 33, 64)]
    kv = make_cache(g, 4, 8, 700, 128, BF)
    q = torch.randn(4, 32, 128, device=DEV, generator=g).to(BF)
    lens = torch.tensor([700, 1, 0, 350], dtype=torch.int32, device=DEV)
    want = [[int4_linear(x, w) for x in xs] for w in weights]
    att = ops.decode_attention_int4(q, kv, lens)
    torch.cuda.synchronize()
    wrong = []

    def work(start):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(start, start + 30):
                    got = [int4_linear(xs[i % 6], w) for w in weights]
                    out = ops.decode_attention_int4(q, kv, lens)
                    torch.cuda.current_stream().synchronize()
                    if not (torch.equal(out, att) and all(torch.equal(y, r[i % 6]) for y, r in zip(got, want))):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_views_off_the_16_byte_grid():
    """Inputs that start in the middle of 16 bytes give what their copies give."""
    g = gen(23)
    codes, s, m = random_weight(g, 128, 128, 64, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=64)
    for tokens in (1, 12, 30):
        x = torch.randn(tokens * 128 + 1, device=DEV, generator=g).to(BF)[1:].view(tokens, 128)
        assert torch.equal(int4_linear(x, w), int4_linear(x.clone(), w))
    kv = make_cache(g, 2, 2, 40, 32, BF)
    q = torch.randn(2 * 4 * 32 + 3, device=DEV, generator=g).to(BF)[3:].view(2, 4, 32)
    ln = torch.tensor([40, 7], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.decode_attention_int4(q, kv, ln), ops.decode_attention_int4(q.clone(), kv, ln))
    qkv = torch.randn(2 * 8 * 32 + 1, device=DEV, generator=g).to(BF)[1:].view(2, 1, 256)
    pos = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    cos, sin = tables(32, 8, BF)
    assert torch.equal(ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, 4),
                       ops.rope_kv_append_int4(qkv.clone(), pos, cos, sin, kv, 4))


def test_weight_from_16_bits_and_back():
    g = gen(8)
    gate = (torch.randn(70, 256, device=DEV, generator=g) * 0.02).to(BF)
    up = (torch.randn(70, 256, device=DEV, generator=g) * 0.02).to(BF)
    for group in (32, 64, 128):
        w = Int4Weight(gate, group_size=group)
        codes, s, m = Int4Weight.quantize(gate, group)
        assert torch.equal(w.dequantize(), weight_ref(codes, s, m).float().to(BF))
        step = s.double().repeat_interleave(group, 1)
        assert ((w.dequantize().double() - gate.double()).abs()
                <= step * (0.5 + 15 * 2.0 ** -8) + gate.double().abs() * 2.0 ** -8).all()
        pair = Int4Weight(gate, up, layout="swiglu", group_size=group)
        fused = Int4Weight(torch.cat([gate, up]), layout="swiglu", group_size=group)
        assert torch.equal(pair.data, fused.data)
        assert torch.equal(pair.dequantize(), fused.dequantize())
        x = torch.randn(3, 256, device=DEV, generator=g).to(BF)
        both = torch.cat([gate, up])
        check_linear(int4_linear(x, pair, "swiglu"), x, *Int4Weight.quantize(both, group), "swiglu")
        odd = both.t().contiguous().t()  # a strided source
        assert torch.equal(Int4Weight(odd, layout="swiglu", group_size=group).data, pair.data)


@pytest.mark.parametrize("n", [512, 8192])
def test_linear_after_a_kernel_that_writes_x_in_graphs_and_streams(n):
    """Launched programmatically under the kernel before it: x, written by that
    kernel, is not read early; the same in a graph and on another stream."""
    g = gen(18)
    codes, s, m = random_weight(g, n, 4096, 128, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    src = torch.randn(4, 4096, device=DEV, generator=g).to(BF)
    nw = torch.ones(4096, dtype=BF, device=DEV)
    want = int4_linear(ops.rmsnorm_forward(src, nw), w)
    check_linear(want, ops.rmsnorm_forward(src, nw), codes, s, m)
    for _ in range(20):
        x = torch.full_like(src, float("nan"))
        x.copy_(src)
        assert torch.equal(int4_linear(ops.rmsnorm_forward(x, nw), w), want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = int4_linear(ops.rmsnorm_forward(src, nw), w)
        y2 = int4_linear(y.new_zeros(1, 4096) + y.view(-1)[:1], w)
    for _ in range(3):
        gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and y2.isfinite().all()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = int4_linear(ops.rmsnorm_forward(src, nw), w)
    st.synchronize()
    assert torch.equal(other, want)


# ---------------------------------------------------------------------------
# refusals of the Python layer
# ---------------------------------------------------------------------------
def test_refusals():
    g = gen(19)
    kv = make_cache(g, 2, 2, 16, 64, BF)
    q = torch.zeros(2, 4, 64, dtype=BF, device=DEV)
    ln = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = [
        (ValueError, lambda: ops.decode_attention_int4(q.cpu(), kv, ln)),
        (ValueError, lambda: ops.decode_attention_int4(q, kv, ln.cpu())),
        (TypeError, lambda: ops.decode_attention_int4(q, kv, ln.long())),
        (TypeError, lambda: ops.decode_attention_int4(q.half(), kv, ln)),
        (ValueError, lambda: ops.decode_attention_int4(q[:, :3], kv, ln)),
        (ValueError, lambda: ops.decode_attention_int4(q[..., :32], kv, ln)),
        (ValueError, lambda: ops.decode_attention_int4(q, kv, ln[:1])),
        (ValueError, lambda: ops.decode_attention_int4(q, kv, ln.repeat(2)[::2])),
        (ValueError, lambda: ops.decode_attention_int4(torch.cat([q, q]), kv, ln.repeat(2))),
        (ValueError, lambda: ops.decode_attention_int4(q, kv, ln, out=q.float())),
        (ValueError, lambda: ops.kv_read_int4(kv, ln)),
        (ValueError, lambda: ops.kv_read_int4(kv, torch.zeros(3, 1, dtype=torch.int64, device=DEV))),
        (TypeError, lambda: ops.kv_read_int4(kv, torch.zeros(2, 1, device=DEV))),
        (ValueError, lambda: ops.Int4KV(kv.key_codes, kv.key_scales[:1], kv.value_codes, kv.value_scales)),
        (ValueError, lambda: ops.Int4KV(kv.key_codes.transpose(1, 2), kv.key_scales, kv.value_codes,
                                        kv.value_scales)),
        (TypeError, lambda: ops.Int4KV(kv.key_codes, kv.key_scales.float(), kv.value_codes, kv.value_scales)),
        (TypeError, lambda: ops.Int4KV(kv.key_codes.char(), kv.key_scales, kv.value_codes, kv.value_scales)),
        (ValueError, lambda: ops.Int4KV(kv.key_codes[0], kv.key_scales[0], kv.value_codes[0],
                                        kv.value_scales[0], seq_base=torch.zeros(1, dtype=torch.int64, device=DEV))),
        (ValueError, lambda: kv.rows(1, 2)),
        (ValueError, lambda: kv.select(ln.long(), ln)),
    ]
    cos, sin = tables(64, 16, BF)
    qkv = torch.zeros(2, 1, 8 * 64, dtype=BF, device=DEV)
    pos = torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    bad += [
        (ValueError, lambda: ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, 5)),
        (TypeError, lambda: ops.rope_kv_append_int4(qkv.half(), pos, cos, sin, kv, 4)),
        (ValueError, lambda: ops.rope_kv_append_int4(qkv, pos[:1], cos, sin, kv, 4)),
        (ValueError, lambda: ops.rope_kv_append_int4(qkv, pos, cos[:, :32], sin[:, :32], kv, 4)),
        (TypeError, lambda: ops.rope_kv_append_int4(qkv, pos, cos.half(), sin.half(), kv, 4)),
    ]
    codes, s, m = random_weight(g, 32, 128, 128, BF)
    w = Int4Weight.from_codes(codes, s, m, group_size=128)
    x = torch.zeros(2, 128, dtype=BF, device=DEV)
    bad += [
        (ValueError, lambda: int4_linear(x.cpu(), w)),
        (ValueError, lambda: int4_linear(x.half(), w)),
        (ValueError, lambda: int4_linear(x[:, :64], w)),
        (ValueError, lambda: int4_linear(x.repeat(33, 1), w)),
        (ValueError, lambda: int4_linear(x, w, "swiglu")),
        (ValueError, lambda: int4_linear(x, w, "gelu")),
        (ValueError, lambda: int4_linear(x, w, "residual")),
        (ValueError, lambda: int4_linear(x, w, resid=torch.zeros(2, 32, dtype=BF, device=DEV))),
        (ValueError, lambda: int4_linear(x, w, out=torch.zeros(2, 31, dtype=BF, device=DEV))),
        (ValueError, lambda: Int4Weight.from_codes(codes, s, m, group_size=64)),
        (ValueError, lambda: Int4Weight.from_codes(codes[:31], s[:31], m[:31], group_size=128, layout="swiglu")),
        (TypeError, lambda: Int4Weight.from_codes(codes, s.float(), m.float(), group_size=128)),
        (TypeError, lambda: Int4Weight(x.float())),
        (ValueError, lambda: Int4Weight(x, x[:1], layout="swiglu")),
    ]
    for kind, call in bad:
        with pytest.raises(kind, match="LlamaPureComputeError"):
            call()
    sq = Int4Weight(torch.zeros(128, 128, dtype=BF, device=DEV))
    with pytest.raises(ValueError, match="out must not be x"):
        int4_linear(x, sq, out=x)
    flat = torch.zeros(5 * 128, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="out must not be x"):
        int4_linear(flat[:256].view(2, 128), sq, out=flat[128:384].view(2, 128))
    with pytest.raises(ValueError, match="out may be resid"):
        int4_linear(x, sq, "residual", resid=flat[:256].view(2, 128), out=flat[128:384].view(2, 128))
    with pytest.raises(ValueError, match="out may be q"):
        flat4 = torch.zeros(2 * 4 * 64 + 64, dtype=BF, device=DEV)
        ops.decode_attention_int4(flat4[:512].view(2, 4, 64), kv, ln, out=flat4[64:].view(2, 4, 64))
    with pytest.raises(ValueError, match="overlap qkv"):
        ops.rope_kv_append_int4(qkv, pos, cos, sin, kv, 4, q_out=qkv.view(-1)[:512].view(2, 4, 1, 64))
    with pytest.raises(ValueError, match="k_out and v_out"):
        both = torch.zeros(2, 2, 1, 64, dtype=BF, device=DEV)
        ops.kv_read_int4(kv, pos, k_out=both, v_out=both)
    # nothing to do is no error
    assert ops.decode_attention_int4(q[:0], kv, ln).shape == (0, 4, 64)
    assert ops.kv_read_int4(kv, pos[:, :0])[0].shape == (2, 2, 0, 64)
    assert ops.rope_kv_append_int4(qkv[:, :0], pos[:, :0], cos, sin, kv, 4).shape == (2, 4, 0, 64)
    assert int4_linear(x[:0], w).shape == (0, 32)
