"""4-bit operators, host side: refusals of the C ABI and of the Python layer
(nothing is launched), and the weight quantiser, which runs on any device."""
import ctypes

import pytest
import torch

from llama_pure_compute_b200 import _lib, int4_linear, ops
from oracle.int4_ref import quantize_rows_ref, rows_ref, weight_ref

INVALID, UNSUPPORTED = _lib.LPC_ERR_INVALID, _lib.LPC_ERR_UNSUPPORTED


def cache(**kw):
    # the addresses are never followed: every call below is refused first
    f = dict(key_codes=16, key_scales=16, value_codes=16, value_scales=16, seq_base=None,
             seq_cap=None, max_batch=2, max_seq_len=64, total_rows=0, kv_heads=4, head_dim=128,
             dtype=2, reserved=0)
    f.update(kw)
    return _lib.Kv4(*[f[n] for n, _ in _lib.Kv4._fields_])


def weight(**kw):
    f = dict(packed=16, n_out=256, k=256, group=128, layout=0, dtype=2)
    f.update(kw)
    return _lib.W4(*[f[n] for n, _ in _lib.W4._fields_])


def attend(c, q=16, lens=16, out=16, ws=None, nbytes=0, batch=2, heads=8):
    return _lib.load().lpc_decode_attention_int4(ctypes.addressof(c), q, lens, out, ws, nbytes,
                                                 batch, heads, 1.0, None)


BAD_CACHES = [
    (dict(key_codes=None), INVALID, b"null cache pointer"),
    (dict(value_scales=None), INVALID, b"null cache pointer"),
    (dict(dtype=0), UNSUPPORTED, b"bf16 and fp16"),
    (dict(head_dim=96), UNSUPPORTED, b"head_dim"),
    (dict(kv_heads=0), INVALID, b"invalid cache sizes"),
    (dict(max_seq_len=0), INVALID, b"invalid cache sizes"),
    (dict(max_seq_len=2 ** 31), INVALID, b"invalid cache sizes"),
    (dict(max_batch=0), INVALID, b"invalid cache sizes"),
    (dict(seq_base=16, total_rows=64), INVALID, b"invalid cache sizes"),
    (dict(seq_base=16, seq_cap=16), INVALID, b"invalid cache sizes"),
    (dict(key_codes=24), INVALID, b"aligned"),
    (dict(value_scales=20), INVALID, b"aligned"),
]


@pytest.mark.parametrize("kw,code,text", BAD_CACHES)
def test_bad_caches_are_refused_by_every_entry_point(kw, code, text):
    lib, c = _lib.load(), cache(**kw)
    ref = ctypes.addressof(c)
    assert attend(c) == code and text in lib.lpc_last_error()
    assert lib.lpc_rope_kv_append_int4(ref, 16, 16, 16, 16, 64, 16, 1, 1, 8, 2, None) == code
    assert text in lib.lpc_last_error()
    assert lib.lpc_kv_read_int4(ref, 16, 16, 16, 1, 1, None) == code
    assert text in lib.lpc_last_error()
    assert lib.lpc_decode_attention_int4_workspace_bytes(ref, 1, 8) == 0


def test_attention_refusals():
    lib, c = _lib.load(), cache()
    assert attend(c, heads=6) == INVALID          # 6 heads on 4 KV heads
    assert attend(c, heads=0) == INVALID
    assert attend(c, batch=3) == INVALID          # beyond max_batch
    assert attend(c, batch=-1) == INVALID
    assert attend(c, q=None) == INVALID and attend(c, out=24) == INVALID
    big = cache(max_seq_len=65535 * 128 + 1)
    assert attend(big) == INVALID and b"invalid sizes" in lib.lpc_last_error()
    long = cache(max_seq_len=4096)                # several splits: needs a workspace
    need = lib.lpc_decode_attention_int4_workspace_bytes(ctypes.addressof(long), 2, 8)
    assert need > 0
    assert attend(long) == INVALID and b"workspace" in lib.lpc_last_error()
    assert attend(long, ws=16, nbytes=64) == INVALID
    assert attend(c, batch=0) == _lib.LPC_OK      # nothing to do


def test_append_and_read_refusals():
    lib, c = _lib.load(), cache()
    ref = ctypes.addressof(c)
    ap = lambda *a: lib.lpc_rope_kv_append_int4(ref, *a, None)  # noqa: E731
    assert ap(16, 16, 16, 16, 64, 16, 3, 1, 8, 2) == INVALID    # beyond max_batch
    assert ap(16, 16, 16, 16, 64, 16, -1, 1, 8, 2) == INVALID
    assert ap(16, 16, 16, 16, 0, 16, 1, 1, 8, 2) == INVALID     # empty tables
    assert ap(16, 16, 16, 16, 64, 16, 1, 1, 0, 2) == INVALID
    assert ap(None, 16, 16, 16, 64, 16, 1, 1, 8, 2) == INVALID
    assert ap(24, 16, 16, 16, 64, 16, 1, 1, 8, 2) == INVALID
    assert ap(16, 16, 16, 16, 64, 16, 1, 1, 8, 1) == UNSUPPORTED  # fp16 tables, bf16 cache
    assert ap(16, 16, 16, 16, 64, 16, 0, 1, 8, 2) == _lib.LPC_OK
    rd = lambda *a: lib.lpc_kv_read_int4(ref, *a, None)  # noqa: E731
    assert rd(16, 16, 16, 3, 1) == INVALID and rd(16, 16, 16, 1, -1) == INVALID
    assert rd(None, 16, 16, 1, 1) == INVALID and rd(16, 16, 24, 1, 1) == INVALID
    assert rd(16, 16, 16, 1, 0) == _lib.LPC_OK


@pytest.mark.parametrize("kw", [dict(packed=None), dict(packed=24), dict(k=100), dict(k=0),
                                dict(k=192, group=128), dict(group=16), dict(layout=2),
                                dict(n_out=0), dict(n_out=(1 << 24) + 1)])
def test_bad_weights_are_refused(kw):
    lib, w = _lib.load(), weight(**kw)
    ref = ctypes.addressof(w)
    assert lib.lpc_int4_linear(ref, 16, 16, None, 1, 0, None, 0, None) == INVALID
    assert lib.lpc_int4_pack(ref, 16, 16, 16, None) == INVALID
    assert lib.lpc_int4_unpack(ref, 16, None) == INVALID


def test_linear_refusals():
    lib = _lib.load()
    w0, w1, bad, wide = weight(), weight(layout=1), weight(dtype=0), weight(n_out=128, k=16384)
    huge = weight(n_out=8192, k=16384)
    ref, pair = ctypes.addressof(w0), ctypes.addressof(w1)

    def call(r, *a, ws=None, nbytes=0):
        return lib.lpc_int4_linear(r, *a, ws, nbytes, None)
    assert call(ref, 16, 16, None, 65, 0) == INVALID
    assert b"at most 64" in lib.lpc_last_error()
    assert call(ref, 16, 16, None, 1, 2) == INVALID   # swiglu on a plain weight
    assert call(pair, 16, 16, None, 1, 0) == INVALID
    assert call(ref, 16, 16, None, 1, 1) == INVALID   # no resid
    assert call(ref, 24, 16, None, 1, 0) == INVALID
    assert call(ref, 16, 16, None, 0, 0) == _lib.LPC_OK
    assert call(ctypes.addressof(bad), 16, 16, None, 1, 0) == UNSUPPORTED
    # the workspace: bf16, more tokens and values than the kernels without one take
    need = lib.lpc_int4_linear_workspace_bytes
    assert need(ref, 64) == 0 and need(ref, 0) == 0 and need(ref, 65) == 0
    large = weight(n_out=8192, k=4096)
    big = ctypes.addressof(large)
    assert need(big, 16) == 0 and need(big, 17) == 17 * 4096 * 2 + 256
    assert need(ctypes.addressof(wide), 8) == 0 and need(ctypes.addressof(huge), 8) == 8 * 16384 * 2 + 256
    half = weight(dtype=1, n_out=8192, k=4096)
    assert need(ctypes.addressof(half), 64) == 0
    assert call(big, 16, 16, None, 17, 0) == INVALID and b"workspace" in lib.lpc_last_error()
    assert call(big, 16, 16, None, 17, 0, ws=16, nbytes=100) == INVALID
    assert call(big, 16, 16, None, 17, 0, ws=24, nbytes=1 << 20) == INVALID
    size = lib.lpc_int4_weight_bytes
    assert size(100, 100, 128, 0) == 0
    # tile rows of 16, a multiple of 8 of them: codes, two sets of numbers, a factor a row
    assert size(17, 256, 128, 0) == size(17, 256, 128, 1) == 8 * (16 * 128 + 2 * 128 + 64)
    assert size(129, 256, 128, 0) == 2 * size(128, 256, 128, 0)


def test_python_layer_refuses_cpu_tensors():
    codes = torch.zeros(1, 2, 8, 64, dtype=torch.uint8)
    sc = torch.zeros(1, 2, 8, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be on CUDA device"):
        ops.Int4KV(codes, sc, codes, sc)
    with pytest.raises(ValueError, match="must be on CUDA device"):
        int4_linear.Int4Weight(torch.zeros(16, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="must be on CUDA device"):
        int4_linear.Int4Weight.from_codes(codes[0, 0], sc[0, 0], sc[0, 0], group_size=64)
    with pytest.raises(ValueError, match="unknown packed layout"):
        int4_linear.Int4Weight(torch.zeros(16, 128), layout="heads")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_weight_quantiser(dtype, group):
    g = torch.Generator().manual_seed(group)
    w = (torch.randn(37, 256, generator=g) * 0.02).to(dtype)
    w[3, :group] = 0.5      # a constant group: scale 0, read exactly
    w[4] = 0.0
    codes, s, m = int4_linear.Int4Weight.quantize(w, group)
    back = weight_ref(codes, s, m)
    # half a step of the stored scale, and what rounding the scale moves at code 15
    step = s.double().repeat_interleave(group, 1)
    half = torch.finfo(dtype).eps / 2
    assert ((back - w.double()).abs() <= step * (0.5 + 15 * half) + 2.0 ** -23).all()
    assert torch.equal(back[3, :group], w[3, :group].double())
    assert (back[4] == 0).all()
    for bad in (float("nan"), float("inf")):
        w[0, 0] = bad
        with pytest.raises(ValueError, match="non-finite"):
            int4_linear.Int4Weight.quantize(w, group)


def test_weight_quantiser_refuses_sizes():
    for k, group in ((96, 32), (100, 32), (192, 128), (256, 16)):
        with pytest.raises(ValueError):
            int4_linear.Int4Weight.quantize(torch.zeros(4, k, dtype=torch.bfloat16), group)


def test_row_oracle_is_within_half_a_step():
    """The oracle that the append kernel is held to keeps each value within half
    a step of its scale (plus what rounding the scale moves at code 15)."""
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.bfloat16, torch.float16):
        for D in (32, 64, 128):
            x = torch.randn(50, D, generator=g).to(dtype)
            codes, n = quantize_rows_ref(x)
            step = n.double()[:, [0, 2]].repeat_interleave(D // 2, 1)
            half = torch.finfo(dtype).eps / 2
            assert ((rows_ref(codes, n) - x.double()).abs()
                    <= step * (0.5 + 15 * half) + 2.0 ** -22).all()
