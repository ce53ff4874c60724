"""C ABI of the 4-bit cache: a batch larger than a ragged cache's index is refused before
anything is launched."""
import ctypes

from llama_pure_compute_b200 import _lib


def test_a_batch_beyond_the_ragged_index():
    lib = _lib.load()
    c = _lib.Kv4(16, 16, 16, 16, 16, 16, 3, 64, 200, 4, 128, 2, 0)  # the addresses are never followed
    ref = ctypes.addressof(c)
    assert lib.lpc_decode_attention_int4(ref, 16, 16, 16, None, 0, 4, 8, 1.0, None) == _lib.LPC_ERR_INVALID
    assert b"max_batch=3" in lib.lpc_last_error()
    assert lib.lpc_rope_kv_append_int4(ref, 16, 16, 16, 16, 64, 16, 4, 1, 8, 2, None) == _lib.LPC_ERR_INVALID
    assert b"max_batch=3" in lib.lpc_last_error()
    assert lib.lpc_kv_read_int4(ref, 16, 16, 16, 4, 1, None) == _lib.LPC_ERR_INVALID
    assert b"max_batch=3" in lib.lpc_last_error()
