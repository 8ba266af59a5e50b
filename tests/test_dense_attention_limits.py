"""Launches of dense_attention and its gradient that would have 2^32 threads are refused, with a reason, before anything is
launched. Without a GPU."""
from dsa_triton_ascend_amd import _lib
from tests.test_dense_attention import BASE, GRAD_BASE, call


def test_many_sequences_and_key_heads():
    lib = _lib.load()
    # 65535 sequences of one token, 16000 key heads of their own: 65535 * 16000 work-groups
    one = [(20, 65535), (21, 65535), (22, 65535), (24, 16000), (25, 16000), (27, 0), (28, 1), (29, 1), (23, 0)]
    assert call(lib.dsa_dense_attn, BASE, one) == -2 and "2^32 threads" in lib.dsa_last_error().decode()
    one = [(26, 65535), (27, 65535), (28, 65535), (29, 0), (30, 0), (31, 16000), (32, 16000), (34, 0), (35, 1), (36, 1), (37, 1)]
    assert call(lib.dsa_dense_attn_grad, GRAD_BASE, one) == -2 and "2^32 threads" in lib.dsa_last_error().decode()


def test_forced_ranges():
    lib = _lib.load()
    # 2^20 rows of 128 heads on as many, 64 ranges of 65536 tokens: 2^20 work-groups of 128 rows, or half as many of 256, by 64
    many = [(20, 16), (21, 1 << 20), (22, 1 << 20), (24, 128), (25, 128), (27, 0), (28, 65536), (29, 65536), (38, 64), (37, (1 << 63) - 1)]
    assert call(lib.dsa_dense_attn, BASE, many) == -2 and "2^32 threads" in lib.dsa_last_error().decode()
