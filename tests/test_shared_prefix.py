"""Refusals of shared_prefix_attention and dsa_prefix_attn, without a GPU."""
import ctypes

import pytest
import torch

import dsa_triton_ascend_amd as dsa
from dsa_triton_ascend_amd import _lib

BF = torch.bfloat16
Z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)


def args(**change):
    a = dict(query=Z(2, 3, 16, 512), key=Z(8, 16, 1, 512), value=None, block_table=Z(2, 4, dtype=torch.int32), prefix_length=32,
             query_rope=Z(2, 3, 16, 64), key_rope=Z(8, 16, 1, 64), actual_seq_lengths_kv=[40, 64])
    a.update(change)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(sparse_mode=1), "sparse_mode"), (dict(query_rope=None), "required"), (dict(layout_kv="BSND"), "layout"),
    (dict(layout_query="SBH"), "layout"), (dict(query=Z(2, 3, 16, 512, dtype=torch.float32)), "dtype"),
    (dict(key=Z(8, 16, 1, 512, dtype=torch.half)), "key dtype"), (dict(layout_query="TND"), "query must be"),
    (dict(query=Z(2, 3, 16, 192)), "D must be"), (dict(query_rope=Z(2, 3, 16, 32)), "rope dim"),
    (dict(key_rope=Z(8, 16, 1, 32)), "rope dim"), (dict(key=Z(8, 16, 2, 512)), "N2=1"), (dict(query=Z(2, 3, 12, 512)), "N1 must"),
    (dict(key=Z(8, 16, 1, 256)), "shapes"), (dict(query_rope=Z(2, 2, 16, 64)), "shapes"), (dict(key_rope=Z(8, 8, 1, 64)), "shapes"),
    (dict(block_table=Z(3, 4)), "block_table"), (dict(actual_seq_lengths_kv=[40]), "batch mismatch"),
    (dict(actual_seq_lengths_kv=[40, 65]), "between 0 and"), (dict(actual_seq_lengths_kv=[-1, 5]), "between 0 and"),
    (dict(actual_seq_lengths_query=[4, 0]), "between 0 and S"), (dict(actual_seq_lengths_query=[1, 1, 1]), "per-batch"),
    (dict(prefix_length=65), "prefix_length"), (dict(prefix_length=-1), "prefix_length"), (dict(kv_splits=65), "kv_splits"),
    (dict(kv_splits=-1), "kv_splits"), (dict(), "GPU")])
def test_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        dsa.shared_prefix_attention(**args(**change))


def test_packed_lengths_refused():
    a = args(query=Z(6, 16, 512), query_rope=Z(6, 16, 64), layout_query="TND")
    for cu, message in (([3, 7], "within the packed"), ([4, 3], "cumulative"), ([6], "block_table")):
        with pytest.raises(ValueError, match=message):
            dsa.shared_prefix_attention(**a, actual_seq_lengths_query=cu)


def test_c_entry_refuses():
    lib = _lib.load()
    p = ctypes.c_void_p(16)   # never dereferenced: validation fails first
    base = [p, p, p, p, 1, p, 64, 16, 8, p, p, p, 2, 4, 16, 512, 64, 32, 2, 1000, 1600, 3, 0.04, p, None, None, p, 1 << 40, 2, None]
    for at, v, what in ([(i, None, "null") for i in (0, 1, 2, 3, 5, 9, 10, 11, 23)] +
                        [(4, 2, "io_dtype"), (21, 1, "sparse_mode"), (20, -1, "shape"), (15, 192, "D must"), (16, 32, "rope dim"), (14, 12, "N1 must"),
                         (12, 0, "shape"), (13, -1, "shape"), (6, 0, "shape"), (7, 0, "shape"), (8, 0, "shape"), (17, -1, "shape"),
                         (18, -1, "shape"), (19, -1, "shape"), (17, 1025, "past"), (19, 1025, "past"), (0, ctypes.c_void_p(24), "aligned"),
                         (23, ctypes.c_void_p(24), "aligned"), (24, p, "both"), (27, 0, "workspace"), (26, None, "workspace")]):
        a = list(base)
        a[at] = v
        assert lib.dsa_prefix_attn(*a) == _lib.DSA_ERR_INVALID, what
        assert what in lib.dsa_last_error().decode(), lib.dsa_last_error()
    for at, v, what in ((28, 65, "kv_splits"), (8, 1 << 31, "2^31"), (13, 1 << 27, "2^31")):
        a = list(base)
        a[at] = v
        assert lib.dsa_prefix_attn(*a) == _lib.DSA_ERR_UNSUPPORTED and what in lib.dsa_last_error().decode()
    a = list(base)
    a[13] = 0
    assert lib.dsa_prefix_attn(*a) == 0   # no rows: no launch


@pytest.mark.parametrize("batch,rows,n1,d,prefix,most,kv", [
    (1, 1, 1, 512, 0, 1, 1), (4, 4, 16, 512, 304, 1, 340), (64, 64, 16, 512, 8192, 1, 9700), (32, 32, 128, 512, 16384, 1, 20001),
    (5, 1965, 64, 512, 2048, 655, 2703), (1, 1, 1, 128, 1 << 20, 1, 1 << 21), (96, 384, 128, 128, 100, 4, 5000),
    (300, 300, 1, 256, 5000, 1, 5000), (2, 4000, 128, 512, 0, 2000, 4000)])
def test_workspace_is_bounded(batch, rows, n1, d, prefix, most, kv):
    """Partials: at most 256 ranges of blocks of 32 head rows (whole tiles of the prefix, a block more for
    each sequence), and no more than a few items per CU ask for (1 GiB at these sizes)."""
    lib = _lib.load()
    for splits in (0, 1, 64):
        w = lib.dsa_prefix_attn_workspace_bytes(batch, rows, n1, d, prefix, most, kv, batch * kv, splits)
        assert w % 16 == 0 and w <= 256 * ((rows * n1 + 32 * (batch + 5)) * 4 * d + rows * n1 * 16) + 256
        if splits == 0:
            assert w <= 1 << 30


def test_packed_without_lengths_is_one_sequence():
    a = args(query=Z(6, 16, 512), query_rope=Z(6, 16, 64), layout_query="TND")
    for change, message in ((dict(), "block_table"), (dict(block_table=Z(1, 4, dtype=torch.int32), actual_seq_lengths_kv=[40]), "GPU")):
        with pytest.raises(ValueError, match=message):
            dsa.shared_prefix_attention(**{**a, **change})


def test_c_entry_refuses_more_head_rows_than_a_launch_holds():
    lib, p = _lib.load(), ctypes.c_void_p(16)
    for rows in ((1 << 25) - 1, 1 << 25, 1 << 26):
        a = [p, p, p, p, 1, p, 64, 16, 8, p, p, p, 2, rows, 16, 512, 64, 32, 2, 1000, 1600, 3, 0.04, p, None, None, p, 1 << 60, 2, None]
        assert lib.dsa_prefix_attn(*a) == _lib.DSA_ERR_UNSUPPORTED and b"2^29" in lib.dsa_last_error()
