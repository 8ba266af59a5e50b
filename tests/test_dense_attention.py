"""Refusals of dense_attention, dense_attention_grad and their C entries, without a GPU."""
import ctypes

import pytest
import torch

import dsa_triton_ascend_amd as dsa
from dsa_triton_ascend_amd import _lib

BF = torch.bfloat16
Z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)


def args(**change):
    a = dict(query=Z(2, 3, 8, 128), key=Z(2, 5, 4, 128), value=Z(2, 5, 4, 128), query_rope=Z(2, 3, 8, 64), key_rope=Z(2, 5, 4, 64))
    a.update(change)
    return a


REFUSED = [
    (dict(sparse_mode=1), "sparse_mode"), (dict(layout="SBH"), "layout"), (dict(layout="TND"), "must be"),
    (dict(query=Z(2, 3, 8, 128, dtype=torch.float32)), "dtype"), (dict(key=Z(2, 5, 4, 128, dtype=torch.half)), "key dtype"),
    (dict(value=Z(2, 5, 4, 128, dtype=torch.half)), "value dtype"), (dict(key_rope=Z(2, 5, 4, 64, dtype=torch.half)), "key_rope dtype"),
    (dict(query_rope=None), "both provided"), (dict(key_rope=None), "both provided"), (dict(query=Z(2, 3, 8, 96)), "D must be"),
    (dict(query=Z(2, 3, 6, 128)), "divisible"), (dict(key=Z(2, 5, 0, 128), value=Z(2, 5, 0, 128)), "divisible"),
    (dict(value=Z(2, 5, 4, 64)), "one shape"), (dict(key=Z(2, 5, 4, 64), value=Z(2, 5, 4, 64)), "one shape"),
    (dict(query_rope=Z(2, 3, 4, 64)), "leading"), (dict(key_rope=Z(2, 5, 1, 64)), "leading"), (dict(query_rope=Z(2, 3, 8, 32)), "rope dim"),
    (dict(query=Z(2, 3, 8, 64), key=Z(2, 5, 4, 64), value=Z(2, 5, 4, 64)), "rope dim"),
    (dict(key=Z(3, 5, 4, 128), value=Z(3, 5, 4, 128), key_rope=Z(3, 5, 4, 64)), "batch mismatch"),
    (dict(actual_seq_lengths_query=[4, 1]), "between 0 and 3"), (dict(actual_seq_lengths_kv=[5, -1]), "between 0 and 5"),
    (dict(actual_seq_lengths_kv=[1, 2, 3]), "per-batch"), (dict(), "GPU")]


@pytest.mark.parametrize("change,message", REFUSED)
def test_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        dsa.dense_attention(**args(**change))


def test_packed_lengths_refused():
    a = dict(query=Z(6, 8, 64), key=Z(9, 8, 64), value=Z(9, 8, 64), layout="TND")
    for cu_q, cu_k, message in (([3, 7], [4, 9], "within the packed"), ([4, 3], [4, 9], "cumulative"), ([3, 6], [4, 10], "within the packed"),
                                ([6], [4, 9], "batch mismatch"), ([3, 6], None, "batch mismatch"), ([3, 6], [3, 9], "GPU"), (None, None, "GPU")):
        with pytest.raises(ValueError, match=message):
            dsa.dense_attention(**a, actual_seq_lengths_query=cu_q, actual_seq_lengths_kv=cu_k)


def test_splits_refused():
    for n in (65, -1):
        with pytest.raises(ValueError, match="kv_splits"):
            dsa.dense_attention(**args(), kv_splits=n)


P = ctypes.c_void_p(16)   # never dereferenced: validation fails first
T = [P, 1024, 128]
BASE = T * 5 + [1, P, P, P, P, 2, 6, 10, 0, 8, 4, 128, 64, 3, 5, 3, 0.1, P, 1, None, None, P, 1 << 40, 0, None]


def call(entry, base, changes):
    a = list(base)
    for at, v in changes:
        a[at] = v
    return entry(*a)


def test_c_entry_refuses():
    lib = _lib.load()
    odd = ctypes.c_void_p(24)
    for changes, st, what in ([([(i, None)], -1, "null") for i in (0, 3, 6, 9, 12, 16, 17, 18, 19, 32)] + [
            ([(15, 2)], -1, "io_dtype"), ([(30, 1)], -1, "sparse_mode"), ([(26, 96)], -1, "D must"), ([(27, 32)], -1, "rope dim"),
            ([(26, 64)], -1, "rope dim"), ([(20, 0)], -1, "shape"), ([(21, -1)], -1, "shape"), ([(24, 0)], -1, "shape"),
            ([(25, 3)], -1, "divisible"), ([(23, 7)], -1, "past"), ([(28, 7)], -1, "past"), ([(29, 11)], -1, "past"), ([(20, 4)], -1, "evenly"),
            ([(21, 1 << 28)], -2, "2^30"), ([(22, 1 << 29)], -2, "2^30"), ([(0, odd)], -1, "16-byte"), ([(13, 12)], -1, "16-byte"),
            ([(7, 1 << 24)], -2, "strides"), ([(7, -8)], -2, "strides"), ([(32, odd)], -1, "aligned"), ([(34, P)], -1, "both"),
            ([(38, 65)], -2, "kv_splits"), ([(38, 2), (22, 1000), (29, 1000), (36, None)], -1, "workspace"),
            ([(38, 2), (22, 1000), (29, 1000), (37, 64)], -1, "workspace")]):
        assert call(lib.dsa_dense_attn, BASE, changes) == st, what
        assert what in lib.dsa_last_error().decode(), (what, lib.dsa_last_error())
    assert call(lib.dsa_dense_attn, BASE, [(21, 0), (28, 0), (23, 0), (20, 1)]) == 0   # no rows: no launch


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.dsa_dense_attn_workspace_bytes(2, 8192, 0, 32, 8, 128, 4096, 4096, 0) == 0     # enough rows: one range each
    w = lib.dsa_dense_attn_workspace_bytes(4, 4, 0, 32, 4, 128, 1, 8190, 0)
    assert 0 < w < 1 << 26
    assert lib.dsa_dense_attn_workspace_bytes(4, 4, 0, 32, 4, 128, 1, 8190, 1) == 0
    assert lib.dsa_dense_attn_workspace_bytes(4, 4, 0, 32, 3, 128, 1, 8190, 0) == 0


def grad_args(**change):
    a = args(d_out=Z(2, 3, 8, 128), out=Z(2, 3, 8, 128), softmax_max=Z(2, 4, 3, 2, dtype=torch.float32),
             softmax_sum=Z(2, 4, 3, 2, dtype=torch.float32))
    a.update(change)
    return a


GRAD_REFUSED = REFUSED[1:3] + REFUSED[4:] + [
    (dict(d_out=Z(2, 3, 8, 64)), "d_out must"), (dict(out=Z(2, 3, 8, 128, dtype=torch.half)), "out must"), (dict(d_out=None), "d_out must"),
    (dict(softmax_max=Z(2, 4, 3, 2)), "softmax_max"), (dict(softmax_sum=Z(2, 1, 3, 8, dtype=torch.float32)), "softmax_max and"),
    (dict(splits=65), "splits"), (dict(splits=-1), "splits")]


@pytest.mark.parametrize("change,message", GRAD_REFUSED)
def test_gradient_refuses(change, message):
    a = grad_args(**change)
    if "query" in change:   # the gradient's operands have the query's shape
        a.update(d_out=a["query"], out=a["query"])
    with pytest.raises(ValueError, match=message):
        dsa.dense_attention_grad(**a)


GRAD_BASE = T * 7 + [1, P, P, P, P, 2, 6, 10, 0, 0, 8, 4, 128, 64, 3, 5, 5, 3, 0.1, 1, P, P, P, P, P, P, P, P, 1 << 40, 0, None]


def test_c_gradient_entry_refuses():
    lib = _lib.load()
    odd = ctypes.c_void_p(24)
    for changes, st, what in ([([(i, None)], -1, "null") for i in (0, 3, 6, 9, 12, 15, 18, 22, 23, 24, 25, 41, 42, 43, 44, 45, 46, 47)] + [
            ([(21, 2)], -1, "io_dtype"), ([(38, 1)], -1, "sparse_mode"), ([(33, 96)], -1, "D must"), ([(34, 32)], -1, "rope dim"),
            ([(26, 0)], -1, "shape"), ([(32, 3)], -1, "divisible"), ([(30, 11)], -1, "past"), ([(36, 11)], -1, "past"),
            ([(30, -1)], -1, "past"), ([(15, odd)], -1, "16-byte"), ([(19, 4)], -1, "16-byte"), ([(16, 1 << 24)], -2, "strides"),
            ([(43, odd)], -1, "aligned"), ([(50, 65)], -2, "splits"), ([(48, None)], -1, "workspace"), ([(49, 16)], -1, "workspace")]):
        assert call(lib.dsa_dense_attn_grad, GRAD_BASE, changes) == st, what
        assert what in lib.dsa_last_error().decode(), (what, lib.dsa_last_error())
    none = [(27, 0), (28, 0), (35, 0), (36, 0), (37, 0), (26, 1)]
    assert call(lib.dsa_dense_attn_grad, GRAD_BASE, none) == 0   # nothing: no launch
