"""Padded batches whose sequences lie apart (slices of a longer cache, heads before rows): operands read in place, without
a GPU."""
import sys

import pytest
import torch

import dsa_triton_ascend_amd as dsa

M = sys.modules["dsa_triton_ascend_amd.dense_attention"]
BF = torch.bfloat16


def lying(how, B=3, S=5, N=4, D=128):
    z = lambda *s: torch.zeros(*s, dtype=BF)
    return {"whole": lambda: z(B, S, N, D), "longer": lambda: z(B, 9, N, D)[:, :S], "middle": lambda: z(B, 9, N, D)[:, 2:2 + S],
            "heads first": lambda: z(B, N, S, D).transpose(1, 2), "wider": lambda: z(B, S, N + 3, D + 8)[:, :, 1:1 + N, 8:],
            "shared": lambda: z(1, S, N, D).expand(B, S, N, D), "heads shared": lambda: z(B, 9, 1, D)[:, :S].expand(B, S, N, D),
            "one row": lambda: z(B, 9, N, D)[:, 3:4], "one": lambda: z(1, 9, N, D)[:, :S], "far apart": lambda: z(2, 70000, 2, D)[:, :S],
            "one row far apart": lambda: z(2, 70000, 2, D)[:, :1]}[how]()


@pytest.mark.parametrize("how", ["whole", "longer", "middle", "heads first", "wider", "shared", "heads shared", "one row", "one", "far apart",
                                 "one row far apart"])
def test_read_in_place(how):
    x = lying(how)
    assert M._packed(x, x.shape[2]).data_ptr() == x.data_ptr()


def test_copied():
    """What the documentation names: strides within the last dimension, borders off 16 bytes, row strides from 2^24 on"""
    z = lambda *s: torch.zeros(*s, dtype=BF)
    for x in (z(2, 5, 4, 256)[..., ::2], z(2, 5, 4, 136)[..., 3:131], z(2, 5, 4, 132)[..., :128], z(2, 2, 4, 1 << 22)[..., :128],
              z(2 * 5 * 512 + 4).as_strided((2, 5, 4, 128), (5 * 512 + 4, 512, 128, 1))):
        y = M._packed(x, 4)
        assert y.data_ptr() != x.data_ptr() and y.data_ptr() % 16 == 0 and torch.equal(y.reshape(x.shape), x)


def test_c_entries_refuse():
    import ctypes

    from dsa_triton_ascend_amd import _lib
    from tests.test_dense_attention import BASE, GRAD_BASE, call
    lib = _lib.load()

    def strides(n, *changes):
        a = [4096] * n
        for i, v in changes:
            a[i] = v
        return ctypes.cast((ctypes.c_int64 * n)(*a), ctypes.c_void_p)

    for entry, base, n, out, behind, rows, keys, padded in (
            (lib.dsa_dense_attn_batched, BASE, 5, 32, 23, 21, 22, 33), (lib.dsa_dense_attn_grad_batched, GRAD_BASE, 7, 43, 29, 27, 28, 40)):
        odd = ctypes.c_void_p(24)
        with_batches = lambda *c: base[:-1] + [strides(n, *c), None]
        for c, changes, st, what in ((((0, 12),), [], -1, "16-byte"), (((n - 1, 4),), [], -1, "16-byte"), (((2, -8),), [], -2, "strides"),
                                     (((4, 1 << 45),), [], -2, "strides"), ((), [(behind, 1)], -1, "padded batches"),
                                     ((), [(padded, 0)], -1, "padded batches"), ((), [(keys, 11)], -1, "padded batches"),
                                     ((), [(rows, 7)], -1, "evenly"), ((), [(out, odd)], -1, "aligned")):
            assert call(entry, with_batches(*c), changes) == st, (what, lib.dsa_last_error())
            assert what in lib.dsa_last_error().decode(), (what, lib.dsa_last_error())
        # without rotary parts theirs are not read
        assert call(entry, with_batches((1, 3), (3, 3)), [(27 if n == 5 else 34, 0), (out, odd)]) == -1
        assert "aligned" in lib.dsa_last_error().decode()
    assert call(lib.dsa_dense_attn_batched, BASE[:-1] + [None, None], [(21, 0), (28, 0), (23, 0), (20, 1)]) == 0   # no rows: no launch
