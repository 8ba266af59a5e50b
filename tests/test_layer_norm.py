"""Refusals of layer_norm, layer_norm_grad and their C entries, without a GPU."""
import ctypes

import pytest
import torch

import dsa_triton_ascend_amd as dsa
from dsa_triton_ascend_amd import _lib

F = torch.float32
Z = lambda *s, dtype=F: torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("args,message", [
    ((Z(3, 0),), "between 1"), ((Z(2, 16385),), "between 1"), ((Z(()),), "tensor"), ((Z(2, 8, dtype=torch.int32),), "x dtype"),
    ((Z(2, 8, dtype=torch.double),), "x dtype"), ((Z(2, 8), None, Z(8)), "needs norm_weight"), ((Z(2, 8), Z(7)), "shape"),
    ((Z(2, 8), Z(8), Z(8, dtype=torch.half)), "share a dtype"), ((Z(2, 8), Z(8, dtype=torch.double)), "norm weights dtype"),
    ((Z(2, 8), Z(8), Z(8, 1)), "shape"), ((Z(2, 8), Z(8)), "GPU"), ((Z(0, 8), Z(8)), "GPU")])
def test_forward_refuses(args, message):
    with pytest.raises(ValueError, match=message):
        dsa.layer_norm(*args)


@pytest.mark.parametrize("change,message", [
    (dict(d_out=Z(2, 7)), "shape and dtype"), (dict(d_out=Z(2, 8, dtype=torch.half)), "shape and dtype"),
    (dict(mean=Z(3)), "mean and rstd"), (dict(rstd=Z(2, dtype=torch.half)), "mean and rstd"), (dict(rstd=Z(2, 1)), "mean and rstd"),
    (dict(norm_weight=None), "needs norm_weight"), (dict(norm_weight=Z(9)), "shape"), (dict(), "GPU")])
def test_gradient_refuses(change, message):
    a = dict(d_out=Z(2, 8), x=Z(2, 8), mean=Z(2), rstd=Z(2), norm_weight=Z(8), norm_bias=Z(8))
    a.update(change)
    with pytest.raises(ValueError, match=message):
        dsa.layer_norm_grad(**a)


def test_c_entries_refuse():
    lib = _lib.load()
    p = ctypes.c_void_p(16)   # never dereferenced: validation fails first
    fwd = [p, 8, 1, 4, 8, p, p, 2, 1e-6, p, p, p, None]
    for at, v, st, what in ((0, None, -1, "null"), (9, None, -1, "null"), (2, 5, -1, "dtype"), (3, -1, -1, "shape"), (4, 0, -1, "shape"),
                            (4, 16385, -2, "width"), (7, 3, -1, "weights"), (5, None, -1, "without norm_weight"), (10, None, -1, "both"),
                            (1, -8, -2, "strides"), (3, 1 << 61, -2, "64 bits"), (1, 1 << 61, -2, "64 bits")):
        a = list(fwd)
        a[at] = v
        assert lib.dsa_layer_norm(*a) == st and what in lib.dsa_last_error().decode(), (at, lib.dsa_last_error())
    a = list(fwd)
    a[3] = 0
    assert lib.dsa_layer_norm(*a) == 0   # no rows: no launch
    need = lib.dsa_layer_norm_grad_workspace_bytes(4, 8)
    assert need == 4 * 2 * 8 * 4 and lib.dsa_layer_norm_grad_workspace_bytes(0, 8) == 0
    assert lib.dsa_layer_norm_grad_workspace_bytes(10 ** 9, 16384) == 512 * 2 * 16384 * 4
    grad = [p, 8, p, 8, 1, 4, 8, p, p, p, 2, p, p, p, p, need, None]
    for at, v, st, what in ((0, None, -1, "null"), (2, None, -1, "null"), (7, None, -1, "null"), (8, None, -1, "null"), (11, None, -1, "null"),
                            (9, None, -1, "without norm_weight"), (14, None, -1, "workspace"), (15, need - 1, -1, "workspace"),
                            (14, ctypes.c_void_p(24), -1, "workspace"), (1, -1, -2, "strides"), (6, 16385, -2, "width"), (4, 7, -1, "dtype")):
        a = list(grad)
        a[at] = v
        assert lib.dsa_layer_norm_grad(*a) == st and what in lib.dsa_last_error().decode(), (at, lib.dsa_last_error())
    a = list(grad)
    a[5], a[12], a[13] = 0, None, None
    assert lib.dsa_layer_norm_grad(*a) == 0


def test_module_keeps_its_parameters():
    m = dsa.LayerNorm(12, bias=False, dtype=torch.bfloat16)
    assert m.bias is None and m.weight.shape == (12,) and m.weight.dtype == torch.bfloat16
    assert [n for n, _ in dsa.LayerNorm(5).named_parameters()] == ["weight", "bias"]
