"""Layer norm and its gradients, on MI355X.

``index_cache_append`` norms an indexer's keys on their way into the cache; these are the norm by itself
and the way back, for training: the gradients ``d_key_index`` of ``dense_loss_backward`` and
``sparse_lightning_indexer_grad_kl_loss`` go through ``rotary_embedding_grad`` and :func:`layer_norm_grad` to
the key projection.
"""
from __future__ import annotations

import torch

from . import _host as H
from . import _lib

MAX_WIDTH = 16384


def _rows(x, what: str):
    """x as rows of its last dimension, (rows, stride between them): x itself where its leading dimensions are
    evenly spaced, else a copy"""
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise ValueError(f"{what} must be a tensor [.., D]")
    width = x.shape[-1]
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"D must lie between 1 and {MAX_WIDTH}, got {width}")
    if width > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    rows = x.reshape(-1, width)
    stride = rows.stride(0)
    if rows.shape[0] > 1 and stride < width:   # rows that share memory (an expanded tensor)
        rows = rows.contiguous()
        stride = width
    return rows, rows.shape[0], stride if rows.shape[0] > 1 else width


def _weights(norm_weight, norm_bias, width: int) -> int:
    if norm_weight is None:
        if norm_bias is not None:
            raise ValueError("norm_bias needs norm_weight")
        return _lib.DSA_DTYPE_F32
    for w in (norm_weight, norm_bias):
        if w is not None and (w.dtype != norm_weight.dtype or tuple(w.shape) != (width,)):
            raise ValueError(f"norm weights must share a dtype and have shape [{width}]")
    return H.dtype_code(norm_weight.dtype, "norm weights", allow_f32=True)


def layer_norm(x, norm_weight=None, norm_bias=None, norm_eps=1e-6, return_stats=False):
    """``(x - mean) / sqrt(var + norm_eps) * norm_weight + norm_bias`` over the last dimension.

    x [.., D], fp16 / bf16 / fp32, any strides, 1 <= D <= 16384; norm_weight and norm_bias [D], fp16 / bf16 /
    fp32 (None: neither, or no bias). Statistics in 32 bits, one rounding. Returns a new contiguous tensor, which
    autograd does not follow (:func:`layer_norm_grad` is the gradient), with `return_stats` also the mean and
    1 / sqrt(var + norm_eps) of each row, [..] fp32."""
    rows, n, stride = _rows(x, "x")
    width = rows.shape[1]
    io = H.dtype_code(x.dtype, "x", allow_f32=True)
    wdt = _weights(norm_weight, norm_bias, width)
    dev = H.require_device(x, norm_weight, norm_bias)
    lib = _lib.load()
    lead = x.shape[:-1]

    def call():
        w, b = (None if t is None else t.contiguous() for t in (norm_weight, norm_bias))
        y = H.empty_as(x)
        mean = rstd = None
        if return_stats:
            mean, rstd = torch.empty((2,) + lead, dtype=torch.float32, device=dev).unbind(0)
        if n:
            _lib.check(lib.dsa_layer_norm(rows.data_ptr(), stride, io, n, width, H.ptr(w), H.ptr(b), wdt, float(norm_eps),
                                          y.data_ptr(), H.ptr(mean), H.ptr(rstd), H.stream_ptr(dev)), "dsa_layer_norm")
        return (y, mean, rstd) if return_stats else y

    return H.on_device(dev, call)


def layer_norm_grad(d_out, x, mean, rstd, norm_weight=None, norm_bias=None):
    """Gradients of :func:`layer_norm`: ``(d_x, d_weight, d_bias)``, d_x in x's dtype, the others [D] in their
    parameters' (None for a parameter that is None).

    d_out [.., D] in x's dtype, any strides; x and the parameters as in the forward (of norm_bias only its presence
    counts); mean and rstd [..] fp32, as it returned them. The sums over rows have a fixed order."""
    if not isinstance(d_out, torch.Tensor) or d_out.shape != x.shape or d_out.dtype != x.dtype:
        raise ValueError("d_out must have the shape and dtype of x")
    rows, n, stride = _rows(x, "x")
    d_rows, _, d_stride = _rows(d_out, "d_out")
    width = rows.shape[1]
    io = H.dtype_code(x.dtype, "x", allow_f32=True)
    wdt = _weights(norm_weight, norm_bias, width)
    for s in (mean, rstd):
        if s.dtype != torch.float32 or s.shape != x.shape[:-1]:
            raise ValueError(f"mean and rstd must be float32 of shape {list(x.shape[:-1])}")
    dev = H.require_device(d_out, x, mean, rstd, norm_weight, norm_bias)
    lib = _lib.load()

    def call():
        w = None if norm_weight is None else norm_weight.contiguous()
        m, r = mean.contiguous(), rstd.contiguous()
        dx = H.empty_as(x)
        dw = db = ws = None
        size = 0
        if w is not None:
            dw = H.empty_as(w)
            db = None if norm_bias is None else H.empty_as(w)
            size = lib.dsa_layer_norm_grad_workspace_bytes(n, width)
            ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        if not n:   # sums of nothing
            return dx, None if dw is None else dw.zero_(), None if db is None else db.zero_()
        _lib.check(lib.dsa_layer_norm_grad(d_rows.data_ptr(), d_stride, rows.data_ptr(), stride, io, n, width, m.data_ptr(),
                                           r.data_ptr(), H.ptr(w), wdt, dx.data_ptr(), H.ptr(dw), H.ptr(db), H.ptr(ws), size,
                                           H.stream_ptr(dev)), "dsa_layer_norm_grad")
        return dx, dw, db

    return H.on_device(dev, call)


class LayerNorm(torch.nn.Module):
    """Module form: keeps weight and bias. autograd does not follow it: a training loop sets their gradients itself,
    ``module.weight.grad, module.bias.grad = d_weight, d_bias`` of :func:`layer_norm_grad`; without that an optimiser leaves
    them as they are."""

    def __init__(self, width, norm_eps=1e-6, bias=True, dtype=torch.float32, device=None):
        super().__init__()
        self.norm_eps = norm_eps
        self.weight = torch.nn.Parameter(torch.ones(width, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(width, dtype=dtype, device=device)) if bias else None

    def forward(self, x, return_stats=False):
        return layer_norm(x, self.weight.detach(), None if self.bias is None else self.bias.detach(), self.norm_eps,
                          return_stats)
