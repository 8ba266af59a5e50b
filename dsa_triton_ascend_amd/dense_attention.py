"""``dense_attention`` and ``dense_attention_grad``: dense attention of whole prompts, packed or padded, with
grouped key heads, on MI355X.

The reference attends sparsely only. The dense form beside it is what the indexer is trained against first:
the statistics of padded batches with heads of 128 are those that ``dense_loss_backward`` and its aliases take, and the
gradients train the attention itself. Keys and values are tensors of their own ([B, S2, N2, D] or [T2, N2, D]); for the paged latent
cache there is ``shared_prefix_attention``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _host as H
from . import _lib

VALID_D = (64, 128)
FEW_STATISTICS = 16384   # fp32 values
D_ROPE = 64
MAX_ROW = 1 << 24   # elements from one row to the next


def _packed(t: torch.Tensor, heads: int) -> torch.Tensor:
    """t as [rows, heads, width], or where a padded batch's sequences do not join as [sequences, rows, heads, width]; in place
    where the kernels can read its strides, else a copy"""
    if t.numel() == 0:
        return t.reshape(-1, heads, t.shape[-1]) if t.shape[-1] and heads else t
    if t.dim() == 4:
        B, S = t.shape[:2]
        batch, row = t.stride()[:2]
        if B == 1:
            t = t[0]
        elif S == 1 and batch < MAX_ROW:
            t = t[:, 0]
        elif S > 1 and batch == S * row:
            t = t.flatten(0, 1)
    if t.dim() == 3:
        row, head, last = t.stride()
        if last == 1 and not (row % 8 or head % 8 or t.data_ptr() % 16) and row < MAX_ROW:
            return t
    *lead, row, head = (x if n > 1 else 0 for x, n in zip(t.stride()[:-1], t.shape))   # (of one, it does not matter)
    if t.stride(-1) != 1 or row % 8 or head % 8 or t.data_ptr() % 16 or row >= MAX_ROW or (lead and lead[0] % 8):
        t = t.contiguous()
        t = _packed(t.clone() if t.data_ptr() % 16 else t, heads)
    return t


class _Arguments:
    """What the forward and the gradient share: checked operands as packed rows, and lengths"""

    batches = None

    def __init__(self, query, key, value, query_rope, key_rope, actual_seq_lengths_query, actual_seq_lengths_kv, scale_value,
                 layout, sparse_mode):
        if sparse_mode not in (0, 3):
            raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
        if layout not in ("BSND", "TND"):
            raise ValueError(f"unsupported layout {layout}")
        dims = 3 if layout == "TND" else 4
        if query.dim() != dims or key.dim() != dims or value.dim() != dims:
            raise ValueError("query, key and value must be " + ("[T, N, D]" if dims == 3 else "[B, S, N, D]"))
        self.io = H.dtype_code(query.dtype, "query")
        if (query_rope is None) != (key_rope is None):
            raise ValueError("query_rope and key_rope must be both provided or both omitted")
        for t, what in ((key, "key"), (value, "value"), (query_rope, "query_rope"), (key_rope, "key_rope")):
            if t is not None and t.dtype != query.dtype:
                raise ValueError(f"{what} dtype {t.dtype} differs from query dtype {query.dtype}")
        self.n1, self.d = query.shape[-2:]
        self.n2 = key.shape[-2]
        if self.d not in VALID_D:
            raise ValueError(f"D must be one of {VALID_D}, got {self.d}")
        if self.n1 <= 0 or self.n2 <= 0 or self.n1 % self.n2:
            raise ValueError("query N1 must be divisible by key N2")
        if key.shape[-1] != self.d or value.shape != key.shape:
            raise ValueError("key and value must have one shape, and the query's D")
        self.dr = 0
        if query_rope is not None:
            if query_rope.shape[:-1] != query.shape[:-1] or key_rope.shape[:-1] != key.shape[:-1]:
                raise ValueError("query_rope and key_rope must have query's and key's leading dimensions")
            if query_rope.shape[-1] != D_ROPE or key_rope.shape[-1] != D_ROPE or self.d != 128:
                raise ValueError(f"rope dim must be {D_ROPE}, beside D = 128")
            self.dr = D_ROPE
        if layout == "TND":
            self.total_rows, self.total_keys = query.shape[0], key.shape[0]

            def packed(x, total, what):
                n = [total] if x is None else H.per_batch_from_cumsum(H.host_lengths(x))
                if min(n, default=0) < 0 or sum(n) > total:
                    raise ValueError(f"{what} must be cumulative and within the packed tokens")
                return n, H.prefix(n)

            self.act_q, self.row_start = packed(actual_seq_lengths_query, self.total_rows, "actual_seq_lengths_query")
            self.act_k, self.key_start = packed(actual_seq_lengths_kv, self.total_keys, "actual_seq_lengths_kv")
            if len(self.act_q) != len(self.act_k):
                raise ValueError(f"batch mismatch: {len(self.act_q)} query batches, {len(self.act_k)} kv lengths")
            self.stat_shape = (self.n2, self.total_rows, self.n1 // self.n2)
        else:
            B, S1 = query.shape[:2]
            S2 = key.shape[1]
            if key.shape[0] != B:
                raise ValueError(f"batch mismatch: {B} query batches, {key.shape[0]} key batches")
            self.total_rows, self.total_keys = B * S1, B * S2

            def padded(x, n, what):
                v = H.batch_lengths(x, B, n, what)
                if min(v, default=0) < 0 or max(v, default=0) > n:
                    raise ValueError(f"{what} must lie between 0 and {n}")
                return v, [b * n for b in range(B + 1)]

            self.act_q, self.row_start = padded(actual_seq_lengths_query, S1, "actual_seq_lengths_query")
            self.act_k, self.key_start = padded(actual_seq_lengths_kv, S2, "actual_seq_lengths_kv")
            self.stat_shape = (B, self.n2, S1, self.n1 // self.n2)
        self.batch, self.padded = len(self.act_q), layout == "BSND"
        rows = [b - a for a, b in zip(self.row_start, self.row_start[1:])]
        self.rows_behind = self.total_rows - self.row_start[-1]
        self.max_rows, self.max_kv = max(rows + [self.rows_behind]), max(self.act_k, default=0)
        keys = [b - a for a, b in zip(self.key_start, self.key_start[1:])]
        self.keys_behind = self.total_keys - self.key_start[-1]
        self.max_keys = max(keys + [self.keys_behind])
        self.scale, self.sparse_mode = float(scale_value), sparse_mode
        self.operands = (query, query_rope, key, key_rope, value)

    def place(self, lib, wait, zero=None):
        """Operands and lengths on the device (and zeros in a tensor), with the device current"""
        heads = (self.n1, self.n1, self.n2, self.n2, self.n2)
        self.q, self.qr, self.k, self.kr, self.v = (None if t is None else _packed(t, n) for t, n in zip(self.operands, heads))
        self.d_lengths, self.at = H.upload_pointers(lib, self.dev, self.row_start, self.key_start, self.act_q, self.act_k,
                                                    zero=zero, wait=wait)

    def tensors(self, *more):
        """Pointers and strides as the C entries take them; `batches`: those of the sequences if some do not join, else None"""
        out, operands = [], (self.q, self.qr, self.k, self.kr, self.v) + more
        for t in operands:
            out += [None, 0, 0] if t is None else [t.data_ptr(), t.stride(-3) if t.shape[-3] > 1 else 0,
                                                   t.stride(-2) if t.shape[-2] > 1 else 0]
        if self.padded and any(t is not None and t.dim() == 4 for t in operands):
            self.batches = (ctypes.c_int64 * len(operands))(*(
                0 if t is None else t.stride(0) if t.dim() == 4 else t.stride(0) * (t.shape[0] // self.batch) for t in operands))
        return out

    def lengths(self):
        return *self.at, self.batch


class DenseAttentionPlan:
    """Validated arguments of one dense_attention call (outputs, workspace, int32 index arrays), all in place when
    the constructor returns; ``run()`` launches on the current stream, which may be another one. The operands are
    read on the device in each run: a loop that keeps the plan may write them anew between runs, also where they are slices of
    longer tensors or transposed ones. Only an operand with strides within the last dimension, with heads, rows or sequences off
    16-byte borders or with 2^24 elements or more from row to row is copied here, once: then the plan's copy (``q``, ``qr``,
    ``k``, ``kr``, ``v``) is what to write. Runs write the same outputs and workspace: the caller orders them."""

    def __init__(self, query, key, value, scale_value=1.0, actual_seq_lengths_query=None, actual_seq_lengths_kv=None,
                 query_rope=None, key_rope=None, layout="BSND", sparse_mode=3, return_softmax_lse=False, kv_splits=0, *,
                 _wait=True):
        a = self.arguments = _Arguments(query, key, value, query_rope, key_rope, actual_seq_lengths_query,
                                        actual_seq_lengths_kv, scale_value, layout, sparse_mode)
        if not 0 <= int(kv_splits) <= 64:
            raise ValueError("kv_splits must lie between 0 and 64")
        self.dev = a.dev = H.require_device(*a.operands)
        self.return_lse = return_softmax_lse
        self.lib = _lib.load()
        self.args = None   # of the launch, but for the stream; None: no row or no key, each run clears the outputs

        def place():
            empty = not (a.batch and a.total_rows and a.total_keys)
            self.out = H.empty_as(query)
            # statistics that nobody asked for are zeros: a small tensor is cleared by the lengths' launch
            total = 2 * a.n1 * a.total_rows
            few = not return_softmax_lse and not empty and total <= FEW_STATISTICS and total % 4 == 0
            both = (torch.empty if return_softmax_lse or empty or few else torch.zeros)(
                (2,) + a.stat_shape, dtype=torch.float32, device=self.dev)
            self.sm_max, self.sm_sum = both.unbind(0)
            if empty:
                self.cleared = (self.out, both)
                H.settle(self.dev, _wait)
                return
            size = self.lib.dsa_dense_attn_workspace_bytes(a.batch, a.total_rows, a.rows_behind, a.n1, a.n2, a.d, a.max_rows,
                                                           a.max_kv, int(kv_splits))
            self.ws = torch.empty(size, dtype=torch.uint8, device=self.dev) if size else None
            a.place(self.lib, _wait, both if few else None)
            self.q, self.qr, self.k, self.kr, self.v = a.q, a.qr, a.k, a.kr, a.v
            lse = return_softmax_lse
            self.args = (*a.tensors(), a.io, *a.lengths(), a.total_rows, a.total_keys, a.rows_behind, a.n1, a.n2, a.d, a.dr,
                         a.max_rows, a.max_kv, a.sparse_mode, a.scale, self.out.data_ptr(), a.padded,
                         self.sm_max.data_ptr() if lse else None, self.sm_sum.data_ptr() if lse else None, H.ptr(self.ws),
                         size, int(kv_splits))
            self.entry = self.lib.dsa_dense_attn
            if a.batches is not None:
                self.entry, self.args = self.lib.dsa_dense_attn_batched, self.args + (a.batches,)

        H.on_device(self.dev, place)

    def run(self):
        if self.args is not None:
            H.on_device(self.dev, lambda: _lib.check(self.entry(*self.args, H.stream_ptr(self.dev)), "dsa_dense_attn"))
        else:
            for t in self.cleared:
                t.zero_()
        return self.out, self.sm_max, self.sm_sum


def dense_attention(query, key, value, scale_value=1.0, actual_seq_lengths_query=None, actual_seq_lengths_kv=None,
                    query_rope=None, key_rope=None, layout="BSND", sparse_mode=3, return_softmax_lse=False, kv_splits=0):
    """Dense attention of prompts, of chunks of them or of single tokens.

    query [B,S1,N1,D] (BSND) or [T1,N1,D] (TND), key and value [B,S2,N2,D] or [T2,N2,D], D 64 or 128, fp16 / bf16; query
    head h reads key head h // (N1 // N2). query_rope and key_rope [..,64] (D = 128) add their product to the scores;
    one rotary key for all heads is passed expanded. Operands are read in place by their strides where sequences, rows
    and heads begin on 16-byte borders, rows less than 2^24 elements from each other (slices of one projection or of a longer
    cache, heads before rows, expanded heads or sequences), else copied.
    actual_seq_lengths_query / _kv: per batch (BSND; default: all) or cumulative (TND; default: one sequence). A query sees
    the tokens up to its own (sparse_mode 3: its sequence's last query is its last token) or all of its sequence (0).
    Returns (attention_out, softmax_max, softmax_sum), the statistics fp32 [B,N2,S1,N1//N2] or (TND) [N2,T1,N1//N2] (zeros
    unless return_softmax_lse); rows that see no token give zeros. ``dense_loss_backward`` takes those of BSND with D = 128: it
    has no heads of 64 and no packed layout, and its D = 256 and 512 have no counterpart here. autograd does not follow
    it: :func:`dense_attention_grad` is the gradient. `kv_splits` > 0 forces the number of token ranges (tuning)."""
    return DenseAttentionPlan(query, key, value, scale_value, actual_seq_lengths_query, actual_seq_lengths_kv, query_rope,
                              key_rope, layout, sparse_mode, return_softmax_lse, kv_splits, _wait=False).run()


class DenseAttentionGradPlan:
    """Validated arguments of one dense_attention_grad call (outputs, workspace, int32 index arrays), all in place when
    the constructor returns; ``run()`` launches on the current stream, which may be another one. Operands, d_out (``d``) and out
    (``o``) are read in each run, as by :class:`DenseAttentionPlan`; the statistics too where they are contiguous."""

    def __init__(self, query, key, value, d_out, out, softmax_max, softmax_sum, scale_value=1.0, query_rope=None, key_rope=None,
                 actual_seq_lengths_query=None, actual_seq_lengths_kv=None, layout="BSND", sparse_mode=3, splits=0, *, _wait=True):
        for t, what in ((d_out, "d_out"), (out, "out")):
            if not isinstance(t, torch.Tensor) or t.shape != query.shape or t.dtype != query.dtype:
                raise ValueError(f"{what} must have the query's shape and dtype")
        a = self.arguments = _Arguments(query, key, value, query_rope, key_rope, actual_seq_lengths_query,
                                        actual_seq_lengths_kv, scale_value, layout, sparse_mode)
        for t in (softmax_max, softmax_sum):
            if t.dtype != torch.float32 or tuple(t.shape) != a.stat_shape:
                raise ValueError(f"softmax_max and softmax_sum must be float32 of shape {list(a.stat_shape)}")
        if not 0 <= int(splits) <= 64:
            raise ValueError("splits must lie between 0 and 64")
        self.dev = a.dev = H.require_device(*a.operands, d_out, out, softmax_max, softmax_sum)
        self.lib = _lib.load()
        self.args = None   # of the launch, but for the stream; None: no row or no key, each run clears the gradients

        def place():
            empty = not (a.batch and a.total_rows and a.total_keys)
            self.grads = tuple(None if t is None else H.empty_as(t) for t in (query, key, value, query_rope, key_rope))
            if empty:
                H.settle(self.dev, _wait)
                return
            size = self.lib.dsa_dense_attn_grad_workspace_bytes(a.batch, a.total_rows, a.total_keys, a.rows_behind,
                                                                a.keys_behind, a.n1, a.n2, a.d, a.dr, a.max_rows, a.max_keys,
                                                                a.max_kv, int(splits))
            self.ws = torch.empty(size, dtype=torch.uint8, device=self.dev)
            self.d, self.o = (_packed(t, a.n1) for t in (d_out, out))
            self.sm_max, self.sm_sum = softmax_max.contiguous(), softmax_sum.contiguous()
            a.place(self.lib, _wait)
            dq, dk, dv, dqr, dkr = self.grads
            self.args = (*a.tensors(self.d, self.o), a.io, *a.lengths(), a.total_rows, a.total_keys, a.rows_behind,
                         a.keys_behind, a.n1, a.n2, a.d, a.dr, a.max_rows, a.max_keys, a.max_kv, a.sparse_mode, a.scale, a.padded,
                         self.sm_max.data_ptr(), self.sm_sum.data_ptr(), dq.data_ptr(), H.ptr(dqr), dk.data_ptr(), H.ptr(dkr),
                         dv.data_ptr(), self.ws.data_ptr(), size, int(splits))
            self.entry = self.lib.dsa_dense_attn_grad
            if a.batches is not None:
                self.entry, self.args = self.lib.dsa_dense_attn_grad_batched, self.args + (a.batches,)

        H.on_device(self.dev, place)

    def run(self):
        if self.args is not None:
            H.on_device(self.dev, lambda: _lib.check(self.entry(*self.args, H.stream_ptr(self.dev)), "dsa_dense_attn_grad"))
        else:
            for t in self.grads:
                if t is not None:
                    t.zero_()
        return self.grads


def dense_attention_grad(query, key, value, d_out, out, softmax_max, softmax_sum, scale_value=1.0, query_rope=None,
                         key_rope=None, actual_seq_lengths_query=None, actual_seq_lengths_kv=None, layout="BSND",
                         sparse_mode=3, splits=0):
    """Gradients of :func:`dense_attention`: ``(d_query, d_key, d_value, d_query_rope, d_key_rope)``, contiguous, in the
    operands' shapes and dtype (None without rotary parts). d_out: the gradient of attention_out; out, softmax_max and
    softmax_sum as the forward returned them with return_softmax_lse; the other arguments as in the forward. The gradients
    of a key head are summed over its query heads in 32 bits; where key heads share one expanded rotary key, each has
    its own d_key_rope, and their sum is the shared one's. Rows and keys that take no part get zeros. Results do not
    depend on timing. `splits` > 0 forces the number of ranges that sums over rows and keys are cut into (tuning)."""
    return DenseAttentionGradPlan(query, key, value, d_out, out, softmax_max, softmax_sum, scale_value, query_rope, key_rope,
                                  actual_seq_lengths_query, actual_seq_lengths_kv, layout, sparse_mode, splits,
                                  _wait=False).run()


class DenseAttention(torch.nn.Module):
    """Module form, with the arguments that stay the same from call to call."""

    def __init__(self, scale_value=1.0, layout="BSND", sparse_mode=3, return_softmax_lse=False):
        super().__init__()
        self.scale_value = scale_value
        self.layout = layout
        self.sparse_mode = sparse_mode
        self.return_softmax_lse = return_softmax_lse

    def forward(self, query, key, value, query_rope=None, key_rope=None, actual_seq_lengths_query=None,
                actual_seq_lengths_kv=None):
        return dense_attention(query, key, value, self.scale_value, actual_seq_lengths_query, actual_seq_lengths_kv,
                               query_rope, key_rope, self.layout, self.sparse_mode, self.return_softmax_lse)
