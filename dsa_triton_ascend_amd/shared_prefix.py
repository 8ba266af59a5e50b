"""``shared_prefix_attention``: dense MLA-absorb attention over a paged latent cache for a batch whose
sequences begin with the same tokens (a system prompt, a document asked about many times), the
shared part computed once for all of them.

The reference attends sparsely only; this is the dense form beside ``sparse_flash_attention``, over
the same PA_BSND caches, block tables and lengths: value = key, D = 128 / 256 / 512 plus a 64-wide
rope, N2 = 1. ``prefix_length=0`` is dense attention without sharing.
"""
from __future__ import annotations

import torch

from . import _host as H
from . import _lib
from .sparse_flash_attention import D_ROPE, VALID_D, VALID_N1


class SharedPrefixPlan:
    """Validated arguments of one shared_prefix_attention call (outputs, workspace, int32 index arrays),
    all in place when the constructor returns; ``run()`` launches on the current stream, which may be
    another one. Query, caches, ``act_k`` and the block table are read on the device in each run: a loop that
    keeps the plan may write them anew between runs. Of an operand that was not contiguous, at a 16-byte border
    and (the block table) int32, the plan reads its own copy (``q``, ``qr``, ``kk``, ``kr``, ``block_table``):
    a cache that grows between runs has to be contiguous.

    The constructor's lengths decide how the work is cut; any others written to ``act_k`` give the right result, but
    all that a sequence grows by falls to its last range, tile after tile (8 sequences of 16 heads after 2048
    shared tokens, 1500 tokens past the plan: 50 us a run, 22 of a plan for them). A loop builds its plan with
    lengths some hundred tokens ahead and writes the present ones to ``act_k`` (made for 1500 more: 20.5 us instead
    of 19.9 at first), or builds it anew every few hundred tokens."""

    def __init__(self, query, key, value, block_table, prefix_length, scale_value=1.0, actual_seq_lengths_query=None,
                 actual_seq_lengths_kv=None, query_rope=None, key_rope=None, layout_query="BSND", layout_kv="PA_BSND",
                 sparse_mode=3, return_softmax_lse=False, kv_splits=0, *, _wait=True):
        if sparse_mode not in (0, 3):
            raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
        if query_rope is None or key_rope is None:
            raise ValueError("query_rope and key_rope are required (no empty rope)")
        if layout_query not in ("BSND", "TND") or layout_kv != "PA_BSND":
            raise ValueError(f"unsupported layout {layout_query}/{layout_kv}")
        io = H.dtype_code(query.dtype, "query")
        for t, n in ((key, "key"), (query_rope, "query_rope"), (key_rope, "key_rope")):
            if t.dtype != query.dtype:
                raise ValueError(f"{n} dtype {t.dtype} differs from query dtype {query.dtype}")
        if query.dim() != (3 if layout_query == "TND" else 4) or key.dim() != 4:
            raise ValueError("query must be [B, S, N, D] (BSND) or [T, N, D] (TND), key [num_blocks, block_size, 1, D]")
        N1, D = query.shape[-2:]
        if D not in VALID_D:
            raise ValueError(f"D must be one of {VALID_D}, got {D}")
        if query_rope.shape[-1] != D_ROPE or key_rope.shape[-1] != D_ROPE:
            raise ValueError(f"rope dim must be {D_ROPE}, got {query_rope.shape[-1]} and {key_rope.shape[-1]}")
        if key.shape[2] != 1:
            raise ValueError("Only N2=1 (MQA) is supported")
        if N1 not in VALID_N1:
            raise ValueError(f"N1 must be one of {VALID_N1}, got {N1}")
        if key.shape[-1] != D or query_rope.shape[:-1] != query.shape[:-1] or key_rope.shape[:-1] != key.shape[:-1]:
            raise ValueError("query, query_rope, key and key_rope shapes do not match")
        if layout_query == "TND":
            act_q = [query.shape[0]] if actual_seq_lengths_query is None \
                else H.per_batch_from_cumsum(H.host_lengths(actual_seq_lengths_query))
            total_rows, per = query.shape[0], max(act_q, default=0)
            row_start = H.prefix(act_q)
            if row_start[-1] > total_rows or min(act_q, default=0) < 0:
                raise ValueError("actual_seq_lengths_query must be cumulative and within the packed query")
        else:
            B, per = query.shape[:2]
            act_q = H.batch_lengths(actual_seq_lengths_query, B, per, "actual_seq_lengths_query")
            if min(act_q, default=0) < 0 or max(act_q, default=0) > per:
                raise ValueError(f"actual_seq_lengths_query must lie between 0 and S = {per}")
            row_start = [b * per for b in range(B + 1)]
            total_rows = B * per
        self.batch, self.total_rows, self.max_rows = len(act_q), total_rows, per
        if block_table.dim() != 2 or block_table.shape[0] != self.batch:
            raise ValueError("block_table must be [batch, max_blocks]")
        self.num_blocks, self.page = key.shape[:2]
        self.max_blocks = block_table.shape[1]
        s2 = self.max_blocks * self.page
        act_k = H.host_lengths(actual_seq_lengths_kv, self.batch, s2)
        if len(act_k) != self.batch:
            raise ValueError(f"batch mismatch: {self.batch} query batches, {len(act_k)} kv lengths")
        if min(act_k, default=0) < 0 or max(act_k, default=0) > s2:
            raise ValueError(f"actual_seq_lengths_kv must lie between 0 and the block table's {s2} tokens")
        self.prefix = int(prefix_length)
        if not 0 <= self.prefix <= s2:
            raise ValueError(f"prefix_length {prefix_length} must lie between 0 and the block table's {s2} tokens")
        self.max_kv, self.total_kv, self.kv_splits = max(act_k, default=0), sum(act_k), int(kv_splits)
        if not 0 <= self.kv_splits <= 64:
            raise ValueError("kv_splits must lie between 0 and 64")
        self.dev = H.require_device(query, key, query_rope, key_rope, block_table)
        self.lib, self.io, self.n1, self.d = _lib.load(), io, N1, D
        self.scale, self.sparse_mode, self.return_lse = float(scale_value), sparse_mode, return_softmax_lse
        self.q, self.qr, self.kk, self.kr = (H.aligned16(t) for t in (query, query_rope, key, key_rope))
        self.empty = not (self.batch and total_rows and self.num_blocks and s2)
        self.args = None   # of the launch, but for the stream; None: nothing to do
        sm_shape = (1, total_rows, N1) if layout_query == "TND" else (self.batch, 1, per, N1)

        def place():
            # a cache without a block, or a table without a column, holds no token: zeros, as for rows that see none
            self.out = (torch.zeros if self.empty else torch.empty)(query.shape, dtype=query.dtype, device=self.dev)
            stats = torch.empty if return_softmax_lse and not self.empty else torch.zeros
            self.sm_max, self.sm_sum = self.sm = stats((2,) + sm_shape, dtype=torch.float32, device=self.dev).unbind(0)
            if self.empty:
                return
            self.block_table = block_table.to(torch.int32).contiguous()
            self.ws_bytes = self.lib.dsa_prefix_attn_workspace_bytes(self.batch, total_rows, N1, D, self.prefix, per,
                                                                     self.max_kv, self.total_kv, self.kv_splits)
            self.ws = torch.empty(self.ws_bytes, dtype=torch.uint8, device=self.dev) if self.ws_bytes else None
            self.row_start, self.act_q, self.act_k = H.upload(self.lib, self.dev, row_start, act_q, act_k, wait=_wait)
            lse = self.return_lse
            self.args = (self.q.data_ptr(), self.qr.data_ptr(), self.kk.data_ptr(), self.kr.data_ptr(), io,
                         self.block_table.data_ptr(), self.max_blocks, self.page, self.num_blocks, self.row_start.data_ptr(),
                         self.act_q.data_ptr(), self.act_k.data_ptr(), self.batch, total_rows, N1, D, D_ROPE, self.prefix, per,
                         self.max_kv, self.total_kv, sparse_mode, self.scale, self.out.data_ptr(),
                         self.sm_max.data_ptr() if lse else None, self.sm_sum.data_ptr() if lse else None, H.ptr(self.ws),
                         self.ws_bytes, self.kv_splits)

        H.on_device(self.dev, place)

    def run(self):
        if self.args is not None:
            H.on_device(self.dev, lambda: _lib.check(self.lib.dsa_prefix_attn(*self.args, H.stream_ptr(self.dev)),
                                                     "dsa_prefix_attn"))
        return self.out, self.sm_max, self.sm_sum


def shared_prefix_attention(query, key, value, block_table, prefix_length, scale_value=1.0, actual_seq_lengths_query=None,
                            actual_seq_lengths_kv=None, query_rope=None, key_rope=None, layout_query="BSND",
                            layout_kv="PA_BSND", sparse_mode=3, return_softmax_lse=False, kv_splits=0):
    """Dense attention over a paged latent cache; the first `prefix_length` tokens of all sequences are
    the same and are computed for the whole batch at once.

    query [B,S,N1,D] (BSND) or [T,N1,D] (TND, cumulative actual_seq_lengths_query; None: one sequence) and query_rope [..,64],
    fp16 / bf16; key [num_blocks, block_size, 1, D] and key_rope [.., 64] (`value` is ignored: value = key,
    as in sparse_flash_attention); block_table [B, max_blocks]; actual_seq_lengths_kv: each sequence's
    length, prefix included (default: the whole table). Tokens below prefix_length are read through
    block_table[0], for every sequence; the rest through each sequence's own row. A query row sees the
    tokens up to its own (sparse_mode 3: its last query is its last token) or all (0). Returns
    (attention_out, softmax_max, softmax_sum), the statistics [B,1,S,N1] / [1,T,N1] fp32 (zeros unless
    return_softmax_lse); rows that see no token give zeros. `kv_splits` > 0 forces the number of token
    ranges (tuning)."""
    return SharedPrefixPlan(query, key, value, block_table, prefix_length, scale_value, actual_seq_lengths_query,
                            actual_seq_lengths_kv, query_rope, key_rope, layout_query, layout_kv, sparse_mode,
                            return_softmax_lse, kv_splits, _wait=False).run()


class SharedPrefixAttention(torch.nn.Module):
    """Module form, with the arguments that stay the same from call to call."""

    def __init__(self, scale_value=1.0, layout_query="BSND", sparse_mode=3, return_softmax_lse=False):
        super().__init__()
        self.scale_value = scale_value
        self.layout_query = layout_query
        self.sparse_mode = sparse_mode
        self.return_softmax_lse = return_softmax_lse

    def forward(self, query, key, value, block_table, prefix_length, query_rope=None, key_rope=None,
                actual_seq_lengths_query=None, actual_seq_lengths_kv=None):
        return shared_prefix_attention(query, key, value, block_table, prefix_length, self.scale_value,
                                       actual_seq_lengths_query, actual_seq_lengths_kv, query_rope, key_rope,
                                       self.layout_query, "PA_BSND", self.sparse_mode, self.return_softmax_lse)
