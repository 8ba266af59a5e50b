"""Rotary positions and the appends to the paged caches, on MI355X.

The reference's operators take queries and keys already rotated and caches already filled; these
are the steps before them: :func:`rotary_embedding` (and :func:`rotary_embedding_grad`) for
``query_rope`` / ``key_rope`` and the indexer's queries, :func:`latent_cache_append` and
:func:`index_cache_append` for the PA_BSND caches that ``sparse_flash_attention``,
``shared_prefix_attention`` and ``lightning_indexer`` read. Layouts, lengths and block tables are
those operators'.
"""
from __future__ import annotations

import ctypes
from array import array

import torch

from . import _host as H
from . import _lib

VALID_D = (128, 256, 512)
D_ROPE = 64
INDEX_WIDTHS = (64, 96, 128, 256, 512)
ARG_SEQUENCES = 18   # sequences whose lengths a call takes from the host
MAX_ROWS = 2 ** 31 - 1 - 4096   # tokens a call takes


def _frequencies(inv_freq, pairs=None) -> torch.Tensor:
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError("inv_freq must be a float32 tensor [rotary_dim / 2]")
    if inv_freq.numel() == 0 or (pairs is not None and inv_freq.numel() != pairs):
        raise ValueError(f"inv_freq holds {inv_freq.numel()} pairs" + ("" if pairs is None else f", {pairs} wanted"))
    return inv_freq.contiguous()


def _sections(sections, pairs: int):
    """(number of position axes, host int32 array or None)"""
    if sections is None:
        return 1, None
    s = [int(v) for v in sections]
    if not 1 <= len(s) <= 4 or min(s) < 0 or sum(s) != pairs:
        raise ValueError(f"sections must be 1 to 4 counts of pairs that add up to {pairs}, got {s}")
    return len(s), (ctypes.c_int32 * len(s))(*s)


def _positions(positions, lead, axes: int, sectioned: bool) -> torch.Tensor:
    """int32 / int64 positions of shape `lead` ([axes] + lead with sections), contiguous"""
    want = ((axes,) if sectioned else ()) + tuple(lead)
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be an int32 or int64 tensor")
    if tuple(positions.shape) != want:
        raise ValueError(f"positions must have shape {list(want)}, got {list(positions.shape)}")
    return positions.contiguous()


def _rows_view(x: torch.Tensor, layout: str, what: str):
    """x with a contiguous last dimension, its (batch, row, head) strides and its rows per batch"""
    if layout == "BSND":
        if x.dim() != 4:
            raise ValueError(f"{what} must be [B, S, N, D], got {list(x.shape)}")
    elif layout != "TND":
        raise ValueError(f"unsupported layout {layout}")
    elif x.dim() != 3:
        raise ValueError(f"{what} must be [T, N, D], got {list(x.shape)}")
    stride = x.stride()
    if stride[-1] != 1 and x.shape[-1] > 1:
        x = x.contiguous()
        stride = x.stride()
    if layout == "BSND":
        return x, stride[0], stride[1], stride[2], max(1, x.shape[1])
    return x, 0, stride[0], stride[1], max(1, x.shape[0])


def _row_positions(lengths, rows: int, dev) -> torch.Tensor:
    """int32 [rows]: each packed row's place in its sequence, 0 behind the last, written on the current stream"""
    def place():
        if not lengths:
            return torch.zeros(rows, dtype=torch.int32, device=dev)
        lib = _lib.load()
        row_start, = H.upload(lib, dev, H.prefix(lengths), wait=False)
        out = torch.empty(rows, dtype=torch.int32, device=dev)
        _lib.check(lib.dsa_row_positions(row_start.data_ptr(), len(lengths), rows, out.data_ptr(), H.stream_ptr(dev)),
                   "dsa_row_positions")
        return out

    return H.on_device(dev, place)


class _Rotation:
    """Validated arguments of one rotation and its output; ``run()`` launches on the current stream."""

    def __init__(self, x, positions, inv_freq, sections, rotary_start, interleaved, layout, inverse, what):
        x, sb, ss, sh, per = _rows_view(x, layout, what)
        freq = _frequencies(inv_freq)
        dtype = H.dtype_code(x.dtype, what, allow_f32=True)
        pairs = freq.numel()
        axes, sec = _sections(sections, pairs)
        shape = x.shape
        n, width = shape[-2:]
        if x.numel() // max(1, n * width) > MAX_ROWS:
            raise ValueError(f"more than {MAX_ROWS} tokens")
        pos = _positions(positions, shape[:-2], axes, sec is not None)
        if rotary_start < 0 or rotary_start + 2 * pairs > width:
            raise ValueError(f"rotary dimensions [{rotary_start}, {rotary_start} + {2 * pairs}) of a width of {width}")
        self.dev = H.require_device(x, pos, freq)
        self.lib = _lib.load()
        self.out = out = torch.empty_like(x, memory_format=torch.contiguous_format)   # (half of torch.empty's time)
        self.keep = (x, pos, freq, sec)
        self.args = (x.data_ptr(), sb, ss, sh, dtype, pos.data_ptr(), pos.dtype == torch.int64, axes, sec, freq.data_ptr(),
                     out.numel() // (n * width), per, n, width, rotary_start, 2 * pairs, bool(interleaved), inverse,
                     out.data_ptr()) if out.numel() else None

    def run(self):
        if self.args is not None:
            H.on_device(self.dev, lambda: _lib.check(self.lib.dsa_rotary(*self.args, H.stream_ptr(self.dev)), "dsa_rotary"))
        return self.out


def rotary_embedding(x, positions, inv_freq, sections=None, rotary_start=0, interleaved=True, layout="BSND"):
    """Rotates the dimensions [rotary_start, rotary_start + 2 * len(inv_freq)) of every head of x by
    its token's position; the others are copied.

    x [B,S,N,D] (BSND) or [T,N,D] (TND), fp16 / bf16 / fp32, any strides; positions int32 / int64
    [B,S] / [T]; inv_freq fp32, one inverse frequency a pair. Pair i is elements (2i, 2i+1) with
    `interleaved`, else (i, i + rotary_dim/2). With `sections` (1 to 4 counts of pairs) positions are
    [axes, B, S] / [axes, T], and each run of consecutive pairs turns by the position on its own axis: the
    time, height and width of an image's or video's tokens (not axes dealt out pair by pair). Angles are
    computed in 64 bits. Returns a new contiguous tensor, which autograd does not follow:
    :func:`rotary_embedding_grad` is the gradient."""
    return _Rotation(x, positions, inv_freq, sections, rotary_start, interleaved, layout, 0, "x").run()


def rotary_embedding_grad(d_out, positions, inv_freq, sections=None, rotary_start=0, interleaved=True, layout="BSND"):
    """Gradient of :func:`rotary_embedding` with respect to x: d_out rotated back. (For the gradients
    ``d_query_rope`` / ``d_key_rope`` of ``sparse_flash_attention_grad``, arguments as in the forward.)"""
    return _Rotation(d_out, positions, inv_freq, sections, rotary_start, interleaved, layout, 1, "d_out").run()


class RotaryEmbedding(torch.nn.Module):
    """Module form: keeps the inverse frequencies (float32 through casts of the module) and the layout."""

    def __init__(self, inv_freq, sections=None, rotary_start=0, interleaved=True, layout="BSND"):
        super().__init__()
        self.register_buffer("inv_freq", _frequencies(inv_freq), persistent=False)
        self.sections = sections
        self.rotary_start = rotary_start
        self.interleaved = interleaved
        self.layout = layout

    def _apply(self, fn, recurse=True):
        freq = self.inv_freq   # follows the module's device, not its type: 16 bits would turn far positions wrongly
        super()._apply(fn, recurse)
        if self.inv_freq.dtype != freq.dtype:
            self.inv_freq = freq.to(self.inv_freq.device)
        return self

    def forward(self, x, positions):
        return rotary_embedding(x, positions, self.inv_freq, self.sections, self.rotary_start, self.interleaved, self.layout)


class _AppendPlan:
    """What both appends share: the new tokens' rows, lengths and block table, and the norm's and the
    rotation's arguments. All in place when the constructor returns, so ``run()`` may be called on
    another stream; calls of one plan, and calls whose caches are the same, are ordered by the caller.
    ``act_k``, ``block_table`` and the operands are read on the device in each run: a loop that keeps the
    plan may write them anew between runs (in the plan's copy, where one had to be made contiguous)."""

    def _setup(self, x, caches, block_table, inv_freq, pairs, actual_seq_lengths_kv, actual_seq_lengths_query, positions,
               sections, layout, norm, more, what, _once):
        shape, dtype = x.shape, x.dtype   # (each .shape builds an object: a call's time is its host path)
        blocks = None
        for c, name in caches:
            if not isinstance(c, torch.Tensor) or not c.is_contiguous() or c.dim() != 4:
                raise ValueError(f"{name} must be a contiguous tensor [num_blocks, block_size, N, D]")
            if c.dtype != dtype:
                raise ValueError(f"{name} dtype {c.dtype} differs from {what} dtype {dtype}")
            num_blocks, page, _, _ = c.shape
            if blocks is not None and blocks != (num_blocks, page):
                raise ValueError("the caches must have the same blocks")
            blocks = num_blocks, page
        self.freq = _frequencies(inv_freq, pairs)
        self.axes, self.sec = _sections(sections, self.freq.numel())
        if positions is None and self.axes > 1:
            raise ValueError("several position axes need positions")
        self.pos = None if positions is None else _positions(positions, shape[:-2], self.axes, self.sec is not None)
        self.io = H.dtype_code(dtype, what)
        self.wdt = self.io
        for w in norm:
            if w is not None:
                self.wdt = H.dtype_code(w.dtype, "norm weights", allow_f32=True)
                if w.dtype != norm[0].dtype or w.shape != (shape[-1],):
                    raise ValueError(f"norm weights must share a dtype and have shape [{shape[-1]}]")
        if layout == "TND":
            self.total_rows = shape[0]
            act_q = H.per_batch_from_cumsum(H.host_lengths(actual_seq_lengths_query)) \
                if actual_seq_lengths_query is not None else [shape[0]]
            row_start = H.prefix(act_q)
            if row_start[-1] > shape[0] or min(act_q, default=0) < 0:
                raise ValueError("actual_seq_lengths_query must be cumulative and within the packed tokens")
        else:
            B, S = shape[0], shape[1]
            self.total_rows = B * S
            act_q = H.batch_lengths(actual_seq_lengths_query, B, S, "actual_seq_lengths_query")
            if min(act_q, default=0) < 0 or max(act_q, default=0) > S:
                raise ValueError(f"actual_seq_lengths_query must lie between 0 and S = {S}")
            row_start = [b * S for b in range(B + 1)]
        act_k = H.host_lengths(actual_seq_lengths_kv)
        if len(act_k) != len(act_q):
            raise ValueError(f"batch mismatch: {len(act_q)} query batches, {len(act_k)} kv lengths")
        table = block_table.shape
        if len(table) != 2 or table[0] != len(act_q):
            raise ValueError("block_table must be [batch, max_blocks]")
        self.num_blocks, self.page = num_blocks, page = blocks
        self.batch, self.max_blocks = batch, max_blocks = table
        if self.total_rows > MAX_ROWS:
            raise ValueError(f"more than {MAX_ROWS} tokens")
        for k in act_k:
            if k < 0 or k > max_blocks * page:
                raise ValueError(f"kv length {k} outside the block table's {max_blocks * page} tokens")
        self.dev = H.require_device(self.x, block_table, self.freq, self.pos, *norm, *more, *[c for c, _ in caches])
        self.norm = tuple(None if w is None else w.contiguous() for w in norm)   # before the upload that is waited for
        self.lib = _lib.load()
        self.args = None   # of the launch, but for the stream; None: nothing to do
        if not (batch and self.total_rows and max_blocks and num_blocks and page):
            return None, None

        if _once and batch <= ARG_SEQUENCES:   # the lengths go with the call: no upload before it
            self.block_table = block_table.to(torch.int32).contiguous()
            self.lengths = array("i", row_start + act_q + act_k)
            at = self.lengths.buffer_info()[0]
            lengths = (at, at + 4 * (batch + 1), at + 4 * (2 * batch + 1), True)
        else:
            def place():
                self.block_table = block_table.to(torch.int32).contiguous()
                return H.upload(self.lib, self.dev, row_start, act_q, act_k, wait=not _once)

            self.row_start, self.act_q, self.act_k = H.on_device(self.dev, place)
            lengths = (self.row_start.data_ptr(), self.act_q.data_ptr(), self.act_k.data_ptr(), False)
        rotation = (H.ptr(self.pos), self.pos is not None and self.pos.dtype == torch.int64, self.axes, self.sec,
                    self.freq.data_ptr())
        return rotation, (*lengths, self.block_table.data_ptr(), batch, self.total_rows, self.per, max_blocks, page,
                          num_blocks)

    def _launch(self, entry, what):
        if self.args is not None:
            H.on_device(self.dev, lambda: _lib.check(entry(*self.args, H.stream_ptr(self.dev)), what))


class LatentAppendPlan(_AppendPlan):
    """Validated arguments of one latent_cache_append call; ``run()`` launches on the current stream."""

    def __init__(self, latent, key_rope, key_cache, key_rope_cache, block_table, inv_freq, actual_seq_lengths_kv,
                 actual_seq_lengths_query=None, positions=None, norm_weight=None, norm_eps=1e-6, sections=None,
                 interleaved=True, layout="BSND", *, _once=False):
        self.x, self.sb, self.ss, self.sh, self.per = _rows_view(latent, layout, "latent")
        self.rope, self.rb, self.rs, _, _ = _rows_view(key_rope, layout, "key_rope")
        shape, rope_shape, cache_shape, rope_cache_shape = latent.shape, key_rope.shape, key_cache.shape, key_rope_cache.shape
        d = shape[-1]
        if d not in VALID_D:
            raise ValueError(f"D must be one of {VALID_D}, got {d}")
        if key_rope.dtype != latent.dtype:
            raise ValueError(f"key_rope dtype {key_rope.dtype} differs from latent dtype {latent.dtype}")
        if rope_shape[-1] != D_ROPE:
            raise ValueError(f"rope dim must be {D_ROPE}, got {rope_shape[-1]}")
        if shape[-2] != 1 or rope_shape[:-1] != shape[:-1]:
            raise ValueError("Only N2=1 (MQA) is supported, key_rope as many tokens as latent")
        if cache_shape[2:] != (1, d) or rope_cache_shape[2:] != (1, D_ROPE):
            raise ValueError(f"caches must be [num_blocks, block_size, 1, {d}] and [.., 1, {D_ROPE}]")
        rotation, places = self._setup(latent, [(key_cache, "key_cache"), (key_rope_cache, "key_rope_cache")], block_table, inv_freq,
                    D_ROPE // 2, actual_seq_lengths_kv, actual_seq_lengths_query, positions, sections, layout,
                    (norm_weight,), (key_rope,), "latent", _once)
        self.norm_weight, = self.norm
        self.key_cache, self.key_rope_cache = key_cache, key_rope_cache
        if places is not None:
            self.args = (self.x.data_ptr(), self.sb, self.ss, self.rope.data_ptr(), self.rb, self.rs, self.io, d,
                         H.ptr(self.norm_weight), self.wdt, float(norm_eps), *rotation, bool(interleaved), *places,
                         key_cache.data_ptr(), key_rope_cache.data_ptr())

    def run(self):
        self._launch(self.lib.dsa_latent_append, "dsa_latent_append")
        return self.key_cache, self.key_rope_cache


class IndexAppendPlan(_AppendPlan):
    """Validated arguments of one index_cache_append call; ``run()`` launches on the current stream."""

    def __init__(self, index_key, index_cache, block_table, inv_freq, actual_seq_lengths_key,
                 actual_seq_lengths_query=None, positions=None, norm_weight=None, norm_bias=None, norm_eps=1e-6,
                 sections=None, rotary_start=0, interleaved=False, layout="BSND", *, _once=False):
        if norm_bias is not None and norm_weight is None:
            raise ValueError("norm_bias needs norm_weight")
        self.x, self.sb, self.ss, self.sh, self.per = _rows_view(index_key, layout, "index_key")
        self.n2, self.w = index_key.shape[-2:]
        if self.w not in INDEX_WIDTHS:
            raise ValueError(f"D must be one of {INDEX_WIDTHS}, got {self.w}")
        if tuple(index_cache.shape[2:]) != (self.n2, self.w):
            raise ValueError(f"index_cache must be [num_blocks, block_size, {self.n2}, {self.w}]")
        self.start, self.rdim = int(rotary_start), 2 * _frequencies(inv_freq).numel()
        if self.start < 0 or self.start % 8 or self.rdim % 16 or self.start + self.rdim > self.w:
            raise ValueError(f"rotary dimensions [{self.start}, {self.start} + {self.rdim}) of {self.w}: the start a "
                             "multiple of 8, the count of 16")
        rotation, places = self._setup(index_key, [(index_cache, "index_cache")], block_table, inv_freq, None, actual_seq_lengths_key,
                    actual_seq_lengths_query, positions, sections, layout, (norm_weight, norm_bias), (), "index_key", _once)
        self.norm_weight, self.norm_bias = self.norm
        self.index_cache = index_cache
        if places is not None:
            self.args = (self.x.data_ptr(), self.sb, self.ss, self.sh, self.io, self.n2, self.w, H.ptr(self.norm_weight),
                         H.ptr(self.norm_bias), self.wdt, float(norm_eps), *rotation, self.start, self.rdim,
                         bool(interleaved), *places, index_cache.data_ptr())

    def run(self):
        self._launch(self.lib.dsa_index_append, "dsa_index_append")
        return self.index_cache


def latent_cache_append(latent, key_rope, key_cache, key_rope_cache, block_table, inv_freq, actual_seq_lengths_kv,
                        actual_seq_lengths_query=None, positions=None, norm_weight=None, norm_eps=1e-6, sections=None,
                        interleaved=True, layout="BSND"):
    """Writes new tokens' latents (normed) and rotary keys (rotated) into the paged caches that
    ``sparse_flash_attention`` and ``shared_prefix_attention`` read, in place.

    latent [B,S,1,D] (BSND) or [T,1,D] (TND), key_rope [..,1,64]; key_cache [num_blocks, block_size, 1, D]
    and key_rope_cache [.., 64], contiguous; block_table [B, max_blocks]; actual_seq_lengths_kv: each
    sequence's length with its new tokens (per batch, as for the paged reads); actual_seq_lengths_query:
    how many tokens are new (per batch, BSND; cumulative, TND; None: all of S, or one packed sequence).
    Token s of batch b goes to position kv - query + s of its sequence, and turns by that position or by `positions` (as in
    :func:`rotary_embedding`). norm_weight [D]: root-mean-square norm of the latent (None: stored as it
    is). Tokens before position 0, or whose block is -1 or outside the cache, are not stored; no other
    row of the caches changes. Two new tokens must not share a place. Returns the two caches."""
    return LatentAppendPlan(latent, key_rope, key_cache, key_rope_cache, block_table, inv_freq, actual_seq_lengths_kv,
                            actual_seq_lengths_query, positions, norm_weight, norm_eps, sections, interleaved, layout,
                            _once=True).run()


def index_cache_append(index_key, index_cache, block_table, inv_freq, actual_seq_lengths_key,
                       actual_seq_lengths_query=None, positions=None, norm_weight=None, norm_bias=None, norm_eps=1e-6,
                       sections=None, rotary_start=0, interleaved=False, layout="BSND"):
    """Writes new tokens' indexer keys into the paged cache that ``lightning_indexer`` (PA_BSND) reads,
    in place: layer norm (norm_weight, norm_bias [D]; none if norm_weight is None), then the rotation of
    the dimensions [rotary_start, rotary_start + 2 * len(inv_freq)), then the store.

    index_key [B,S,N2,D] or [T,N2,D], index_cache [num_blocks, block_size, N2, D], D in
    (64, 96, 128, 256, 512); places, positions and rules as :func:`latent_cache_append`. Returns the
    cache."""
    return IndexAppendPlan(index_key, index_cache, block_table, inv_freq, actual_seq_lengths_key,
                           actual_seq_lengths_query, positions, norm_weight, norm_bias, norm_eps, sections, rotary_start,
                           interleaved, layout, _once=True).run()
