"""A paged KV cache in 4 bits, decode attention over it, and the weights that eviction goes by.

`KVPoolQ4` is a `KVPool` of bytes whose head rows are 4-bit rows (the format is in include/emm_kv.h): whole blocks
move through gather, scatter, copy_blocks, migration and compaction like any other pool's. `append` takes 16-bit keys
and values, `read` gives them back, `attend` is one decode step's attention. `ScorePool` holds the attention weight that
every cached token has gathered; `select_tokens` says which tokens stay, and `KVPool.keep_tokens` moves them.

None of the calls is differentiable; all are asynchronous on the current stream of the pool's device, allocate what they
return (and a workspace) from torch's allocator on that stream, and replay from a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib
from .kv_pool import Context, KVPool, _stream_ptr, check_block_tables

_DTYPES = {torch.float16: _lib.DTYPE_FP16, torch.bfloat16: _lib.DTYPE_BF16}
_MAX_SIGNATURES = 64
_INT32_MAX = 0x7FFFFFFF
# torch.empty_strided allocates as torch.empty does, in about half its time per call (1.5 against 3-4 us on a slow host)
_new = torch.empty_strided


def _remember(cache: Dict[tuple, tuple], sig: tuple, got: tuple) -> None:
    if len(cache) >= _MAX_SIGNATURES:
        cache.clear()
    cache[sig] = got


class ScorePool(KVPool):
    """The accumulated attention weight of every cached token, per layer and KV head.

    `layers` are L fp32 tensors [NB, H, BS], one entry for each slot and KV head of the KV pool beside it. It is a
    single-plane block pool, so a request's weights move with its blocks (gather, scatter, copy_blocks).
    """

    def __init__(self, layers: Sequence[torch.Tensor], ctx: Optional[Context] = None):
        layers = list(layers)
        if not layers or layers[0].dim() != 3 or layers[0].dtype != torch.float32:
            raise ValueError("a score pool needs fp32 layer tensors [NB, H, BS]")
        if layers[0].device.type != "cuda":
            raise ValueError("a score pool lives on a CUDA device")
        super().__init__(layers, ctx)

    @classmethod
    def like(cls, pool: KVPool) -> "ScorePool":
        """Zero weights for a KV pool's slots."""
        if pool.num_planes != 2:
            raise ValueError("weights belong to a KV pool (two planes)")
        shape = (pool.num_blocks, pool.num_kv_heads, pool.block_size)
        return cls([torch.zeros(shape, dtype=torch.float32, device=pool.device) for _ in range(pool.num_layers)], pool.ctx)

    def reset(self, slot_mapping: torch.Tensor) -> None:
        """Zeroes the weights of newly appended tokens (all layers and heads); slot < 0 is skipped."""
        if (slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.device != self.device
                or not slot_mapping.is_contiguous()):
            raise ValueError("slot_mapping must be a contiguous 1-D int64 tensor on the pool's device")
        _lib.check(self.ctx._lib.emm_reset_scores(self._h, slot_mapping.data_ptr(), slot_mapping.numel(),
                                                  _stream_ptr(self.ctx.device)))

    def select_tokens(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, keep: int, recent: int = 0,
                      sink: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Which tokens stay when every sequence is cut to `keep` tokens.

        A sequence of n > keep tokens keeps its first `sink`, its last `recent`, and of the others those with the
        largest weights (equal weights: the earlier token; a NaN is the smallest). Returns (index, new_lens), both
        int32: index [L, B, H, keep] has the kept positions in ascending order (0 .. n-1 and then -1 for a sequence
        within its budget), new_lens [B] is min(n, keep). Changes nothing: pass index to keep_tokens of the KV pool
        and of this pool.
        """
        B, width = check_block_tables(self, block_tables, seq_lens)
        heads = self.block_size  # a block is [H, BS]
        if keep <= 0 or max(keep, abs(recent), abs(sink)) > _INT32_MAX:
            raise ValueError("keep must be positive, and the three counts fit 32 bits")
        device, per_layer = self.ctx.device, B * heads * keep
        index = _new((self.num_layers, B, heads, keep), (per_layer, heads * keep, keep, 1), dtype=torch.int32, device=device)
        new_lens = _new((B,), (1,), dtype=torch.int32, device=device)
        rc = self.ctx._lib.emm_select_tokens(
            self._h, block_tables.data_ptr(), block_tables.stride(0), width, seq_lens.data_ptr(), B, keep, recent, sink,
            index.data_ptr(), new_lens.data_ptr(), _stream_ptr(device))
        if rc:
            _lib.check(rc)
        return index, new_lens


class KVPoolQ4(KVPool):
    """A paged KV pool in 4 bits.

    `layers` are L uint8 tensors of logical shape [2, NB, BS, H, row_bytes(head_size)] (token-major, or the permuted
    view of a head-major allocation), `head_size` the channels of a head: 64, 128 or 256.
    """

    def __init__(self, layers: Sequence[torch.Tensor], head_size: int, ctx: Optional[Context] = None):
        layers = list(layers)
        row = self.row_bytes(head_size)
        if not layers or layers[0].dim() != 5 or layers[0].dtype != torch.uint8 or layers[0].shape[-1] != row:
            raise ValueError(f"a 4-bit pool of head size {head_size} needs uint8 layer tensors [2, NB, BS, H, {row}]")
        if layers[0].device.type != "cuda":
            raise ValueError("a 4-bit pool lives on a CUDA device")
        super().__init__(layers, ctx)
        if any(p % 16 for p in self.layer_ptrs) or any(s % 16 for s in (self.desc.plane_stride, self.desc.block_stride,
                                                                        self.desc.token_stride, self.desc.head_stride)):
            raise ValueError("rows of a 4-bit pool must lie on 16-byte boundaries")
        self.head_dim = head_size
        self._row_sigs: Dict[tuple, tuple] = {}
        self._attend_sigs: Dict[tuple, tuple] = {}
        self._emm_q4_append = self.ctx._lib.emm_q4_append
        self._emm_q4_read = self.ctx._lib.emm_q4_read
        self._emm_q4_attend = self.ctx._lib.emm_q4_attend

    @staticmethod
    def row_bytes(head_size: int) -> int:
        """Bytes of one 4-bit row (one token of one head of one plane)."""
        row = _lib.load().emm_q4_row_bytes(int(head_size))
        if row == 0:
            raise ValueError(f"4-bit rows have 64, 128 or 256 channels, not {head_size}")
        return row

    @classmethod
    def allocate(cls, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_size: int,
                 device: Optional[torch.device] = None, layout: str = "nhd", ctx: Optional[Context] = None) -> "KVPoolQ4":
        """A pool of zeros; layout "nhd" is token-major, "hnd" head-major."""
        return cls(alloc_q4_layers(num_layers, num_blocks, block_size, num_kv_heads, head_size,
                                   "cuda" if device is None else device, layout), head_size, ctx)

    # -- rows -----------------------------------------------------------------
    def _check_rows(self, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor, lead: int) -> tuple:
        """Validates [L, T, H, D] (lead = 1) or [T, H, D] keys and values; (T, dtype code, byte strides)."""
        want_tail = (self.num_kv_heads, self.head_dim)
        if key.dtype not in _DTYPES:
            raise ValueError(f"keys and values are float16 or bfloat16, got {key.dtype}")
        for name, t in (("key", key), ("value", value)):
            if t.dim() != lead + 2 + 1 or tuple(t.shape[-2:]) != want_tail:
                raise ValueError(f"{name} must be [{'L, ' if lead else ''}T, H, D] with H, D = {want_tail}")
            if t.dtype != key.dtype or t.device != self.device:
                raise ValueError(f"{name} must have the key's dtype and the pool's device")
            if t.stride(-1) != 1 or (t.stride(-2) != self.head_dim and self.num_kv_heads > 1):
                raise ValueError(f"{name} heads must be contiguous ([H, D] dense per token)")
        if key.shape != value.shape:
            raise ValueError("key and value shapes differ")
        T = key.shape[lead]
        self._check_slots(slot_mapping, T)
        ls = (key.stride(0) * 2, value.stride(0) * 2) if lead else (0, 0)
        row = self.num_kv_heads * self.head_dim * 2
        # a stride over a dimension of one token (or layer) addresses nothing: torch leaves it arbitrary
        kts, vts = (key.stride(lead) * 2, value.stride(lead) * 2) if T > 1 else (row, row)
        return T, _DTYPES[key.dtype], (ls[0], kts, ls[1], vts)

    def _check_slots(self, slot_mapping: torch.Tensor, T: Optional[int] = None) -> None:
        if (slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or (T is not None and slot_mapping.numel() != T)
                or slot_mapping.device != self.device or not slot_mapping.is_contiguous()):
            raise ValueError("slot_mapping must be a contiguous int64 device tensor with one entry per token")

    def _rows_sig(self, key, value, slot_mapping, lead):
        sig = (lead, key.shape, key.stride(), key.dtype, key.device, value.shape, value.stride(), value.dtype,
               value.device, slot_mapping.shape, slot_mapping.stride(), slot_mapping.dtype, slot_mapping.device)
        got = self._row_sigs.get(sig)
        if got is None:
            got = self._check_rows(key, value, slot_mapping, lead)
            if lead and key.shape[0] != self.num_layers:
                raise ValueError(f"key has {key.shape[0]} layers, pool has {self.num_layers}")
            _remember(self._row_sigs, sig, got)
        return got

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """Quantises one layer's new rows [T, H, D] (fp16 or bf16) into their slots; slot < 0 is skipped.
        The slots must be distinct: one that appears twice ends with bytes of both rows."""
        T, dt, (_, kts, _, vts) = self._rows_sig(key, value, slot_mapping, 0)
        rc = self._emm_q4_append(self._h, self.head_dim, dt, layer, 1, key.data_ptr(), value.data_ptr(), 0, kts, 0, vts,
                                 slot_mapping.data_ptr(), T, _stream_ptr(self.ctx.device))
        if rc:
            _lib.check(rc)

    def append_all_layers(self, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """The same for every layer in one launch; key/value are [L, T, H, D]."""
        T, dt, (kls, kts, vls, vts) = self._rows_sig(key, value, slot_mapping, 1)
        rc = self._emm_q4_append(self._h, self.head_dim, dt, 0, self.num_layers, key.data_ptr(), value.data_ptr(), kls, kts,
                                 vls, vts, slot_mapping.data_ptr(), T,
                                 _stream_ptr(self.ctx.device))
        if rc:
            _lib.check(rc)

    def bind_append(self, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor):
        """Pre-validated per-layer append over static [L, T, H, D] buffers (see KVPool.bind_append):
        returns append(layer, stream=None), which is refused once the pool is closed or `append.release()` was called."""
        T, dt, (kls, kts, vls, vts) = self._check_rows(key, value, slot_mapping, 1)
        if key.shape[0] != self.num_layers:
            raise ValueError(f"key has {key.shape[0]} layers, pool has {self.num_layers}")
        fn, device, L, pool = self._emm_q4_append, self.ctx.device, self.num_layers, self
        D, k, v, s = self.head_dim, key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr()

        def raw(layer: int, stream: int) -> int:
            if not 0 <= layer < L:  # the addresses below are per layer
                return _lib.ERR_BAD_ARG
            # the pool's handle is looked up in each call: a closed pool's is null, which the library refuses
            return fn(pool and pool._h, D, dt, layer, 1, k + layer * kls, v + layer * vls, 0, kts, 0, vts, s, T, stream)

        def append(layer: int, stream: Optional[int] = None) -> None:
            if not 0 <= layer < L:
                raise _lib.EmmError(_lib.ERR_BAD_ARG, f"layer {layer} outside [0, {L})")
            rc = raw(layer, _stream_ptr(device) if stream is None else stream)
            if rc:
                _lib.check(rc)

        def release() -> int:
            nonlocal pool
            pool = None
            return _lib.OK

        append.buffers = (key, value, slot_mapping, self)
        append.release = release
        append.raw = raw
        return append

    def read(self, slot_mapping: torch.Tensor, dtype: torch.dtype, layer_begin: int = 0,
             layer_count: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(key, value) [layer_count, T, H, D] of `dtype` (fp16 or bf16): what the rows at these slots stand for.
        A slot < 0 gives zeros."""
        dt = _DTYPES.get(dtype)
        if dt is None:
            raise ValueError(f"rows are read as float16 or bfloat16, not {dtype}")
        self._check_slots(slot_mapping)
        lc = self.num_layers - layer_begin if layer_count is None else layer_count
        if layer_begin < 0 or lc < 0 or layer_begin + lc > self.num_layers:
            raise ValueError(f"layer range [{layer_begin}, {layer_begin + lc}) outside [0, {self.num_layers})")
        T, H, D = slot_mapping.shape[0], self.num_kv_heads, self.head_dim
        device, row = self.ctx.device, H * D
        shape, strides = (lc, T, H, D), (T * row, row, D, 1)
        key, value = _new(shape, strides, dtype=dtype, device=device), _new(shape, strides, dtype=dtype, device=device)
        ts = row * 2
        rc = self._emm_q4_read(self._h, D, dt, layer_begin, lc, key.data_ptr(), value.data_ptr(), T * ts, ts, T * ts, ts,
                               slot_mapping.data_ptr(), T, _stream_ptr(device))
        if rc:
            _lib.check(rc)
        return key, value

    # -- attention --------------------------------------------------------------
    def _check_attend(self, query, block_tables, seq_lens, out, scores, max_len) -> tuple:
        dt = _DTYPES.get(query.dtype)
        if dt is None:
            raise ValueError(f"queries are float16 or bfloat16, got {query.dtype}")
        if query.dim() != 3 or query.shape[2] != self.head_dim or query.shape[1] == 0 or query.shape[1] % self.num_kv_heads:
            raise ValueError(f"query must be [B, heads, {self.head_dim}] with a multiple of {self.num_kv_heads} heads")
        B, width = check_block_tables(self, block_tables, seq_lens)
        heads, D = query.shape[1], self.head_dim
        if heads // self.num_kv_heads > _lib.MAX_QUERY_GROUP:
            raise ValueError(f"at most {_lib.MAX_QUERY_GROUP} query heads on one KV head")
        if B != query.shape[0]:
            raise ValueError(f"{query.shape[0]} queries, {B} sequences")
        for name, t in (("query", query), ("out", out)):
            if t is None:
                continue
            if t.shape != query.shape or t.dtype != query.dtype or t.device != self.device:
                raise ValueError(f"{name} must have the query's shape and dtype on the pool's device")
            if B and (t.stride(2) != 1 or (heads > 1 and t.stride(1) != D) or (B > 1 and t.stride(0) < heads * D)):
                raise ValueError(f"{name} heads must be contiguous ([heads, D] dense per sequence)")
        cap = width * self.block_size
        limit = cap if max_len is None else int(max_len)
        if limit < 0 or limit > cap or limit > _INT32_MAX:
            raise ValueError(f"max_len {limit} outside [0, {cap}], what the tables can hold")
        nbytes = C.c_uint64()
        _lib.check(self.ctx._lib.emm_q4_attend_workspace(self._h, D, B, heads, limit, int(scores is not None),
                                                             C.byref(nbytes)))
        dense = heads * D * 2
        qs = query.stride(0) * 2 if B > 1 else dense
        os_ = dense if out is None or B <= 1 else out.stride(0) * 2
        return dt, B, heads, width, limit, qs, os_, nbytes.value, D ** -0.5

    def attend(self, layer: int, query: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None, scores: Optional[ScorePool] = None,
               max_len: Optional[int] = None) -> torch.Tensor:
        """One decode step's attention of one layer: [B, heads, D], the query's dtype.

        `query` [B, heads, D] has one token per sequence, heads a multiple of the pool's KV heads (query head h reads
        KV head h // (heads / H)). Position t of sequence b is token t % BS of block block_tables[b, t // BS];
        `seq_lens[b]` tokens count (the appended new token among them), and a sequence of none gives zeros. Both are
        int32 device tensors; table entries behind the last block are not read. `scale` defaults to D ** -0.5. `out`,
        where given, must not overlap the query unless it is the same tensor.

        With `scores`, each token's weight, summed over the query heads of its KV head, is added to its entry of this
        layer; a block may then appear once in the tables, and in no call that overlaps on the GPU. `max_len` (default: what the tables can hold) bounds the
        lengths and sizes the workspace; a length outside is clamped and reported by Context.check_status.
        """
        sig = (query.shape, query.stride(), query.dtype, query.device, block_tables.shape, block_tables.stride(),
               block_tables.dtype, block_tables.device, seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device,
               None if out is None else (out.shape, out.stride(), out.dtype, out.device), scores is None, max_len)
        got = self._attend_sigs.get(sig)
        if got is None:
            got = self._check_attend(query, block_tables, seq_lens, out, scores, max_len)
            _remember(self._attend_sigs, sig, got)
        dt, B, heads, width, limit, qs, os_, nbytes, default_scale = got
        if scores is not None and not scores._h:
            raise ValueError("the score pool is closed")
        device = self.ctx.device
        if out is None:
            D = self.head_dim
            out = _new((B, heads, D), (heads * D, D, 1), dtype=query.dtype, device=device)
        ws = _new((nbytes,), (1,), dtype=torch.uint8, device=device) if nbytes else None
        rc = self._emm_q4_attend(
            self._h, self.head_dim, dt, layer, query.data_ptr(), qs, out.data_ptr(), os_, block_tables.data_ptr(),
            block_tables.stride(0), width, seq_lens.data_ptr(), B, heads, limit, default_scale if scale is None else scale,
            None if scores is None else scores._h, None if ws is None else ws.data_ptr(), nbytes,
            _stream_ptr(device))
        if rc:
            _lib.check(rc)
        return out


def alloc_q4_layers(num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_size: int, device,
                    layout: str = "nhd") -> List[torch.Tensor]:
    """Zeroed layer tensors of a 4-bit pool (zero bytes stand for zeros)."""
    if layout not in ("nhd", "hnd"):
        raise ValueError(f"unknown pool layout {layout!r}")
    row = KVPoolQ4.row_bytes(head_size)
    if layout == "nhd":
        shape = (2, num_blocks, block_size, num_kv_heads, row)
        return [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(num_layers)]
    shape = (2, num_blocks, num_kv_heads, block_size, row)
    return [torch.zeros(shape, dtype=torch.uint8, device=device).permute(0, 1, 3, 2, 4) for _ in range(num_layers)]
