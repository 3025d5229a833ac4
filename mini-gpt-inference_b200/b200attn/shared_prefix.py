"""Paged decode attention of a batch whose sequences share a prefix.

``paged_attention_batch_b200`` reads every sequence's whole context; where
many requests stand behind one system prompt or document, its bytes are
mostly the same prefix again and again.  :func:`shared_prefix_decode_b200`
reads the prefix once for the batch and each sequence's own keys once.  It
also takes grouped heads (several query heads to a key/value head).
"""
from __future__ import annotations

import functools
import operator

import torch

from . import _lib
from .ops import (_DTYPES, _INDEX, _DeviceCall, _index_arg, _inference_only, _launch,
                  _pool_fields, _status_ptr)
from .rope import _check_place

_PACK = _lib.packer(_lib.SharedPrefixArgs).pack


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index: int, *sizes) -> int:
    """The workspace that a call of these sizes needs on device ``index``."""
    with torch.cuda.device(index):
        return _lib.load().b200_shared_prefix_decode_workspace_size(*sizes)


def shared_prefix_decode_b200(q: torch.Tensor, pool, prefix_table, prefix_len: int,
                              block_tables: torch.Tensor, context_lengths: torch.Tensor,
                              layer_idx: int, *, out: torch.Tensor | None = None,
                              status: torch.Tensor | None = None, prepare: bool = False):
    """Decode attention of a batch with its shared prefix computed once.

    q: [B, Hq, D] (any strides), Hq a multiple of the pool's heads H (query
    head h reads head h // (Hq // H)); pool.k / pool.v: contiguous
    [L, P, S, H, D], float32 or bfloat16; prefix_table: the blocks of the
    first ``prefix_len`` positions, 1-D integer CUDA tensor or (not
    while a graph is captured) host ints;
    block_tables: [B, M] int32/int64, whose columns from
    ``prefix_len // S`` on hold the sequences' own blocks (earlier entries
    are not read); context_lengths: [B], prefix included.  The new token's K/V
    are already in the pool (``rope_kv_append_b200`` or ``kv_scatter_b200``).

    The launch and its workspace are sized by M, since the lengths are the
    device's: of tables much wider than the sequences need, pass a view of the
    columns that the longest one does, ``block_tables[:, :n]``.

    Scores, weights and sums are float32.  With bf16 q and pool and more than
    128 query rows to a key head (``B * Hq // H``) the prefix's weights are
    rounded to bf16 for their product with v (relative error 2^-8 each at most);
    elsewhere they keep 2^-16 or better.

    Where a prefix ends inside a block, position ``prefix_len`` is row
    ``prefix_len % S`` of the sequence's own block of that column.
    ``prefix_len`` 0 is a plain paged decode.  A sequence shorter than the
    prefix (a padding row) or longer than its table gets zero rows and sets
    DEV_BAD_LENGTH in ``status``.  Returns [B, Hq, D] in q.dtype, or fills
    ``out`` (any float dtype; q itself, or apart from it).
    """
    _inference_only(q)
    lib = _lib.load()
    if not q.is_cuda:
        raise ValueError("CUDA q required for the b200 backend")
    if q.ndim != 3:
        raise ValueError("q must have shape [B,Hq,D]")
    b, hq, d = q.shape
    if b == 0 or hq == 0 or d == 0:
        raise ValueError("q dimensions must be nonzero")
    if q.dtype not in _DTYPES:
        raise ValueError("q must be float32, bfloat16 or float16")
    index = q.get_device()
    pool_fields = _pool_fields(pool, index, layer_idx)
    _, _, _, _, block, h, pd, kv_dtype = pool_fields
    if pd != d or h == 0 or hq % h:
        raise ValueError("the KV pool needs q's head dimension and a divisor of its heads")
    if block_tables.ndim != 2:
        raise ValueError("block_tables must have shape [B,M]")
    rows, width = block_tables.shape
    if rows != b or width < 1:
        raise ValueError("block_tables must have shape [B,M] with at least one block column")
    if context_lengths.shape != (b,):
        raise ValueError("context_lengths must have shape [B]")
    if block_tables.dtype not in _INDEX or context_lengths.dtype not in _INDEX:
        raise ValueError("block_tables and context_lengths must contain integers")
    prefix_len = operator.index(prefix_len)
    if prefix_len < 0:
        raise ValueError("prefix_len must be >= 0")
    if block_tables.get_device() != index or context_lengths.get_device() != index:
        raise ValueError("all inputs must reside on same CUDA device")
    table = _index_arg(prefix_table, q.device, index, "prefix_table")
    if table.ndim != 1:
        raise ValueError("prefix_table must be 1-D")
    entries = table.shape[0]
    if entries * block < prefix_len:
        raise ValueError("incomplete KV block table for prefix")
    sp = 0 if status is None else _status_ptr(status, index)
    if out is None:
        out = q.new_empty((b, hq, d))
    elif out.shape != (b, hq, d) or out.dtype not in _DTYPES or out.get_device() != index:
        raise ValueError("out must be a [B,Hq,D] tensor on the q device")
    else:
        _check_place(out, q, "out")
    qd = _DTYPES[q.dtype]
    # A workspace of the call's own, from the allocator of the current stream
    # (or of the graph being captured): calls on other streams, and other
    # graphs' replays, have others.
    nbytes = _workspace_bytes(index, b, hq, h, d, prefix_len, width, block, kv_dtype, qd)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    args = _PACK(
        *pool_fields, layer_idx, b, hq, prefix_len, width, q.data_ptr(), *q.stride(), out.data_ptr(),
        *out.stride(), table.data_ptr(), entries, *table.stride(), block_tables.data_ptr(),
        *block_tables.stride(), context_lengths.data_ptr(), *context_lengths.stride(),
        ws.data_ptr(), nbytes, sp, qd, _DTYPES[out.dtype], _INDEX[table.dtype],
        _INDEX[block_tables.dtype], _INDEX[context_lengths.dtype], 0)
    if prepare:
        return _DeviceCall(lib.b200_shared_prefix_decode, args, index, out, "shared prefix decode",
                           (q, pool.k, pool.v, table, block_tables, context_lengths, status, ws))
    _launch(lib.b200_shared_prefix_decode, args, index, "shared prefix decode")
    return out
