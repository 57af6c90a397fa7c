"""Attention of one new token of each sequence over a KVPagePool.

The decode step's counterpart of ``packed_attention``: grouped query heads over
the quantized rows that a page table names, dequantized on the way and never
written out, the cache's length split over the chip and joined.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from .. import _native
from .page_pool import KVPagePool


def paged_attention(q: torch.Tensor, pool: KVPagePool, page_table: torch.Tensor,
                    lengths: torch.Tensor, sm_scale: Optional[float] = None,
                    window: Optional[int] = None, return_lse: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``q`` ``[B, heads, D]`` (fp32, fp16 or bf16; the query heads a multiple of
    the pool's kv heads, head h reading kv head h // (heads / kv heads)) over
    positions 0 .. ``lengths[b]`` - 1 of sequence b, position t in page
    ``page_table[b, t // page_size]`` (int32 ``[B, pages]`` and int32 ``[B]``, both
    read on the device). Returns ``[B, heads, D]`` in q's dtype and, with
    ``return_lse``, the fp32 natural log-sum-exp of the scores ``[B, heads]``.

    ``window``: only the last so many positions. Positions of a page outside the
    pool (-1: dropped) take no part, lengths are cut to the table, negative ones
    are 0. A sequence without positions gives zeros and -inf. Several query heads
    of one kv head share its read; scores, softmax and sums are fp32. Not recorded by
    autograd."""
    index = q.get_device()
    if index < 0:
        _native.require_device(q, "paged_attention")
    shape = q.shape
    if len(shape) != 3 or shape[2] != pool.head_dim or shape[1] == 0 or shape[1] % pool.num_heads:
        raise ValueError(f"q must be [sequences, heads, {pool.head_dim}] with heads a multiple of "
                         f"{pool.num_heads}, got {tuple(shape)}")
    code = _native.dtype_code(q.dtype)
    B, H, D = shape
    if page_table.dtype is not torch.int32 or lengths.dtype is not torch.int32:
        raise TypeError(f"page_table and lengths must be int32, got {page_table.dtype} and "
                        f"{lengths.dtype}")
    tshape = page_table.shape
    if len(tshape) != 2 or tshape[0] != B or lengths.shape != shape[:1]:
        raise ValueError(f"need a page table [{B}, pages] and lengths [{B}], got "
                         f"{tuple(tshape)} and {tuple(lengths.shape)}")
    if pool._index != index or page_table.get_device() != index or lengths.get_device() != index:
        raise ValueError("q, the pool, page_table and lengths must be on one device")
    if window is None:
        window = 0
    elif not 1 <= window < 1 << 31:
        raise ValueError(f"window must be >= 1 (and below 2**31), got {window}")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    # copies stay bound until the launch is queued
    qs, ts, width = q.stride(), page_table.stride(), tshape[1]
    if qs[2] != 1:
        q = q.contiguous()
        qs = q.stride()
    if ts[1] != 1 and width > 1:
        page_table = page_table.contiguous()
        ts = page_table.stride()
    if B > 1 and lengths.stride(0) != 1:
        lengths = lengths.contiguous()
    out = q.new_empty(shape)
    lse = q.new_empty(shape[:2], dtype=torch.float32) if return_lse else None
    ws_bytes = _native.size_query("si_paged_attn_workspace_bytes", B, H, pool.num_heads, D,
                                  width * pool.page_size, window)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8) if ws_bytes else None
    _native.call_on(index, "si_paged_attn", pool._spec, q.data_ptr(), code, B, H, qs[0], qs[1],
                    page_table.data_ptr(), ts[0], width, lengths.data_ptr(), window, float(sm_scale),
                    out.data_ptr(), _native.ptr(lse), _native.ptr(ws), ws_bytes)
    return (out, lse) if return_lse else out
