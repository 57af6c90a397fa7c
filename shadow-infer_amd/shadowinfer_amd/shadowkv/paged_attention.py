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
from .page_pool import _PREC_CODE, KVPagePool


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
    of one kv head share its read; scores, softmax and sums are fp32."""
    _native.require_device(q, "paged_attention")
    if q.dim() != 3 or q.shape[2] != pool.head_dim or q.shape[1] == 0 or q.shape[1] % pool.num_heads:
        raise ValueError(f"q must be [sequences, heads, {pool.head_dim}] with heads a multiple of "
                         f"{pool.num_heads}, got {tuple(q.shape)}")
    code = _native.dtype_code(q.dtype)
    B, H, D = q.shape
    dev = q.device
    if page_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError(f"page_table and lengths must be int32, got {page_table.dtype} and "
                        f"{lengths.dtype}")
    if page_table.dim() != 2 or page_table.shape[0] != B or lengths.shape != (B,):
        raise ValueError(f"need a page table [{B}, pages] and lengths [{B}], got "
                         f"{tuple(page_table.shape)} and {tuple(lengths.shape)}")
    if pool.k.device != dev or page_table.device != dev or lengths.device != dev:
        raise ValueError("q, the pool, page_table and lengths must be on one device")
    if window is not None and not 1 <= window < 1 << 31:
        raise ValueError(f"window must be >= 1 (and below 2**31), got {window}")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    # copies stay bound until the launch is queued
    qc = q if q.stride(2) == 1 else q.contiguous()
    table = page_table if page_table.shape[1] < 2 or page_table.stride(1) == 1 else page_table.contiguous()
    lens = lengths.contiguous()
    out = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, H, dtype=torch.float32, device=dev) if return_lse else None
    width = page_table.shape[1]
    ws_bytes = _native.size_query("si_paged_attn_workspace_bytes", H, pool.num_heads, D,
                                  width * pool.page_size, window or 0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _native.call_on(dev, "si_paged_attn", qc.data_ptr(), code, B, H, qc.stride(0), qc.stride(1),
                    pool.num_heads, D, table.data_ptr(), table.stride(0), width, lens.data_ptr(),
                    window or 0, float(sm_scale), pool.num_pages, pool.page_size,
                    _PREC_CODE[pool.precision], pool._dtype_code, pool.int4_group_size, pool._table,
                    out.data_ptr(), _native.ptr(lse), _native.ptr(ws), ws_bytes)
    return (out, lse) if return_lse else out
