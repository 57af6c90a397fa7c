"""Page pool of many sequences: quantized KV rows written to and read from slots
that the caller's scheduler hands out.

``PagedKVStore`` is one batch of equal lengths with its bookkeeping on the host;
this is the serving form of the same row format. Pages of all sequences lie in
one allocation per tensor, ``[pages, heads, page_size, ...]``, every page in the
pool's one precision; which sequence a page belongs to is in the caller's page
tables. Every argument that changes from step to step is a device tensor, so the
calls capture into graphs.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from .. import _native

_PREC_CODE = {"fp32": 0, "fp16": 1, "int8": 2, "int4": 3}


class KVPagePool:
    """``num_pages`` pages of ``page_size`` positions for ``num_heads`` kv heads
    of one layer. ``precision``: ``"fp32"`` keeps rows in ``dtype`` as they are,
    ``"fp16"``, ``"int8"`` (a scale per row) or ``"int4"`` (a scale per
    ``int4_group_size`` values, or per row where that does not divide
    ``head_dim``); scales are in ``dtype``. The rows are bit-identical to
    ``PagedKVStore``'s. ``k``, ``v``, ``scale_k`` and ``scale_v`` are the
    tensors (scales None where there are none)."""

    def __init__(self, num_pages: int, num_heads: int, head_dim: int, page_size: int = 32,
                 precision: str = "int8", dtype: torch.dtype = torch.bfloat16,
                 device: Any = "cuda", int4_group_size: int = 16) -> None:
        if precision not in _PREC_CODE:
            raise ValueError(f"Unsupported page precision: {precision}")
        for name, n in (("num_pages", num_pages), ("num_heads", num_heads),
                        ("page_size", page_size), ("int4_group_size", int4_group_size)):
            if n < 1:
                raise ValueError(f"{name} must be >= 1, got {n}")
        if not 1 <= head_dim <= 512:
            raise ValueError(f"head_dim must be in 1..512, got {head_dim}")
        if num_pages * num_heads * page_size >= 1 << 31:
            raise ValueError("a pool holds fewer than 2**31 rows (pages x heads x page_size)")
        self._dtype_code = _native.dtype_code(dtype)
        self.num_pages, self.num_heads = int(num_pages), int(num_heads)
        self.head_dim, self.page_size = int(head_dim), int(page_size)
        self.precision, self.dtype = precision, dtype
        g = int(int4_group_size)
        self.int4_group_size = g if head_dim % g == 0 else self.head_dim
        self.device = torch.device(device)
        payload, row, scales = {"fp32": (dtype, head_dim, None),
                                "fp16": (torch.float16, head_dim, None),
                                "int8": (torch.int8, head_dim, 1),
                                "int4": (torch.uint8, (head_dim + 1) // 2,
                                         head_dim // self.int4_group_size)}[precision]
        lead = (self.num_pages, self.num_heads, self.page_size)

        def zeros(n, kind):
            return torch.zeros(*lead, n, dtype=kind, device=self.device)

        self._k, self._v = zeros(row, payload), zeros(row, payload)
        self._sk = None if scales is None else zeros(scales, dtype)
        self._sv = None if scales is None else zeros(scales, dtype)
        self._table = _native.table4([_native.ptr(t) for t in (self._k, self._v, self._sk, self._sv)])

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    scale_k = property(lambda self: self._sk)
    scale_v = property(lambda self: self._sv)

    @property
    def num_slots(self) -> int:
        return self.num_pages * self.page_size

    def data_plane_bytes(self) -> int:
        """Bytes of the payload and scale tensors."""
        return sum(t.numel() * t.element_size() for t in (self._k, self._v, self._sk, self._sv)
                   if t is not None)

    def _check_slots(self, slots: torch.Tensor) -> None:
        if slots.dtype != torch.int64:
            raise TypeError(f"slots must be int64, got {slots.dtype}")
        if slots.dim() != 1:
            raise ValueError(f"slots must be [tokens], got {tuple(slots.shape)}")
        if slots.device != self._k.device:
            raise ValueError(f"slots must be on the pool's device ({self._k.device}), got {slots.device}")

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rotary=None,
              positions: Optional[torch.Tensor] = None) -> None:
        """K and V ``[T, heads, head_dim]`` in the pool's dtype (any strides) of
        token t into slot ``slots[t] = page * page_size + offset`` (int64). Slots
        outside the pool (-1 for padding) are skipped. No other slot may come
        twice in one call: which of its rows stays, and with which scale, would
        be open. With ``rotary`` (a RotaryEmbedding) K is rotated to
        ``positions`` ``[T]`` on its way, to the bytes that rotating first would
        give."""
        _native.require_device(k, "KVPagePool.write")
        if k.dim() != 3 or k.shape[1:] != (self.num_heads, self.head_dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be [tokens, {self.num_heads}, {self.head_dim}], got "
                             f"{tuple(k.shape)} and {tuple(v.shape)}")
        if k.dtype != self.dtype or v.dtype != self.dtype:
            raise TypeError(f"k and v must be {self.dtype}, got {k.dtype} and {v.dtype}")
        if k.device != self._k.device or v.device != self._k.device:
            raise ValueError(f"k and v must be on the pool's device ({self._k.device})")
        self._check_slots(slots)
        T = k.shape[0]
        if slots.shape[0] != T:
            raise ValueError(f"need {T} slots, got {slots.shape[0]}")
        turn = (0, 0, None, 1.0, None, 0, 0)
        if rotary is not None:
            if positions is None:
                raise ValueError("rotary needs positions")
            if rotary.head_dim != self.head_dim or rotary.turns.device != k.device:
                raise ValueError("rotary must have the pool's head_dim and device")
            _, step = rotary.check_positions(positions, k.shape[:1], k.device)
            turn = (rotary.rotary_dim // 2, 1 if rotary.layout == "interleaved" else 0,
                    rotary.turns.data_ptr(), rotary.value_factor, positions.data_ptr(),
                    1 if positions.dtype == torch.int64 else 0, step)
        elif positions is not None:
            raise ValueError("positions are of use with rotary only")
        # copies stay bound until the launch is queued
        kc = k if k.stride(2) == 1 else k.contiguous()
        vc = v if v.stride(2) == 1 else v.contiguous()
        sc = slots.contiguous()
        _native.call_on(k.device, "si_pool_write", kc.data_ptr(), vc.data_ptr(), self._dtype_code, T,
                        self.num_heads, self.head_dim, kc.stride(0), kc.stride(1), vc.stride(0),
                        vc.stride(1), sc.data_ptr(), self.num_pages, self.page_size,
                        _PREC_CODE[self.precision], self.int4_group_size, self._table, *turn)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float32
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) ``[T, heads, head_dim]`` of the slots (int64 ``[T]``) in
        ``dtype``: the values the stored rows stand for, zeros for a slot outside
        the pool."""
        _native.require_device(self._k, "KVPagePool.read")
        self._check_slots(slots)
        T = slots.shape[0]
        code = _native.dtype_code(dtype)
        sc = slots.contiguous()
        k = torch.empty(T, self.num_heads, self.head_dim, dtype=dtype, device=self._k.device)
        v = torch.empty_like(k)
        _native.call_on(k.device, "si_pool_read", sc.data_ptr(), T, self.num_heads, self.head_dim,
                        self.num_pages, self.page_size, _PREC_CODE[self.precision], self._dtype_code,
                        self.int4_group_size, self._table, k.data_ptr(), v.data_ptr(), code)
        return k, v

    def __repr__(self) -> str:
        return (f"KVPagePool(pages={self.num_pages}, heads={self.num_heads}, "
                f"head_dim={self.head_dim}, page_size={self.page_size}, "
                f"precision={self.precision!r}, dtype={self.dtype})")
