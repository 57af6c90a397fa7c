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

import ctypes
from typing import Any, Optional, Tuple

import torch

from .. import _native

_PREC_CODE = {"fp32": 0, "fp16": 1, "int8": 2, "int4": 3}
_SPEC = ctypes.c_int64 * 11  # si_page_pool


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
        self._bind()

    def _bind(self) -> None:
        self._spec = _SPEC(self.num_pages, self.num_heads, self.page_size, self.head_dim,
                           _PREC_CODE[self.precision], self._dtype_code, self.int4_group_size,
                           *(_native.ptr(t) or 0 for t in (self._k, self._v, self._sk, self._sv)))
        self._index = self._k.get_device()

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k not in ("_spec", "_index")}

    def __setstate__(self, state: dict) -> None:  # a copy has tensors of its own
        self.__dict__.update(state)
        self._bind()

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

    def _rows(self, slots: torch.Tensor) -> int:
        """The number of slots; refuses what is not an int64 vector on the pool's device."""
        if slots.dtype is not torch.int64:
            raise TypeError(f"slots must be int64, got {slots.dtype}")
        if slots.get_device() != self._index:
            raise ValueError(f"slots must be on the pool's device ({self._k.device}), got {slots.device}")
        shape = slots.shape
        if len(shape) != 1:
            raise ValueError(f"slots must be [tokens], got {tuple(shape)}")
        return shape[0]

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rotary=None,
              positions: Optional[torch.Tensor] = None) -> None:
        """K and V ``[T, heads, head_dim]`` in the pool's dtype (any strides) of
        token t into slot ``slots[t] = page * page_size + offset`` (int64). Slots
        outside the pool (-1 for padding) are skipped. No other slot may come
        twice in one call: which of its rows stays, and with which scale, would
        be open. With ``rotary`` (a RotaryEmbedding) K is rotated to
        ``positions`` ``[T]`` on its way, to the bytes that rotating first would
        give. Not recorded by autograd."""
        index = self._index
        if k.get_device() < 0 or index < 0:
            _native.require_device(k, "KVPagePool.write")
            _native.require_device(self._k, "KVPagePool.write")
        if k.dtype is not self.dtype or v.dtype is not self.dtype:
            raise TypeError(f"k and v must be {self.dtype}, got {k.dtype} and {v.dtype}")
        if k.get_device() != index or v.get_device() != index:
            raise ValueError(f"k and v must be on the pool's device ({self._k.device})")
        shape = k.shape
        if len(shape) != 3 or shape[1] != self.num_heads or shape[2] != self.head_dim or v.shape != shape:
            raise ValueError(f"k and v must be [tokens, {self.num_heads}, {self.head_dim}], got "
                             f"{tuple(shape)} and {tuple(v.shape)}")
        T = self._rows(slots)
        if T != shape[0]:
            raise ValueError(f"need {shape[0]} slots, got {T}")
        spec, at, wide, step = None, None, 0, 0
        if rotary is not None:
            if positions is None:
                raise ValueError("rotary needs positions")
            if rotary.head_dim != self.head_dim or rotary.turns.get_device() != index:
                raise ValueError("rotary must have the pool's head_dim and device")
            wide, _, step = rotary.check_positions(positions, shape[:1], index)
            spec, at = rotary._spec, positions.data_ptr()
        elif positions is not None:
            raise ValueError("positions are of use with rotary only")
        # copies stay bound until the launch is queued
        ks, vs = k.stride(), v.stride()
        if ks[2] != 1:
            k = k.contiguous()
            ks = k.stride()
        if vs[2] != 1:
            v = v.contiguous()
            vs = v.stride()
        if T > 1 and slots.stride(0) != 1:
            slots = slots.contiguous()
        _native.call_on(index, "si_pool_write", self._spec, k.data_ptr(), v.data_ptr(), T, ks[0], ks[1],
                        vs[0], vs[1], slots.data_ptr(), spec, at, wide, step)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float32
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) ``[T, heads, head_dim]`` of the slots (int64 ``[T]``) in
        ``dtype``: the values the stored rows stand for, zeros for a slot outside
        the pool."""
        if self._index < 0:
            _native.require_device(self._k, "KVPagePool.read")
        T = self._rows(slots)
        code = _native.dtype_code(dtype)
        if T > 1 and slots.stride(0) != 1:
            slots = slots.contiguous()
        k = self._k.new_empty((T, self.num_heads, self.head_dim), dtype=dtype)
        v = torch.empty_like(k)
        _native.call_on(self._index, "si_pool_read", self._spec, slots.data_ptr(), T, k.data_ptr(),
                        v.data_ptr(), code)
        return k, v

    def __repr__(self) -> str:
        return (f"KVPagePool(pages={self.num_pages}, heads={self.num_heads}, "
                f"head_dim={self.head_dim}, page_size={self.page_size}, "
                f"precision={self.precision!r}, dtype={self.dtype})")
