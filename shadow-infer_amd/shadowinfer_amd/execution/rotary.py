"""Rotary positions for decoding: pairs in either layout, part of the head, and
the scalings that stretch a model past the context it was trained on.

``rope_split`` (row_ops.py) is the denoising step's fixed form (half layout,
whole head, tables in the row dtype, the reference's roundings). Here the angles
come from the positions themselves in 64 bits, so there is no table and no last
position, the products are fp32 and every value is rounded once.
"""

from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from typing import List, Optional, Tuple, Union

import torch

from .. import _native

_ROWS = ctypes.c_int64 * 9  # si_rotary_rows
_KINDS = ("linear", "ntk", "yarn", "bands")


@dataclass(frozen=True)
class RotaryScaling:
    """How the angles per position change for contexts ``factor`` times as long
    as the ``original_positions`` a model was trained on.

    * ``"linear"``: every angle divided by ``factor`` (position interpolation).
    * ``"ntk"``: the base times ``factor ** (r / (r - 2))``, r the rotary size, so
      that the slowest pair is divided by ``factor`` and the fastest kept.
    * ``"yarn"``: pairs that turn more than ``fast`` times over the original
      context kept, those that turn less than ``slow`` times divided by
      ``factor``, a linear ramp over the pair index between; values times
      ``0.1 ln(factor) + 1`` (Peng et al., arXiv 2309.00071).
    * ``"bands"``: kept above ``high`` turns over the original context, divided
      by ``factor`` below ``low``, a ramp that is linear in the turns between.
    """

    kind: str
    factor: float
    original_positions: int = 4096
    fast: float = 32.0
    slow: float = 1.0
    low: float = 1.0
    high: float = 4.0

    def __post_init__(self) -> None:
        if self.kind not in _KINDS:
            raise ValueError(f"scaling kind must be one of {_KINDS}, got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"factor must be >= 1, got {self.factor}")
        if self.original_positions < 1:
            raise ValueError(f"original_positions must be >= 1, got {self.original_positions}")
        if not (self.fast > self.slow > 0.0 and self.high > self.low > 0.0):
            raise ValueError("need fast > slow > 0 and high > low > 0")

    def angles(self, size: int, base: float) -> Tuple[List[float], float]:
        """(radians per position of each of the size / 2 pairs, factor on the
        values) in Python floats."""
        if self.kind == "ntk":
            if size < 4:
                raise ValueError("ntk scaling needs a rotary size of 4 at least")
            return _plain(size, base * self.factor ** (size / (size - 2))), 1.0
        f = _plain(size, base)
        if self.kind == "linear":
            return [x / self.factor for x in f], 1.0
        known = float(self.original_positions)
        if self.kind == "bands":
            out = []
            for x in f:
                turns = known * x / (2.0 * math.pi)
                keep = min(1.0, max(0.0, (turns - self.low) / (self.high - self.low)))
                out.append(keep * x + (1.0 - keep) * (x / self.factor))
            return out, 1.0

        def pair(turns: float) -> float:  # the pair that turns so often over the known context
            return size * math.log(known / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        first = max(math.floor(pair(self.fast)), 0)
        last = min(math.ceil(pair(self.slow)), size - 1)
        width = last - first if last != first else 0.001
        out = []
        for i, x in enumerate(f):
            slow = min(1.0, max(0.0, (i - first) / width))
            out.append(slow * (x / self.factor) + (1.0 - slow) * x)
        return out, 0.1 * math.log(self.factor) + 1.0


def _plain(size: int, base: float) -> List[float]:
    return [base ** (-2.0 * i / size) for i in range(size // 2)]


class RotaryEmbedding:
    """Rotates the first ``rotary_dim`` values (default: all) of query and key
    heads by their positions. ``layout``: ``"half"`` pairs value i with
    i + rotary_dim / 2, ``"interleaved"`` pairs 2i with 2i + 1."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 layout: str = "half", scaling: Optional[RotaryScaling] = None,
                 device: Union[str, torch.device] = "cuda") -> None:
        size = head_dim if rotary_dim is None else rotary_dim
        if not 0 < head_dim <= 1024:
            raise ValueError(f"head_dim must be in 1..1024, got {head_dim}")
        if size < 2 or size % 2 or size > head_dim:
            raise ValueError(f"rotary_dim must be even and in 2..{head_dim}, got {size}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if not (math.isfinite(base) and base > 1.0):
            raise ValueError(f"base must be > 1, got {base}")
        self.head_dim, self.rotary_dim = int(head_dim), int(size)
        self.base, self.layout, self.scaling = float(base), layout, scaling
        angles, self.value_factor = ((_plain(size, base), 1.0) if scaling is None
                                     else scaling.angles(size, base))
        self.angles = tuple(angles)  # radians per position of each pair
        self.device = torch.device(device)
        # turns per position, in fp64 on the device
        self._turns = torch.tensor([x / (2.0 * math.pi) for x in angles], dtype=torch.float64,
                                  device=self.device)
        self._bind()

    def _bind(self) -> None:
        self._spec = ctypes.create_string_buffer(struct.pack(  # si_rotation
            "=qqQd", self.rotary_dim // 2, 1 if self.layout == "interleaved" else 0,
            self._turns.data_ptr(), self.value_factor))

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k != "_spec"}

    def __setstate__(self, state: dict) -> None:  # a copy has a tensor of its own
        self.__dict__.update(state)
        self._bind()

    turns = property(lambda self: self._turns)

    def _rows(self, x: torch.Tensor, shape, what: str, inplace: bool):
        """(source, output, their si_rotary_rows). The source may be a copy."""
        s = x.stride()
        if inplace:
            if s[-1] != 1 or 0 in s and any(a == 0 and n > 1 for a, n in zip(s, shape)):
                raise ValueError(f"{what} cannot be rotated in place: strides {s}")
            out, o = x, s
        else:
            if s[-1] != 1:
                x = x.contiguous()
                s = x.stride()
            out = torch.empty_like(x)
            o = out.stride()
            if o[-1] != 1:  # of an expanded tensor
                out = torch.empty_like(x, memory_format=torch.contiguous_format)
                o = out.stride()
        if len(s) == 4:
            rows = _ROWS(x.data_ptr(), out.data_ptr(), shape[2], s[0], s[1], s[2], o[0], o[1], o[2])
        else:
            rows = _ROWS(x.data_ptr(), out.data_ptr(), shape[1], 0, s[0], s[1], 0, o[0], o[1])
        return x, out, rows

    def check_positions(self, positions: torch.Tensor, lead, index: int) -> Tuple[int, int, int]:
        """Refuses positions that are not one integer per token of ``lead`` on
        device ``index`` (``[S]`` also serves every row of ``[B, S]``); returns
        whether they are int64 and their element strides between batches and
        tokens."""
        wide = positions.dtype is torch.int64
        if not wide and positions.dtype is not torch.int32:
            raise TypeError(f"positions must be int64 or int32, got {positions.dtype}")
        if positions.get_device() != index:
            raise ValueError(f"positions must be on device {index}, got {positions.device}")
        shape = positions.shape
        if shape != lead and not (len(lead) == 2 and shape == lead[1:]):
            raise ValueError(f"positions must be {list(lead)}, got {list(shape)}")
        s = positions.stride()
        return wide, (s[0] if len(s) == 2 else 0), s[-1]

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None,
                 *, transpose: bool = False, inplace: bool = False
                 ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """Rotated ``q``, or ``(q, k)``: tensors ``[T, heads, D]`` or ``[B, S,
        heads, D]`` (any strides; fp32, fp16 or bf16; the head counts may differ),
        in one launch. ``positions``: int64 or int32 ``[T]``, ``[B, S]`` or, for
        every row of a batch, ``[S]``; any value. ``transpose=True`` turns the
        other way: the gradient of this call with respect to its input, and,
        where ``value_factor`` is 1, its inverse. ``inplace=True`` writes into q
        and k, which share no values then. Not recorded by autograd."""
        index = q.get_device()
        if index < 0:
            _native.require_device(q, "RotaryEmbedding")
        if index != self.turns.get_device():
            raise ValueError(f"this RotaryEmbedding is on {self.turns.device}, q on {q.device}")
        code = _native.dtype_code(q.dtype)
        shape = q.shape
        if len(shape) not in (3, 4) or shape[-1] != self.head_dim:
            raise ValueError(f"q must be [tokens, heads, {self.head_dim}] or [batch, tokens, heads, "
                             f"{self.head_dim}], got {tuple(shape)}")
        lead = shape[:-2]
        if k is not None:
            if k.dtype is not q.dtype or k.get_device() != index:
                raise ValueError("q and k must share device and dtype")
            kshape = k.shape
            if len(kshape) != len(shape) or kshape[:-2] != lead or kshape[-1] != self.head_dim:
                raise ValueError("q and k must hold the same tokens, got "
                                 f"{tuple(shape)} and {tuple(kshape)}")
            if inplace and k.data_ptr() == q.data_ptr() and k.numel():
                raise ValueError("q and k cannot be the same values in place")
        wide, pb, ps = self.check_positions(positions, lead, index)
        # sources stay bound until the launch is queued
        src_q, out_q, rows_q = self._rows(q, shape, "q", inplace)
        src_k, out_k, rows_k = (None, None, None) if k is None else self._rows(k, kshape, "k", inplace)
        B, S = lead if len(lead) == 2 else (1, lead[0])
        _native.call_on(index, "si_rotary", self._spec, rows_q, rows_k, code, B, S, self.head_dim,
                        transpose, positions.data_ptr(), wide, pb, ps)
        return out_q if k is None else (out_q, out_k)

    def __repr__(self) -> str:
        return (f"RotaryEmbedding(head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, "
                f"base={self.base}, layout={self.layout!r}, scaling={self.scaling})")
