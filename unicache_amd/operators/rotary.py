"""Rotary positions of several axes (time, height and width of images and
video; one axis for text): queries and keys turned alone, or on their way into
a PagedKVCache.  No reference counterpart: UniCache receives rotated keys."""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from .. import _native as nat

_HALVES = (torch.bfloat16, torch.float16)
_POSITION_BYTES = {torch.int32: 4, torch.int64: 8}


def check_rows(t: torch.Tensor, what: str) -> None:
    """Refuses rows that the kernels cannot read, or whose gradient they would drop."""

    if t.dtype not in _HALVES:
        raise ValueError(f"{what} must be bf16 or fp16 (got {t.dtype})")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which this call does not give; detach it")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} carries a forward-mode gradient, which this call does not give; detach it")


class MultiAxisRotary:
    """Turns pairs of a head's channels by angles positions[axis] * frequency.

    ``sections`` are the pairs of each axis, in turn: (16, 24, 24) gives the
    first 16 pairs to axis 0, the next 24 to axis 1, the last 24 to axis 2;
    ``axes`` names each pair's axis instead, in any order.  Pair i has frequency
    theta^(-i / pairs), or ``frequencies[i]`` (radians per position).  With
    pairing "halves" pair i is channels (i, i + pairs), with "adjacent"
    (2 i, 2 i + 1); channels from 2 pairs on stay as they are.

        (a, b) -> (a cos - b sin, b cos + a sin)

    Angles are 64-bit products of which whole turns are taken off, so far
    positions keep their precision; sines, cosines and the turn are fp32, rounded once to the rows' dtype.
    The plan belongs to one device and holds two small tensors there."""

    def __init__(self, head_dim: int, sections, *, theta: float = 10000.0, frequencies=None, pairing: str = "halves",
                 axes=None, device: torch.device | str = "cuda") -> None:
        sections = [int(n) for n in sections]
        if not sections or any(n < 0 for n in sections):
            raise ValueError("Rotary sections must name an axis at least, with no negative number of pairs")
        if len(sections) >= 1 << 16:
            raise ValueError("Rotary sections: too many axes")
        pairs = sum(sections)
        head_dim = int(head_dim)
        if head_dim <= 0 or head_dim % 16 or head_dim > 512:
            raise ValueError("Rotary head_dim must be a multiple of 16, and 512 at most")
        if pairs <= 0 or pairs % 8 or 2 * pairs > head_dim:
            raise ValueError("Rotary sections must have a multiple of 8 pairs in all, and no more than half of head_dim")
        if pairing not in ("halves", "adjacent"):
            raise ValueError(f"Rotary pairing must be 'halves' or 'adjacent' (got {pairing!r})")
        if axes is None:
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
        else:
            axes = [int(a) for a in axes]
            if len(axes) != pairs or [axes.count(a) for a in range(len(sections))] != sections:
                raise ValueError("Rotary axes must name each pair's axis, as many of each as its section")
        if frequencies is None:
            if not (math.isfinite(theta) and theta > 0.0):
                raise ValueError("Rotary theta must be positive")
            frequencies = [float(theta) ** (-i / pairs) for i in range(pairs)]
        else:
            frequencies = [float(f) for f in frequencies]
            if len(frequencies) != pairs or not all(math.isfinite(f) for f in frequencies):
                raise ValueError("Rotary frequencies must be one finite number for each pair")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"Rotary positions require a GPU (got {device})")
        self.head_dim, self.pairs, self.num_axes, self.pairing = head_dim, pairs, len(sections), pairing
        turns = [f / (2.0 * math.pi) for f in frequencies]
        self._turns = torch.tensor(turns, dtype=torch.float64, device=device)
        self._axis = torch.tensor(axes, dtype=torch.int32, device=device)
        self._adjacent = 1 if pairing == "adjacent" else 0
        self.device = self._turns.device

    def plan(self, positions: torch.Tensor | None, sequences: int, tokens: int, *, inverse: bool = False):
        """The C plan for [axes, sequences, tokens] positions (None: a cache's own), and the tensor it points to."""

        size, at = 0, None
        if positions is not None:
            size = _POSITION_BYTES.get(positions.dtype, 0)
            if not size:
                raise ValueError(f"Rotary positions must be int32 or int64 (got {positions.dtype})")
            if positions.dim() == 2 and sequences == 1:
                positions = positions.unsqueeze(1)
            if positions.shape != (self.num_axes, sequences, tokens):
                raise ValueError(f"Rotary positions must be [{self.num_axes}, {sequences}, {tokens}] (axes, sequences, "
                                 f"tokens), got {tuple(positions.shape)}")
            if positions.device != self.device:
                raise RuntimeError(f"Rotary positions must be on the plan's device {self.device}")
            if not positions.is_contiguous():
                positions = positions.contiguous()
            at = positions.data_ptr()
        return nat.RotaryPlan(self._turns.data_ptr(), self._axis.data_ptr(), at, self.num_axes, self.pairs, size,
                              self._adjacent, 1 if inverse else 0, 0), positions

    def rotate(self, query: torch.Tensor, key: torch.Tensor | None = None, *, positions: torch.Tensor,
               inverse: bool = False):
        """Rows [S, n, H, D] ([n, H, D] for one sequence) of bf16 or fp16 turned
        by positions [axes, S, n] (int32 or int64, below 2^31 in magnitude):
        new contiguous tensors, (query, key) or query alone.  Key heads may be fewer.
        ``inverse`` turns back, which is also what a gradient of the rotated rows takes."""

        flat = query.dim() == 3
        if flat:
            query, key = query.unsqueeze(0), None if key is None else key.unsqueeze(0)
        if positions is None:
            raise ValueError("Rotary rows need positions")
        shape, outs, args = query.shape, [], []
        for t, what in ((query, "Rotary queries"), (key, "Rotary keys")):
            if t is None:
                continue
            if t.dim() != 4 or t.shape[3] != self.head_dim or t.shape[:2] != shape[:2] or not t.shape[2]:
                raise ValueError(f"{what}: expected [sequences, tokens, heads, {self.head_dim}], got {tuple(t.shape)}")
            check_rows(t, what)
            if t.dtype != query.dtype:
                raise ValueError("Rotary queries and keys must have one dtype")
        for t in (query, key):
            if t is None:
                args += (None, 0, 0, 0, 0, None)
                continue
            if t.device.type != "cuda":
                raise RuntimeError(f"Rotary positions requires GPU tensors (got {t.device})")
            if t.device != self.device:
                raise RuntimeError(f"Rotary positions: rows must be on the plan's device {self.device}")
            t, a, b, c = nat.rows16(t)
            out = nat.empty_like(t)
            outs.append((t, out))  # (the inputs stay alive until the launch)
            args += (t.data_ptr(), a, b, c, t.shape[2], out.data_ptr())
        struct, held = self.plan(positions, shape[0], shape[1], inverse=inverse)
        if shape[0] and shape[1]:
            nat.call_on(self.device, "uc_rotary", struct, shape[0], shape[1], self.head_dim,
                        nat.dtype_code(query.dtype), *args)
        outs = [out[0] if flat else out for _, out in outs]
        return outs[0] if key is None else tuple(outs)
