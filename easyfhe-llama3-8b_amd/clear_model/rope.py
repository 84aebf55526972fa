"""Rotary positions of the clear decoder (reference approx/attention.py:22-70
applies the half layout over whole heads; this one also takes interleaved
pairs, part of a head, and wavelengths scaled for long contexts).

Pair j of a head turns by the angle ``position * w_j`` with
``w_j = theta^(-2j / rotary_dim)``: elements j and j + rotary_dim/2 in the
"half" layout, 2j and 2j + 1 in the "interleaved" one; elements from
rotary_dim on stay as they are.  The gradient is the same turn backwards.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._native import ROPE_ARGS, TYPES

LAYOUTS = ("half", "interleaved")


@dataclass(frozen=True)
class WavelengthScaling:
    """Frequencies for contexts beyond the trained length: waves longer than
    ``original / low`` positions are stretched by ``factor``, waves shorter
    than ``original / high`` are kept, and those between are blended linearly
    in the number of turns over ``original`` positions."""

    factor: float
    low: float
    high: float
    original: int

    def __post_init__(self):
        if not self.factor > 0 or not self.original > 0:
            raise ValueError("the scaling factor and the original length are positive.")
        if not 0 < self.low < self.high:
            raise ValueError("the scaling borders satisfy 0 < low < high.")

    def apply(self, frequency: float) -> float:
        turns = self.original * frequency / (2.0 * math.pi)
        keep = min(1.0, max(0.0, (turns - self.low) / (self.high - self.low)))
        return frequency * (keep + (1.0 - keep) / self.factor)


class RopeTable:
    """The turns per position of every pair of a head, in fp64: made once, and
    laid out once on each device that it is used on."""

    def __init__(self, dim: int, *, rotary_dim: int | None = None, theta: float = 500000.0,
                 layout: str = "half", scaling: WavelengthScaling | None = None):
        rotary = int(dim) if rotary_dim is None else int(rotary_dim)
        if int(dim) < 1 or int(dim) > 1024:
            raise ValueError("a head has 1 to 1024 elements.")
        if rotary < 0 or rotary > int(dim) or rotary % 2:
            raise ValueError("rotary_dim is even and at most the head's dim.")
        if layout not in LAYOUTS:
            raise ValueError(f"layout is one of {LAYOUTS}, got {layout!r}.")
        if layout == "interleaved" and int(dim) % 2:
            raise ValueError("interleaved pairs need an even head.")
        if not theta > 0:
            raise ValueError("theta is positive.")
        self.dim, self.rotary_dim, self.theta = int(dim), rotary, float(theta)
        self.layout, self.scaling = layout, scaling
        w = [self.theta ** (-2.0 * j / rotary) for j in range(rotary // 2)]
        if scaling is not None:
            w = [scaling.apply(x) for x in w]
        self.frequencies = torch.tensor(w, dtype=torch.float64)
        self.interleaved = layout == "interleaved"
        self._turns: dict[torch.device, tuple[torch.Tensor, int]] = {}

    def turns_on(self, device: torch.device) -> int:
        """The address of the turns on the device."""
        held = self._turns.get(device)
        if held is None:
            t = (self.frequencies / (2.0 * math.pi)).to(device)
            # once a device: the copy is there for every stream from here on
            torch.cuda.current_stream(device).synchronize()
            held = self._turns[device] = (t, t.data_ptr())
        return held[1]


def _rope(table: RopeTable, q, k, positions, inverse: bool):
    shape, dtype, dev = q.shape, q.dtype, q.device
    if len(shape) != 4:
        raise ValueError("q is [batch, tokens, heads, dim].")
    b, n, h, d = shape
    if d != table.dim:
        raise ValueError(f"heads have {d} elements, the table is for {table.dim}.")
    kind = TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"rope takes bf16, fp16 and fp32, got {dtype}.")
    if not q.is_cuda or positions.device != dev:
        raise ValueError("q, k and positions are on one GPU.")
    wide = positions.dtype == torch.int64
    if not wide and positions.dtype != torch.int32:
        raise ValueError("positions are int32 or int64.")
    if positions.dim() == 1:
        positions = positions.expand(b, -1)
    if positions.shape != (b, n):
        raise ValueError(f"positions are [{n}] or [{b}, {n}], got {tuple(positions.shape)}.")
    qs, ps = q.stride(), positions.stride()
    if qs[3] != 1 and d > 1:
        q = q.contiguous()
        qs = q.stride()
    qo = q.new_empty(shape)
    if k is None:
        ko, kh, ks, kp, kop = None, 0, (0, 0, 0), 0, 0
    else:
        kshape = k.shape
        if len(kshape) != 4 or kshape[0] != b or kshape[1] != n or kshape[3] != d:
            raise ValueError("k is [batch, tokens, kv heads, dim] with q's batch, tokens and dim.")
        if k.dtype != dtype or k.device != dev:
            raise ValueError("k has q's type and device.")
        ks, kh = k.stride(), kshape[2]
        if ks[3] != 1 and d > 1:
            k = k.contiguous()
            ks = k.stride()
        ko = k.new_empty(kshape)
        kp, kop = k.data_ptr(), ko.data_ptr()
    args = ROPE_ARGS.pack(
        q.data_ptr(), kp, qo.data_ptr(), kop, positions.data_ptr(), table.turns_on(dev), kind,
        wide, b, n, h, kh, d, table.rotary_dim, table.interleaved, inverse, qs[0], qs[1], qs[2],
        ks[0], ks[1], ks[2], ps[0], ps[1])
    _native.call(_native.lib.clear_rope, args, dev.index)
    return qo, ko


def rope(table: RopeTable, q, k=None, *, positions):
    """(q', k') of q [B, T, H, D] and k [B, T, Hk, D] (or None) at the integer
    positions [T] or [B, T].  Any strides; the results are new and contiguous.
    Angles are reduced in fp64, the result is rounded once.  No graph is kept:
    tensors that require gradients go through ``apply_rope``."""
    _native.without_graph("apply_rope", q, k)
    return _rope(table, q, k, positions, False)


def rope_backward(table: RopeTable, dq, dk=None, *, positions):
    """The gradients of ``rope``'s inputs from those of its outputs."""
    return _rope(table, dq, dk, positions, True)


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, positions, q, k):
        ctx.table = table
        ctx.save_for_backward(positions)
        return rope(table, q, k, positions=positions)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        return (None, None) + rope_backward(ctx.table, dq, dk, positions=positions)


def apply_rope(table: RopeTable, q, k, *, positions):
    """``rope`` of both q and k, with gradients."""
    return _Rope.apply(table, positions, q, k)


__all__ = ["RopeTable", "WavelengthScaling", "apply_rope", "rope", "rope_backward"]
