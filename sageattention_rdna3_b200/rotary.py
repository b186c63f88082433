"""Rotary positions with one or several axes, in front of ``sageattn``.

Text has one axis, a picture two or three (frame, row, column), a video three: each axis turns some of the pairs of a
head.  The reference leaves the rotation to the model; here q and k take one launch together, and the
gradient another:

    rope = rotary_axes(128, (32, 48, 48), interleaved=True)       # kept: the frequencies on the device
    q, k = apply_rotary(q, k, positions, rope, tensor_layout="NHD")     # positions: [S, 3]
    o = sageattn(q, k, v, tensor_layout="NHD")
"""
from __future__ import annotations

import decimal
import functools
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _native
from .core import _LAYOUT_CODE

MAX_AXES = 4


@dataclass
class RotaryAxes:
    """The frequencies of every pair on a device, made by :func:`rotary_axes`."""
    head_dim: int
    axes: Tuple[int, ...]       # widths: values of a head that each axis turns
    interleaved: bool
    freq: torch.Tensor          # [pairs] int64: turns per position in units of 2^-64
    axis: torch.Tensor          # [pairs] int32

    @property
    def n_axes(self) -> int:
        return len(self.axes)

    @property
    def rotary_dim(self) -> int:
        return sum(self.axes)


@functools.lru_cache(maxsize=8)
def _pi(digits: int) -> decimal.Decimal:
    """pi to `digits` digits, by the arithmetic-geometric mean (Gauss, Legendre)."""
    with decimal.localcontext(decimal.Context(prec=digits + 10)):
        a, b, t, p = decimal.Decimal(1), decimal.Decimal("0.5").sqrt(), decimal.Decimal("0.25"), 1
        for _ in range(digits.bit_length() + 1):              # twice the digits each time
            mean = (a + b) / 2
            a, b, t, p = mean, (a * b).sqrt(), t - p * (a - mean) ** 2, 2 * p
        return (a + b) ** 2 / (4 * t)


def _turn_units(frequencies) -> list:
    """Frequencies in radians per position (decimals) as turns in units of 2^-64, the nearest one, as int64 holds them."""
    digits = 50 + max(0, max(f.adjusted() for f in frequencies))      # whole turns are taken off: 20 digits are left, and some
    with decimal.localcontext(decimal.Context(prec=digits)):
        per_radian = 2 ** 63 / _pi(digits)
        units = [int((f * per_radian).to_integral_value()) % 2 ** 64 for f in frequencies]
    return [u - 2 ** 64 if u >= 2 ** 63 else u for u in units]


def rotary_axes(head_dim: int, axes: Union[int, Sequence[int]], base: Union[float, Sequence[float]] = 10000.0,
                interleaved: bool = False, inv_freq: Optional[Sequence[float]] = None,
                device: Union[torch.device, int, str, None] = None) -> RotaryAxes:
    """The table of :func:`apply_rotary` and ``paged_kv_append``.

    axes: how many values of a head each axis turns, e.g. ``(32, 48, 48)`` (even numbers, 1 to 4 of them; their sum is a
    multiple of 16 and at most ``head_dim``; the values behind them stay as they are).  Pair i of an axis of width w has the
    frequency ``base ** (-2 i / w)`` radians per position; ``base`` may be one number per axis, and ``inv_freq`` (one
    number per pair, the pairs of axis 0 first) takes its place.  Pairs are ``(x[i], x[i + rotary_dim / 2])``, or
    neighbours ``(x[2i], x[2i + 1])`` with ``interleaved``.  A frequency is kept as the nearest of 2^64 parts
    of a turn: the angle at position p is off by at most p * 2^-65 turns for that (at 2^40 positions 1.9e-7 radians)."""
    widths = (axes,) if isinstance(axes, int) else tuple(int(w) for w in axes)
    assert head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}."
    assert 1 <= len(widths) <= MAX_AXES, f"1 to {MAX_AXES} axes, got {len(widths)}."
    assert all(w > 0 and w % 2 == 0 for w in widths), f"axes must be positive even widths, got {widths}."
    total = sum(widths)
    assert total % 16 == 0 and total <= head_dim, (
        f"the axes must add up to a multiple of 16 that is at most head_dim, got {total}.")
    if inv_freq is None:
        bases = [float(base)] * len(widths) if isinstance(base, (int, float)) else [float(b) for b in base]
        assert len(bases) == len(widths) and all(b > 0 for b in bases), "base must be positive: one number, or one per axis."
        with decimal.localcontext(decimal.Context(prec=40)):
            values = []
            for b, w in zip(bases, widths):                  # (powers by products: a power of its own for each took 2 ms)
                step, f = decimal.Decimal(b) ** (decimal.Decimal(-2) / w), decimal.Decimal(1)
                for _ in range(w // 2):
                    values.append(f)
                    f = f * step
    else:
        values = [decimal.Decimal(float(f)) for f in inv_freq]
        assert len(values) == total // 2, f"inv_freq must have one number per pair ({total // 2}), got {len(values)}."
    assert all(f.is_finite() for f in values), "frequencies must be finite."
    freq = _turn_units(values)
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else (
        torch.device("cuda", device) if isinstance(device, int) else torch.device(device))
    return RotaryAxes(head_dim, widths, bool(interleaved), torch.tensor(freq, dtype=torch.int64).to(dev),
                      torch.tensor([a for a, w in enumerate(widths) for _ in range(w // 2)], dtype=torch.int32).to(dev))


def _vector_aligned(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it that 16-byte loads can read."""
    unit = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in t.stride()[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary: RotaryAxes,
                 tensor_layout: str = "HND") -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q and k with every pair turned by its frequency times the token's position on the pair's axis.

    q: ``[B,H,S,D]`` ("HND") or ``[B,S,H,D]`` ("NHD"), fp16 / bf16 / fp32; k likewise with its own number of heads, or
    None (then only q is returned).  positions: int32 or int64 on the device, ``[S]`` or ``[B,S]`` for one axis, else
    ``[S, axes]`` or ``[B, S, axes]``; any integers, negative ones too.  Returns new tensors; the arithmetic is fp32 with
    one rounding at the end.  Differentiable in q and k (reverse mode, any order); the result of one that needs no gradient needs
    none.  Forward and backward can be captured in one
    CUDA graph; as with every operator of torch, no graph of the same leaves that was recorded outside may be alive then: its
    nodes accumulate on their own stream, which a capture cannot join."""
    assert isinstance(rotary, RotaryAxes), "rotary must come from rotary_axes()."
    module = _native.load_module()
    if not torch.compiler.is_compiling():
        got = module.rotary_plain(q, k, positions, rotary.freq, rotary.axis, len(rotary.axes), rotary.interleaved, rotary.head_dim, tensor_layout)
        if got is not None:                  # None: not a plain call, or one that the checks below refuse
            return got
    assert q.dtype in (torch.float16, torch.bfloat16, torch.float32), "Input tensors must be fp16, bf16, or fp32."
    assert tensor_layout in _LAYOUT_CODE, f"tensor_layout must be 'HND' or 'NHD', got {tensor_layout!r}."
    assert q.dim() == 4 and q.size(3) == rotary.head_dim, f"q must be 4-D with head_dim {rotary.head_dim}, got {tuple(q.shape)}."
    seq_dim = 2 if tensor_layout == "HND" else 1
    B, S = q.size(0), q.size(seq_dim)
    if k is not None:
        assert k.device == q.device and k.dtype == q.dtype, "q and k must have the same device and dtype."
        assert k.dim() == 4 and k.size(3) == q.size(3) and k.size(0) == B and k.size(seq_dim) == S, (
            "q and k must have the same batch, length and head_dim (call twice for different lengths).")
    assert rotary.freq.device == q.device, "the rotary table is on another device than q."
    assert positions.device == q.device and positions.dtype in (torch.int32, torch.int64), (
        "positions must be int32 or int64 on the device of q.")
    n = rotary.n_axes
    if n == 1 and tuple(positions.shape) in ((S,), (B, S)):
        positions = positions.unsqueeze(-1)
    assert tuple(positions.shape) in ((S, n), (B, S, n)), (
        f"positions must be {'[S] or [B, S]' if n == 1 else '[S, axes] or [B, S, axes]'} with S = {S} and {n} axes, "
        f"got {tuple(positions.shape)}.")
    assert q.is_cuda, "Input tensors must be on a CUDA device."
    if n > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    out = _native.load_ops().rotary(q, k, positions, rotary.freq, rotary.axis, int(rotary.interleaved), _LAYOUT_CODE[tensor_layout], 0)
    return out[0] if k is None else (out[0], out[1])
