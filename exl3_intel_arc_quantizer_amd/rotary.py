"""Rotary positions of queries and keys on the GPU (``exl3_rotary``, HIP).

Every pair of a head's values turns by an angle of its own per position:
``apply_rotary`` takes the angles' frequencies from ``rotary_frequencies`` (or
any float64 tensor a model brings) and turns queries and keys in one launch,
with the gradient where torch follows them. ``kv_cache.append_tokens`` does the
same on the way into a cache.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

from . import _native
from .hadamard import records

LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0,
                       scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, fast: float = 32.0,
                       slow: float = 1.0, device="cuda") -> Tuple[torch.Tensor, float]:
    """Frequencies (radians a position) of the ``rotary_dim / 2`` pairs, as a
    float64 tensor on ``device``, and the magnitude that turned values take:
    ``base ** (-2 i / rotary_dim)``, scaled for contexts ``factor`` times
    longer than the model was trained on:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: base times ``factor ** (d / (d - 2))``, which leaves the
      fastest pair as it is and divides the slowest by ``factor``;
    * ``"ramp"``: pairs that turn more than ``fast`` times in
      ``original_length`` positions stay, those that turn less than ``slow``
      times are divided by ``factor``, those between are blended linearly in
      the pair's index; magnitude ``0.1 ln(factor) + 1``.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError(f"needs base > 1 and factor >= 1, got {base} and {factor}")
    if scaling == "base":
        if rotary_dim < 4:
            raise ValueError("base scaling needs rotary_dim >= 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        if not original_length or original_length < 1 or not fast > slow > 0:
            raise ValueError("ramp scaling needs original_length and fast > slow > 0")

        def pair_of(turns: float) -> float:
            return (rotary_dim * math.log(original_length / (turns * 2 * math.pi))
                    / (2 * math.log(base)))

        low, high = math.floor(pair_of(fast)), math.ceil(pair_of(slow))
        low, high = max(low, 0), min(high, rotary_dim - 1)
        divided = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - divided) + freq / factor * divided
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f'scaling must be None, "linear", "base" or "ramp", got {scaling!r}')
    return freq.to(device), magnitude


def rotary_axes(sections: Sequence[int], *, interleaved: bool = False,
                device="cuda") -> torch.Tensor:
    """The axis of every pair, int32 on ``device``, for models whose tokens have
    several positions (time, height and width): ``sections[a]`` pairs of axis a,
    one axis after the other, or (``interleaved``) in turn, each round a pair of
    every axis that has some left."""
    sections = [int(n) for n in sections]
    if not sections or min(sections) < 0 or not sum(sections):
        raise ValueError(f"sections must hold pairs of each axis, got {sections}")
    if interleaved:
        axes = [a for turn in range(max(sections)) for a, n in enumerate(sections) if turn < n]
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(axes, dtype=torch.int32, device=device)


class _Rotary(torch.autograd.Function):
    """The rotation is linear: its gradient turns back, its tangent turns the
    same way. Both can be differentiated again."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, axes, layout, magnitude, inverse):
        # Saved, so that torch refuses a backward pass after they were written to.
        ctx.save_for_backward(positions, frequencies, axes)
        ctx.save_for_forward(positions, frequencies, axes)
        ctx.given = (layout, magnitude, inverse)
        ctx.two = k is not None
        ctx.shapes = q.shape, k.shape if ctx.two else None
        ctx.set_materialize_grads(False)
        q_out, k_out = _native.rotary(q, k, positions, frequencies, layout, magnitude, inverse,
                                      axes=axes)
        return (q_out, k_out) if ctx.two else (q_out,)

    @staticmethod
    def backward(ctx, *grads):
        layout, magnitude, inverse = ctx.given
        out = _turned(grads[0], grads[1] if ctx.two else None, *ctx.saved_tensors, layout,
                      magnitude, not inverse)
        return (*out, None, None, None, None, None, None)

    @staticmethod
    def jvp(ctx, *tangents):
        layout, magnitude, inverse = ctx.given
        q, k = _turned(tangents[0], tangents[1], *ctx.saved_tensors, layout, magnitude, inverse)
        if not ctx.two:
            return (q,)
        # torch asks for a tangent of every output: that of an input without one is 0.
        return tuple(other.new_zeros(shape) if x is None else x
                     for x, other, shape in ((q, k, ctx.shapes[0]), (k, q, ctx.shapes[1])))


def _turned(q, k, positions, frequencies, axes, layout, magnitude, inverse):
    """Both turned; either may be None (and stays None)."""
    if q is None:
        return (None, None) if k is None else \
            (None, _turned(k, None, positions, frequencies, axes, layout, magnitude, inverse)[0])
    # A gradient may arrive expanded or with any strides.
    q, k = (x if x is None or x.stride(-1) == 1 else x.contiguous() for x in (q, k))
    if records(q) or (k is not None and records(k)):
        out = _Rotary.apply(q, k, positions, frequencies, axes, layout, magnitude, inverse)
        return out if k is not None else (out[0], None)
    return _native.rotary(q, k, positions, frequencies, layout, magnitude, inverse, axes=axes)


def layout_code(layout: str) -> int:
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    return LAYOUTS[layout]


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 frequencies: torch.Tensor, *, layout: str = "half", magnitude: float = 1.0,
                 out: Optional[tuple] = None, axes: Optional[torch.Tensor] = None) -> tuple:
    """(q, k) turned by their positions, as new contiguous tensors or into
    ``out`` (a pair like q and k: the inputs themselves, or tensors that share no
    memory with them or each other), where torch records neither the inputs nor
    ``out``.

    q and k are (tokens, heads, head_dim) of one type, float32, float16 or
    bfloat16, with any strides of tokens and heads; k may be None, and is then
    None in the result. ``positions`` are int32 or int64 (tokens,),
    ``frequencies`` float64 of up to head_dim / 2 pairs: (i, i + pairs) for
    layout ``"half"``, (2 i, 2 i + 1) for ``"interleaved"``; the values past
    the pairs are copied; frequencies have no gradient. Angles are taken in 64
    bits and products in 32, so positions in the millions are as exact as the
    first ones.

    With ``axes`` (int32, one of every pair: ``rotary_axes``) ``positions`` are
    (axes, tokens), and pair i turns by its frequency times the position on axis
    ``axes[i]``; pairs whose axis is not one of those do not turn."""
    code = layout_code(layout)
    if isinstance(frequencies, torch.Tensor) and records(frequencies):
        raise RuntimeError("apply_rotary has no gradient of frequencies: detach them")
    recorded = records(q) or (k is not None and records(k))
    if out is not None and (recorded or any(isinstance(t, torch.Tensor) and records(t)
                                            for t in out)):
        raise RuntimeError("apply_rotary: out cannot be given where torch records it or the inputs")
    if recorded:
        return _turned(q, k, positions, frequencies, axes, code, magnitude, False)
    return _native.rotary(q, k, positions, frequencies, code, magnitude, False, out, axes)
