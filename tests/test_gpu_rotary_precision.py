"""Rotary positions to the last float32 places, element by element."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_frequencies


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim, first", [(128, 0), (64, 131_000), (20, 4_000_000)])
def test_one_rounding_of_cosine_and_sine(dim, first, layout):
    """Cosine and sine, times the magnitude, are float32 values nearest to those
    of the exact angle: 2^-24 of themselves. So are the two products, and their
    sum: (1 + 1 + 1) 2^-24 of |x1 c| + |x2 s|. The angle, at most 2^22 turns in 64
    bits here and in the reference, is off by 2^-28 radians."""
    g = torch.Generator().manual_seed(dim)
    tokens, magnitude = 500, 1.2
    x = torch.randn(tokens, 8, dim, generator=g)
    x *= torch.exp2(torch.randint(-12, 1, x.shape, generator=g).float())  # neighbours of other sizes
    freq, _ = rotary_frequencies(dim, base=500000.0, device="cpu")
    at = torch.arange(tokens) * 3 + first
    got, _ = apply_rotary(x.cuda(), None, at.cuda(), freq.cuda(), layout=layout, magnitude=magnitude)
    n = dim // 2
    a, b = (np.s_[..., :n], np.s_[..., n:]) if layout == "half" else (np.s_[..., 0::2], np.s_[..., 1::2])
    angle = (at.double()[:, None] * freq).numpy()[:, None]
    m = float(np.float32(magnitude))
    c, s = np.cos(angle) * m, np.sin(angle) * m
    x64, y = x.double().numpy(), got.cpu().double().numpy()
    x1, x2 = x64[a], x64[b]
    for value, want, terms in ((y[a], x1 * c - x2 * s, np.abs(x1 * c) + np.abs(x2 * s)),
                               (y[b], x2 * c + x1 * s, np.abs(x2 * c) + np.abs(x1 * s))):
        bound = 3 * 2.0 ** -24 * (1 + 2.0 ** -20) * terms + 2.0 ** -28 * m * (np.abs(x1) + np.abs(x2)) + 2.0 ** -140
        assert (np.abs(value - want) <= bound).all()
