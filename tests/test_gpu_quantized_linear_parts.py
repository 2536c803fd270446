"""The bits that rows of quantized_linear count with: rows whose high parts cancel
in the product, and rows scaled by powers of two."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd.quantized_linear import quantized_linear

from .test_gpu_quantized_linear import _blocks, _given, _tiles

# (rows, in, out, K, type): each kernel and each way it holds two parts of a row.
CASES = [(rows, 256, 384, 4, torch.float16) for rows in (1, 4, 6, 13, 20, 40, 60, 96)]
CASES += [(rows, 512, 256, 3, torch.bfloat16) for rows in (2, 7, 16, 32, 48, 64)]
CASES += [(3, 1024, 256, 6, torch.bfloat16), (100, 1280, 256, 5, torch.float16), (1000, 256, 8192, 2, torch.float16)]

# What an output's error may be of the row's outputs, in norm. A row's halves are
# v and d - v, their weights alike, so the output is that of d, whose transformed
# values are 2^-12 of v's. Errors are of both signs. In those of d they are
#   - of two parts, 2^-22 / sqrt(3) of a value of v for each half: 2^-10;
#   - of the transform in float32, eight steps of 2^-24 each: 2^-10;
#   - of 2 k sums, 2^-24 of partial ones of sqrt(k / 2) values of v: 2^-12 sqrt(2 k),
#     2^-6.3 for the largest k here;
#   - of the output, UNIT at most.
# One part is off by half a place, 2^-12 to 2^-11 of a value: as much as d.
LIMIT = 1 / 8


def _cancelling(rows, k, n, K, dtype):
    """(x, words, su, sv): v in the first half, d - v in the second."""
    x, words, su, sv = _given(rows, k, n, K, dtype, seed=3)
    half, rng = k // 2, np.random.default_rng(rows + k)
    words[half // 16:], su[half:] = words[:half // 16], su[:half]
    x[:, :half:8] = 0
    x[:, half:] = -x[:, :half]
    # An eighth of the channels hold d, so these are sqrt(8) larger than its
    # transformed values.
    size = 2.0 ** -12 * 8 ** 0.5 * x.double().norm(dim=1, keepdim=True).numpy() / k ** 0.5
    x[:, half::8] = torch.from_numpy(rng.normal(size=(rows, half // 8)) * size).to(dtype)
    return x, words, su, sv * 64                         # (outputs of 2^-7 or so)


def _product(x, words, su, sv, K, cb, parts):
    """In 64 bits, but with the transformed rows in so many float16 parts (0: whole)."""
    z = _blocks(x.double().numpy() * su.double().numpy())
    if parts:
        power = 2.0 ** (11 - np.ceil(np.log2(np.abs(z).max(1, keepdims=True))))
        high = (z * power).astype(np.float16).astype(np.float64)
        low = (z * power - high).astype(np.float16).astype(np.float64)
        z = (high + low * (parts - 1)) / power
    return _blocks(z @ _tiles(words.numpy(), K, cb)) * sv.double().numpy()


def _error(got, want):
    """The largest of the rows' errors, in norm."""
    return (np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)).max()


@pytest.mark.parametrize("rows, k, n, K, dtype", [case for case in CASES if case[0] < 1000])
def test_one_part_would_show(rows, k, n, K, dtype):
    given = _cancelling(rows, k, n, K, dtype)
    want = _product(*given, K, K % 3, 0)
    one, two = (_product(*given, K, K % 3, parts) for parts in (1, 2))
    errors = np.linalg.norm(one - want, axis=1) / np.linalg.norm(want, axis=1)
    assert errors.min() > 3 * LIMIT and _error(two, want) < LIMIT / 32


@pytest.mark.gpu
@pytest.mark.parametrize("rows, k, n, K, dtype", CASES)
def test_rows_count_with_two_parts(rows, k, n, K, dtype):
    given = _cancelling(rows, k, n, K, dtype)
    got = quantized_linear(*(t.cuda() for t in given), K, K % 3)
    assert _error(got.double().cpu().numpy(), _product(*given, K, K % 3, 0)) < LIMIT


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 6, 14, 40, 130])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_power_of_two_scales_a_row(rows, dtype):
    """Exactly, where the row's values and its results keep their places; the other
    rows stay as they are."""
    x, words, su, sv = (t.cuda() for t in _given(rows, 384, 256, 4, dtype))
    x[x.abs() < 2.0 ** -6] = 0
    power = 2.0 ** -8 if dtype == torch.float16 else 2.0 ** 70
    scaled = x.clone()
    scaled[-1] = x[-1].double().mul(power).to(dtype)
    assert torch.equal(scaled[-1].double(), x[-1].double() * power) and scaled[-1].any()
    want, got = quantized_linear(x, words, su, sv, 4), quantized_linear(scaled, words, su, sv, 4)
    assert torch.equal(got[:-1], want[:-1])
    # A float16 result under 2^-14 is off by half a place, 2^-25, and the larger one
    # by half of one of its own, which 256 times smaller is 2^-26.
    off, whole = (got[-1].double() - want[-1].double() * power).abs(), got[-1].double().abs() >= 2.0 ** -14
    assert whole.any() and not off[whole].any()
    assert (off <= (1.5 * 2.0 ** -25 if dtype == torch.float16 else 0.0)).all()
