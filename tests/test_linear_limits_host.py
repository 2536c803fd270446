"""Sizes that a launch of quantized_linear cannot take are refused."""

from __future__ import annotations

import pytest

from exl3_intel_arc_quantizer_amd import _native


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("rows, k, taken", [
    (1 << 22, 4096, True), (1 << 22, 16384, True), ((1 << 22) - 1, 16512, True), (1 << 22, 16512, False), (1 << 22, 1 << 24, False)])
def test_launches_have_fewer_than_32_bits_of_threads(rows, k, taken, kind):
    lib = _native.load_library()
    size = lib.exl3_linear_workspace(rows, k, 128, kind)
    assert size > 0 if taken else size == -1
    if not taken:
        assert lib.exl3_linear(None, 0, rows, kind, None, None, None, 0, k, 128, 4, 2, None, None, 1 << 62, None) == 1
        assert b"bad sizes" in lib.exl3_last_error()
