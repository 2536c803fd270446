"""Requests of more drafted tokens than the masks of their trees have bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import _native
from exl3_intel_arc_quantizer_amd.kv_cache import accept_drafts

from .test_gpu_trees import _accepted, _forest, _ints


def _given(new, ids, seed):
    rng = np.random.default_rng(seed)
    tokens, choices = (rng.integers(0, ids, sum(new)).tolist() for _ in range(2))
    return _forest(new, rng, 30), tokens, choices, [n + int(rng.integers(0, 99)) for n in new], rng


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("most, new", [
    (1, [65, 5, 64, 66, 0, 200]), (64, [300, 64, 65]), (65, [129, 128, 300, 1]), (200, [257, 256, 30]), (1024, [1025, 1024, 2500]),
    (None, [1025, 1024, 40, 2500])])
def test_long_requests_are_accepted_as_runs(most, new, dtype):
    """Branching parents beside ordinary trees; a few ids, so that choices are met."""
    bits = 64 * -(-(most or 1024) // 64)
    for ids in (1, 2, 3):
        parents, tokens, choices, lengths, rng = _given(new, ids, sum(new) + ids)
        certain = [int(c) for c in rng.choice([1, 3, 70, 1 << 20], len(new))]
        at = np.concatenate([[0], np.cumsum(new)])
        counted = [p for r, n in enumerate(new) for p in (range(-1, n - 1) if n > bits else parents[at[r]:at[r + 1]])]
        args = _ints(tokens, dtype), _ints(choices, dtype), _ints(parents), _ints(at), _ints(lengths)
        for given in (None, certain):
            got = accept_drafts(*args, certain=None if given is None else _ints(given), max_new=most)
            places, kept, after = _accepted(new, lengths, counted, tokens, choices, given or [1] * len(new))
            assert got.places.tolist() == places and got.lengths.tolist() == kept and got.next.tolist() == after


def test_refuses_bounds_past_the_masks():
    one, many = torch.zeros(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for most in (0, -3, 1025):
        with pytest.raises(ValueError, match="max_new"):
            accept_drafts(many, many, many, one, one, max_new=most)
    lib = _native.load_library()
    for words in (0, 17):
        assert lib.exl3_accept_trees(None, None, 0, None, None, None, None, 1, 4, words, None, None, None, None) == 1
        assert b"words" in lib.exl3_last_error()
