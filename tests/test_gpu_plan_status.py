"""The status of plans that follow a plan without enough pages."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import kv_cache
from exl3_intel_arc_quantizer_amd.kv_cache import plan_step


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


@pytest.mark.gpu
def test_tokens_in_a_missing_page_are_reported():
    """Request 1 gets no page in the first step; its next tokens fall into the
    same page, for which the second step takes nothing."""
    tables = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    free = _ints([9])
    first = plan_step(_ints([0, 0]), _ints([3, 4]), tables, free, _ints([0]), page_size=32, max_tokens=7)
    assert int(first.status) == kv_cache.PAGES_RAN_OUT
    second = plan_step(first.lengths, _ints([1, 2]), tables, free, first.taken, page_size=32, max_tokens=3)
    assert second.slots.tolist() == [9 * 32 + 3, -1, -1]
    assert int(second.status) == kv_cache.PAGES_RAN_OUT
    with pytest.raises(RuntimeError, match="pages"):
        second.check()
    # No new token falls into the missing page: nothing to report.
    third = plan_step(first.lengths, _ints([1, 0]), tables, free, first.taken, page_size=32, max_tokens=1)
    assert int(third.status) == 0
    # A full last page takes none of the new tokens, whatever its entry.
    full = plan_step(_ints([32, 0]), _ints([1, 0]), torch.full_like(tables, -1), _ints([4]), _ints([0]), page_size=32,
                     max_tokens=1)
    assert int(full.status) == 0 and full.slots.tolist() == [4 * 32]


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 1024, 1025, 4096])
def test_status_says_whether_all_tokens_have_slots(requests):
    rng = np.random.default_rng(requests)
    page, width = 32, 4
    for hole in (None, 0, requests - 1):
        cached = rng.integers(1, page, requests)
        new = rng.integers(1, 3, requests)
        tables = rng.integers(0, 100, (requests, width))
        if hole is not None:
            tables[hole, 0] = -1
        tokens = int(new.sum())
        plan = plan_step(_ints(cached), _ints(new), _ints(tables), _ints(np.arange(2 * requests)), _ints([0]),
                         page_size=page, max_tokens=tokens)
        assert (int(plan.status) == 0) == bool((plan.slots >= 0).all()) == (hole is None)
