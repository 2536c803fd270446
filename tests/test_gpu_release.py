"""Pages that come back to a stack with fewer places for them."""

from __future__ import annotations

import numpy as np
import pytest

from exl3_intel_arc_quantizer_amd.kv_cache import plan_step, release_pages

from .test_gpu_trees import _ints


@pytest.mark.gpu
@pytest.mark.parametrize("requests, width", [(1, 4), (5, 7), (90, 40), (3000, 2)])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.99, 1.0, 1.5])
def test_pages_without_a_place_stay_in_their_rows(requests, width, share):
    rng = np.random.default_rng(requests + width)
    page = 32
    before = rng.integers(0, width * page + 1, requests)
    after = np.minimum(before, rng.integers(0, page + 1, requests))
    tables = rng.permutation(requests * width).reshape(requests, width)
    tables[rng.random(tables.shape) < 0.1] = -1
    entries = [(r, p) for r in range(requests) for p in range(-(-after[r] // page), -(-before[r] // page)) if tables[r, p] >= 0]
    taken = int(share * len(entries))
    # As many free entries as were taken, or fewer: those past the end have no place.
    for free_count in (taken + 3, max(taken - 2, 0)):
        free = np.arange(free_count) + 10 ** 6
        want_tables, want_free, top = tables.copy(), free.copy(), taken - len(entries)
        for rank, (r, p) in enumerate(entries):
            if 0 <= top + rank < free_count:
                want_free[top + rank] = tables[r, p]
                want_tables[r, p] = -1
        got_tables, got_free = _ints(tables), _ints(free)
        left = release_pages(_ints(before), _ints(after), got_tables, got_free, _ints([taken]), page_size=page)
        assert int(left) == max(top, 0)
        assert np.array_equal(got_tables.cpu().numpy(), want_tables) and np.array_equal(got_free.cpu().numpy(), want_free)
        # Every page is still known to one of the two.
        held = np.concatenate([got_tables.cpu().numpy().ravel(), got_free.cpu().numpy()[max(top, 0):taken]])
        assert set(tables[tables >= 0]) <= set(held)


@pytest.mark.gpu
def test_a_prefilled_table_gives_back_what_was_taken():
    """Pages 10 and 11 are the caller's own; a step takes 0 and 1 behind them."""
    tables, free = _ints([[10, 11, -1, -1, -1]]), _ints([0, 1, 2])
    plan = plan_step(_ints([64]), _ints([40]), tables, free, _ints([0]), page_size=32, max_tokens=40)
    plan.check()
    assert tables.tolist() == [[10, 11, 0, 1, -1]]
    left = release_pages(plan.lengths, _ints([0]), tables, free, plan.taken, page_size=32)
    assert int(left) == 0 and tables.tolist() == [[10, 11, -1, -1, -1]] and free.tolist() == [0, 1, 2]
