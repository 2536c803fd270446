"""What attention of trees may be off where scores are large: trees of one branch,
which attend what sequences do, in the kernels that are compiled for trees."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd.kv_cache import cache_attention, plan_tree

from . import cache_ref as ref
from .test_gpu_attention_precision import _few, _ints, _tables, _within


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("strength", [8, 16])
@pytest.mark.parametrize("dim, group, new, context", [
    (64, 4, [12, 16], [700, 300]), (64, 4, [130], [2000]), (64, 1, [7, 2], [90, 400]), (128, 8, [4, 9], [900, 1500]),
    (128, 2, [7, 8], [600, 64]), (128, 4, [30, 40, 1], [1000, 2100, 50]), (128, 4, [300], [1700]), (128, 4, [13], [4097]),
    (256, 4, [20, 70], [300, 1200]), (256, 2, [3, 4], [500, 700]), (128, 4, [1000], [1000])])
def test_sharp_scores(dim, group, new, context, strength, dtype):
    rng = np.random.default_rng(dim + strength + len(new))
    page, heads = 64, 2
    pages = sum(-(-n // page) for n in context) + 1
    cache = ref.Cache(pages, page, heads, dim, rng)
    tables = _tables(context, page, -(-max(context) // page), pages, rng)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.normal(size=(starts[-1], heads * group, dim)) * strength).to(dtype).cuda()
    args = torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(context)
    tree = plan_tree(_ints([i - 1 for n in new for i in range(n)]), _ints(starts), _ints(context), max_new=max(new))
    keys, values = (torch.from_numpy(x).cuda() for x in cache.values())
    exact = ref.attention_dense(q, keys, values, page, tables, starts, context, dim ** -0.5, None)
    for hint in (None, max(new), 1):
        _within(cache_attention(q, *args, max_new=hint, trees=tree.masks), exact, dtype, hint == 1 or _few(new, group, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, group, length", [(128, 4, 2), (64, 4, 6), (256, 2, 10), (64, 8, 2), (128, 4, 400), (64, 8, 2500)])
def test_small_trees_keep_the_weights_bits(dim, group, length, dtype):
    """Values of neighbouring positions are opposite and their weights nearly equal,
    so that an output is small beside its terms: a tree of two tokens, of which each
    attends the cached ones and itself."""
    rng = np.random.default_rng(dim + length)
    page = 32
    pages = -(-(length + 1) // page) + 1
    cache = ref.Cache(pages, page, 1, dim, rng)
    cache.codes = np.maximum(cache.codes, -7)
    cache.codes[1, 1::2], cache.scales[1, 1::2] = -cache.codes[1, ::2], cache.scales[1, ::2]
    tables = _tables([length + 1], page, pages, pages, rng)
    q = torch.from_numpy(rng.normal(size=(2, group, dim)) * 0.3).to(dtype)
    held = torch.from_numpy(cache.bytes()).cuda(), _ints(tables)
    tree = plan_tree(_ints([-1, -1]), _ints([0, 2]), _ints([length + 1]), max_new=2)
    keys, values = cache.values()
    # The second token as a sequence whose place the first one's entry has left.
    slots = tables[0][np.arange(length + 1) // page] * page + np.arange(length + 1) % page
    exact = [ref.attention(q[:1].double().numpy(), keys, values, page, tables, [0, 1], [length], dim ** -0.5, None)]
    keys, values = keys.copy(), values.copy()
    keys[slots[length - 1]], values[slots[length - 1]] = keys[slots[length]], values[slots[length]]
    exact.append(ref.attention(q[1:].double().numpy(), keys, values, page, tables, [0, 1], [length], dim ** -0.5, None))
    exact = tuple(np.concatenate(parts) for parts in zip(*exact))
    for hint in (None, 2, 1):
        got = cache_attention(q.cuda(), *held, _ints([0, 2]), _ints([length + 1]), max_new=hint, trees=tree.masks)
        _within(got, exact, dtype, True)
