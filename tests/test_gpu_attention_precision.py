"""What attention's results may be off, request by request, where scores are
large and where calls choose different kernels for the same rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd.kv_cache import cache_attention

from . import cache_ref as ref

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _tables(lengths, page, width, pages, rng):
    ids, at = rng.permutation(pages), 0
    tables = np.full((len(lengths), width), -1)
    for r, n in enumerate(lengths):
        used = -(-n // page)
        tables[r, :used] = ids[at:at + used]
        at += used
    return tables


def _tolerance(want, spread, basis, reach, dtype, few):
    """Queries count with 22 bits whatever their type, so scores (sums of up to
    256 products in float32) are off by at most 2^-18 of |q| |k| scale and move
    a weight by that share, numerator and sum. Weights count with 22 bits in
    requests of few rows to a kv head, with 11 beyond (2^-11 in numerator and
    sum each); float32 sums 2^-17. Then the output's own rounding."""
    weights = 2.0 ** -17 + np.where(few, 0.0, 2.0 ** -10)
    return UNIT[dtype] * np.abs(want) + (2 * 2.0 ** -18 * reach + weights) * spread + 2.0 ** -17 * basis + 2.0 ** -24


def _few(new, group, dim):
    """By row: whether its request has few rows to a kv head."""
    return np.repeat(np.asarray(new) * group <= (32 if dim == 256 else 16), new)[:, None, None]


def _within(got, exact, dtype, few):
    want, spread, basis, reach = exact
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want) - _tolerance(want, spread, basis, reach, dtype, few)
    assert not (off > 0).any(), f"{np.nanmax(off)} too far, of {np.nanmax(np.abs(want))}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("strength", [8, 16])
@pytest.mark.parametrize("dim, group, new, context", [
    (64, 4, [12, 16], [700, 300]), (64, 4, [130], [2000]), (128, 8, [4, 9], [900, 1500]), (128, 4, [300], [1700]),
    (256, 4, [20, 70], [300, 1200]), (128, 4, [1100], [1100])])
def test_sharp_scores_of_many_rows(dim, group, new, context, strength, dtype):
    """Scores of tens: an error of a score is one of its weight, many times the
    output's own rounding if queries have fewer bits than their type's sums."""
    rng = np.random.default_rng(dim + strength)
    page, heads = 64, 2
    pages = sum(-(-n // page) for n in context) + 1
    cache = ref.Cache(pages, page, heads, dim, rng)
    tables = _tables(context, page, -(-max(context) // page), pages, rng)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.normal(size=(starts[-1], heads * group, dim)) * strength).to(dtype).cuda()
    args = torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(context)
    keys, values = (torch.from_numpy(x).cuda() for x in cache.values())
    exact = ref.attention_dense(q, keys, values, page, tables, starts, context, dim ** -0.5, None)
    for hint in (None, max(new), 1):
        _within(cache_attention(q, *args, max_new=hint), exact, dtype, hint == 1 or _few(new, group, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim, group, length", [
    (128, 4, 2), (64, 4, 6), (256, 2, 10), (64, 8, 2), (128, 4, 400), (64, 8, 2500)])
def test_a_single_request_of_few_rows_among_padding(dim, group, length, dtype):
    """One token of one request, in a step padded to 64 rows or with a bound of
    64 new tokens: the rows that it has, not those it might have, say how many
    bits its weights count with. Values of neighbouring positions are opposite
    and their weights nearly equal, so that an output is small beside its terms
    and their errors stand out."""
    rng = np.random.default_rng(dim + length)
    page = 32
    pages = -(-length // page) + 1
    cache = ref.Cache(pages, page, 1, dim, rng)
    cache.codes = np.maximum(cache.codes, -7)
    cache.codes[1, 1::2], cache.scales[1, 1::2] = -cache.codes[1, ::2], cache.scales[1, ::2]
    tables = _tables([length], page, pages, pages, rng)
    q = torch.from_numpy(rng.normal(size=(64, group, dim)) * 0.3).to(dtype)
    exact = ref.attention(q[:1].double().numpy(), *cache.values(), page, tables, [0, 1], [length], dim ** -0.5, None)
    held = torch.from_numpy(cache.bytes()).cuda(), _ints(tables)
    alone = cache_attention(q[:1].cuda(), *held, _ints([0, 1]), _ints([length]), max_new=1)
    _within(alone, exact, dtype, True)
    for rows, hint in ((64, None), (64, 64), (64, 1), (1, 64), (2, 2)):
        got = cache_attention(q[:rows].cuda(), *held, _ints([0, 1]), _ints([length]), max_new=hint)
        _within(got[:1], exact, dtype, True)
        assert not got[1:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group, new, window", [
    (64, 4, [1, 4, 5, 0, 70], None), (128, 16, [1, 2, 1, 3], 40), (128, 4, [1, 33, 4, 200], None),
    (256, 16, [1, 2, 3, 2], None), (256, 5, [6, 7, 1, 60], 33), (64, 1, [16, 17, 1, 300], 100)])
def test_bits_of_each_request(dim, group, new, window, dtype):
    """Requests of few rows keep the weights' bits beside those of many."""
    rng = np.random.default_rng(dim + group)
    page, heads = 32, 2
    context = [n + c for n, c in zip(new, (3, 700, 0, 90, 400))]
    pages = sum(-(-n // page) for n in context) + 1
    cache = ref.Cache(pages, page, heads, dim, rng)
    tables = _tables(context, page, -(-max(context) // page) + 1, pages, rng)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.normal(size=(starts[-1], heads * group, dim)) * 3).to(dtype)
    args = torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(context)
    exact = ref.attention(q.double().numpy(), *cache.values(), page, tables, starts, context, dim ** -0.5, window)
    for hint in (None, max(new)):
        _within(cache_attention(q.cuda(), *args, window=window, max_new=hint), exact, dtype, _few(new, group, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_reaches_exactly_its_rows(dim, new):
    """A finite number where a NaN is due is as wrong as the reverse."""
    rng = np.random.default_rng(dim)
    page, context = 32, [90, 130]
    cache = ref.Cache(9, page, 1, dim, rng)
    tables = _tables(context, page, 5, 9, rng)
    for r, at, which, part in ((0, 89, 1, 1), (1, 120, 0, 0), (1, 127, 1, 0)):
        cache.scales[which][tables[r][at // page] * page + at % page, 0, part] = np.nan
    starts = np.array([0, new, 2 * new])
    q = torch.from_numpy(rng.normal(size=(2 * new, 2, dim))).half()
    for window in (None, 3):
        exact = ref.attention(q.double().numpy(), *cache.values(), page, tables, starts, context, dim ** -0.5, window)
        got = cache_attention(q.cuda(), torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts),
                              _ints(context), window=window)
        assert np.isnan(exact[0]).any()
        _within(got, exact, torch.float16, _few([new, new], 2, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 300])
def test_requests_that_claim_the_same_rows(rows):
    """Starts that are no prefix sums: each row is one claimant's result, or 0."""
    rng = np.random.default_rng(rows)
    cache = ref.Cache(3, 32, 1, 64, rng)
    pages, tables = torch.from_numpy(cache.bytes()).cuda(), _ints([[0, 1], [2, 5], [1, -3]])
    q = torch.from_numpy(rng.normal(size=(rows, 2, 64))).half().cuda()
    got = cache_attention(q, pages, tables, _ints([0, rows, 0, rows]), _ints([64, 32, 60]))
    assert torch.isfinite(got).all()
    most = cache.values()[1]
    assert got.abs().max() <= np.abs(most).max() * (1 + 2.0 ** -9)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("most", [1, 3, 40])
def test_as_many_requests_as_a_call_takes(dim, most):
    """4096 requests, some empty, of up to `most` tokens of up to 70 positions."""
    rng = np.random.default_rng(most)
    page, requests = 32, 4096
    new = rng.integers(0, most + 1, requests)
    if most > 3:
        new[rng.random(requests) < 0.9] = 0
    context = new + rng.integers(0, 30, requests)
    pages = int((-(-context // page)).sum()) + 1
    cache = ref.Cache(pages, page, 1, dim, rng)
    tables = _tables(context, page, 3, pages, rng)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.normal(size=(starts[-1] + 2, 2, dim)) * 2).to(torch.bfloat16)
    got = cache_attention(q.cuda(), torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(context))
    exact = ref.attention(q.double().numpy(), *cache.values(), page, tables, starts, context, dim ** -0.5, None)
    few = np.concatenate([_few(new, 2, dim), np.ones((2, 1, 1), bool)])
    _within(got, exact, torch.bfloat16, few)
    assert not got[starts[-1]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, new", [(64, 1), (64, 100), (128, 1), (128, 12), (256, 1), (256, 30)])
def test_scales_of_zero_and_below(dim, new, dtype):
    """A scale of 0 is the mean of what is attended, a negative one prefers the
    smallest products."""
    rng = np.random.default_rng(dim + new)
    page, context = 32, 150
    cache = ref.Cache(6, page, 1, dim, rng)
    tables = _tables([context], page, 5, 6, rng)
    q = torch.from_numpy(rng.normal(size=(new, 2, dim)) * 2).to(dtype)
    args = torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints([0, new]), _ints([context])
    for scale in (0.0, -0.0, -0.1):
        *exact, reach = ref.attention(q.double().numpy(), *cache.values(), page, tables, [0, new], [context], scale, None)
        got = cache_attention(q.cuda(), *args, scale=scale)
        _within(got, (*exact, np.abs(reach)), dtype, _few([new], 2, dim))
