"""The 4-bit attention cache: step plans, writes, reads and attention against
their 64-bit definitions."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import kv_cache
from exl3_intel_arc_quantizer_amd.kv_cache import (append_tokens, cache_attention, cache_pages, plan_step,
                                                   read_tokens)
from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_frequencies

from . import cache_ref as ref

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------- plans

@pytest.mark.gpu
@pytest.mark.parametrize("requests, width, page, most_cached, most_new, pad", [
    (1, 1, 32, 0, 1, 0), (1, 40, 256, 5000, 1, 7), (3, 9, 32, 200, 60, 64), (64, 20, 64, 1000, 1, 0),
    (700, 6, 32, 90, 40, 100), (1025, 5, 128, 300, 300, 1), (4096, 3, 32, 60, 3, 10)])
def test_plan_matches_definition(requests, width, page, most_cached, most_new, pad):
    rng = np.random.default_rng(requests + page)
    cached = rng.integers(0, most_cached + 1, requests)
    new = rng.integers(0, most_new + 1, requests)
    new[rng.random(requests) < 0.3] = 0
    tables = rng.integers(0, 1000, (requests, width))
    free = rng.permutation(5000 + int(new.sum()) // page + requests)
    taken = 5
    tokens = int(new.sum()) + pad
    want = ref.plan(cached, new, tables, free, taken, page, tokens)
    table = _ints(tables)
    got = plan_step(_ints(cached), _ints(new), table, _ints(free), _ints([taken]), page_size=page, max_tokens=tokens)
    for name, a, b in zip(("slots", "positions", "starts", "lengths", "taken", "status"), got, want):
        assert np.array_equal(a.cpu().numpy().reshape(-1), np.reshape(b, -1)), name
    assert np.array_equal(table.cpu().numpy(), want[6])
    if want[5] == 0:
        got.check()


@pytest.mark.gpu
def test_plan_that_does_not_fit():
    # Pages run out in request 1; request 2 outgrows its row; 3 tokens too many.
    cached, new = [30, 31, 60, -4], [3, 40, 9, -2]
    tables, free = np.full((4, 2), 7), np.array([50])
    want = ref.plan(cached, new, tables, free, 0, 32, 49)
    table = _ints(tables)
    got = plan_step(_ints(cached), _ints(new), table, _ints(free), _ints([0]), page_size=32, max_tokens=49)
    assert want[5] == 7
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy().reshape(-1), np.reshape(b, -1))
    assert np.array_equal(table.cpu().numpy(), want[6])
    with pytest.raises(RuntimeError, match="ran out.*outgrew.*max_tokens"):
        got.check()
    none = plan_step(_ints([5]), _ints([1]), _ints([[3]]), _ints([]), _ints([0]), page_size=32, max_tokens=0)
    assert none.slots.numel() == 0 and int(none.status) == kv_cache.TOO_MANY_TOKENS


# ------------------------------------------------------------- writes and reads

def _slots(tokens, capacity, rng):
    slots = rng.permutation(capacity)[:tokens].astype(np.int64)
    return slots


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens, heads, dim, page", [(1, 1, 64, 32), (37, 3, 128, 64), (300, 2, 256, 128), (65, 5, 64, 256)])
def test_append_and_read_are_the_definition(tokens, heads, dim, page, dtype):
    rng = np.random.default_rng(tokens)
    pages = cache_pages(-(-tokens // page) + 1, page, heads, dim)
    x = torch.from_numpy(rng.normal(size=(tokens, 2 * heads, dim)) * np.exp(rng.normal(size=(tokens, 2 * heads, 1)) * 3)).to(dtype)
    x[0, 0, :32] = 0
    if tokens > 1:
        x[1, 0, 5] = float("nan")
        x[1, heads, 40] = float("inf")
        x[2, 0, :32] = 6e4  # the scale is at its limit, codes saturate
        x[3, heads] *= 1e-6
    slots = _slots(tokens, pages.shape[0] * page, rng)
    k, v = x[:, :heads].cuda(), x[:, heads:].cuda()
    assert append_tokens(pages, k, v, torch.from_numpy(slots).cuda()) is None
    got = read_tokens(pages, torch.from_numpy(slots).cuda(), dtype=torch.float32)
    for a, b in zip((x[:, :heads], x[:, heads:]), got):
        codes, scale = ref.encode(a.float().numpy())
        with np.errstate(all="ignore"):
            want = ref.butterfly32(codes.astype(np.float32) * scale.astype(np.float32)) * np.float32(0.25)
        assert np.array_equal(b.cpu().numpy(), want.reshape(b.shape), equal_nan=True)
        y = read_tokens(pages, torch.from_numpy(slots).cuda(), dtype=dtype)[0 if b is got[0] else 1]
        assert torch.equal(y.nan_to_num(7.0), b.to(dtype).nan_to_num(7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dim, page, heads", [(64, 32, 2), (128, 64, 3), (256, 256, 1)])
def test_layout_is_the_documented_one(dim, page, heads):
    """Bytes made from the documented layout read back as what they stand
    for, and writing the same tokens gives codes at the documented places."""
    rng = np.random.default_rng(dim)
    cache = ref.Cache(2, page, heads, dim, rng)
    cache.codes = np.maximum(cache.codes, -7)
    pages = torch.from_numpy(cache.bytes()).cuda()
    slots = torch.from_numpy(rng.permutation(2 * page)).cuda()
    for got, want in zip(read_tokens(pages, slots, dtype=torch.float32), cache.values()):
        # 5 sums of products of 3 and 8 bits in float32: 5 * 2^-24 of 32 terms of at most 7 s / 4.
        assert np.abs(got.cpu().numpy() - want[slots.cpu().numpy()]).max() <= 5 * 2.0 ** -24 * 8 * 7 * cache.scales.max()
    x = rng.normal(size=(2, 2 * page, heads, dim)).astype(np.float32)
    for i in range(2):
        codes, scale = ref.encode(x[i])
        cache.codes[i], cache.scales[i] = codes, scale
    append_tokens(pages, torch.from_numpy(x[0]).cuda(), torch.from_numpy(x[1]).cuda(),
                  torch.arange(2 * page, device="cuda"))
    assert np.array_equal(pages.cpu().numpy(), cache.bytes())


@pytest.mark.gpu
def test_append_touches_only_its_tokens():
    rng = np.random.default_rng(0)
    before = torch.from_numpy(ref.Cache(3, 64, 2, 128, rng).bytes()).cuda()
    pages = before.clone()
    k, v = (torch.randn(6, 2, 128, device="cuda", dtype=torch.float16) for _ in range(2))
    slots = torch.tensor([70, -1, 5, 192, 191, 1 << 40], device="cuda")
    append_tokens(pages, k, v, slots)
    others = torch.tensor([s for s in range(192) if s not in (70, 5, 191)], device="cuda")
    for a, b in zip(read_tokens(pages, others), read_tokens(before, others)):
        assert torch.equal(a, b)
    got, _ = read_tokens(pages, slots, dtype=torch.float32)
    want = ref.decode(*ref.encode(k.float().cpu().numpy()))
    inside = [0, 2, 4]
    assert np.abs(got.cpu().numpy()[inside] - want[inside]).max() <= 1e-5
    assert not got[[1, 3, 5]].any()
    empty = read_tokens(pages, slots[:0])
    assert empty[0].shape == (0, 2, 128)
    append_tokens(pages, k[:0], v[:0], slots[:0])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_heads, heads, dim, pairs", [(4, 2, 64, 32), (5, 1, 128, 16), (1, 1, 256, 128)])
def test_append_turns_keys_and_queries(q_heads, heads, dim, pairs, dtype, layout):
    rng = np.random.default_rng(dim + pairs)
    tokens = 70
    x = torch.from_numpy(rng.normal(size=(tokens, q_heads + 2 * heads, dim))).to(dtype).cuda()
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    freq, _ = rotary_frequencies(2 * pairs)
    at = torch.arange(tokens, device="cuda") + 12345
    pages = cache_pages(2, 64, heads, dim)
    slots = torch.randperm(128, device="cuda")[:tokens]
    turned = append_tokens(pages, k, v, slots, q=q, positions=at, frequencies=freq, layout=layout, magnitude=1.1)
    assert torch.equal(turned, apply_rotary(q, None, at, freq, layout=layout, magnitude=1.1)[0])
    assert turned.dtype == dtype
    got, values = read_tokens(pages, slots, dtype=torch.float32)
    exact = ref.turned(k.double().cpu(), at.cpu(), freq.cpu().numpy(), layout, 1.1)
    groups = exact.reshape(tokens, heads, -1, 32)
    y = groups @ ref.sylvester() / 8
    scale = np.abs(y).max(-1) / 7
    # Half a step in each of 32 transformed values, and up to 2^-8 of 7 steps
    # where the scale's rounding clips the largest; back in the basis (a factor
    # sqrt(32) / 4 in the 2-norm) that is sqrt(32) / 4 * sqrt(32) * 0.53 s.
    off = np.linalg.norm(got.cpu().double().numpy().reshape(groups.shape) - groups, axis=-1)
    assert (off <= 32 / 4 * 0.53 * scale * (1 + 2.0 ** -7)).all()
    # As the float32 steps give it but for codes that the angle's last bits move.
    codes, s = ref.encode(exact.astype(np.float32))
    near = np.abs(ref.decode(codes, s) - got.cpu().numpy()) <= 1e-5 * np.repeat(scale, 32, -1).reshape(exact.shape) * 32
    assert near.mean() > 0.98
    plain = cache_pages(2, 64, heads, dim)
    append_tokens(plain, k, v, slots)
    assert torch.equal(read_tokens(plain, slots, dtype=torch.float32)[1], values)


# ------------------------------------------------------------- attention

def _tables(lengths, page, width, pages, rng):
    ids = rng.permutation(pages)
    tables, at = np.full((len(lengths), width), -1), 0
    for r, n in enumerate(lengths):
        used = min(-(-n // page), width)
        tables[r, :used] = ids[at:at + used]
        at += used
    assert at <= pages
    return tables


def _tolerance(want, spread, basis, reach, dtype, few):
    """|o| rounded to its type; scores off by at most 2^-18 of |q| |k| scale
    (sums of up to 256 products in float32, operands of 22 bits) move a weight
    by that share; weights of 22 bits and float32 sums over tokens 2^-17 of
    sum p |v|, the sums in the transformed basis. Rows beyond `few` to a kv head may take weights, and bfloat16
    queries, in 11 bits: 2^-11 more of each."""
    scores = 2 * 2.0 ** -18 + (0 if few or dtype == torch.float16 else 2 * 2.0 ** -11)
    weights = 2.0 ** -17 + (0 if few else 2.0 ** -10)
    return UNIT[dtype] * np.abs(want) + (scores * reach + weights) * spread + 2.0 ** -17 * basis + 2.0 ** -24


def _check(q, cache, page, tables, starts, lengths, dtype, window=None, scale=None, max_new=None, group=1):
    keys, values = cache.values()
    dim = q.shape[-1]
    pages = torch.from_numpy(cache.bytes()).cuda()
    got = cache_attention(q.cuda(), pages, _ints(tables), _ints(starts), _ints(lengths), window=window, scale=scale,
                          max_new=max_new)
    s = dim ** -0.5 if scale is None else scale
    want, spread, basis, reach = ref.attention(q.double().numpy(), keys, values, page, tables, starts, lengths, s, window)
    few = max(np.diff(starts), default=0) * group <= 16
    off = np.abs(got.cpu().double().numpy() - want)
    assert got.dtype == dtype and got.shape == q.shape
    assert np.array_equal(np.isnan(off), np.isnan(want)) or np.array_equal(np.isnan(got.cpu().double().numpy()), np.isnan(want))
    good = ~np.isnan(want)
    assert (off <= _tolerance(want, spread, basis, reach, dtype, few))[good].all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, group, dim, page", [
    (2, 4, 128, 64), (1, 1, 64, 32), (3, 8, 64, 128), (2, 2, 256, 256), (1, 16, 128, 32), (1, 20, 256, 32), (2, 5, 64, 64)])
def test_single_tokens(heads, group, dim, page, dtype):
    rng = np.random.default_rng(dim + group)
    lengths = [1, 2, 31, 32, 33, 0, 64, 200, 257, 700]
    cache = ref.Cache(sum(-(-n // page) for n in lengths) + 2, page, heads, dim, rng)
    tables = _tables(lengths, page, -(-700 // page) + 1, cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(len(lengths), heads * group, dim)) * 2).to(dtype)
    starts = np.arange(len(lengths) + 1)
    a = _check(q, cache, page, tables, starts, lengths, dtype, max_new=1, group=group)
    assert not a[5].any()
    b = _check(q, cache, page, tables, starts, lengths, dtype, window=33, group=group)
    assert not torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, group, dim, page, window", [
    (2, 4, 128, 64, None), (1, 1, 64, 32, 40), (2, 8, 64, 32, 1), (1, 2, 256, 128, 100), (1, 32, 128, 64, None)])
def test_drafts_chunks_and_prompts(heads, group, dim, page, window, dtype):
    """Requests with nothing new, one token, drafts, chunks and whole prompts
    in one call, and rows of no request after them."""
    rng = np.random.default_rng(dim + group + 1)
    new = [3, 0, 1, 40, 129, 8, 65]
    lengths = [130, 50, 1, 40, 300, 5, 257]  # the sixth has rows before its first position
    starts = np.concatenate([[0], np.cumsum(new)])
    cache = ref.Cache(sum(-(-n // page) for n in lengths) + 1, page, heads, dim, rng)
    tables = _tables(lengths, page, -(-300 // page), cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(starts[-1] + 5, heads * group, dim)) * 2).to(dtype)
    got = _check(q, cache, page, tables, starts, lengths, dtype, window=window, group=group)
    assert not got[starts[-1]:].any() and not got[starts[5]:starts[5] + 3].any()
    for hint in (1, 129):
        other = _check(q, cache, page, tables, starts, lengths, dtype, window=window, max_new=hint, group=group)
        assert other.shape == got.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, new", [(64, 1), (128, 1), (256, 1), (64, 30), (128, 30), (64, 200), (128, 200), (256, 60)])
def test_small_weights_of_a_long_context(dim, new, dtype):
    """Every 32nd position has a value of 0 and outweighs each of the others by
    about 2^20.3: what is left of the output is all theirs, 2^-15 of a value. (In
    every tile, so that no share of the context is without one.)"""
    context, page, group = 20000, 256, 4
    g = torch.Generator().manual_seed(dim + new)
    u = torch.sign(torch.randn(dim, generator=g))
    k, v = torch.zeros(context, 1, dim), 64 * torch.randn(context, 1, dim, generator=g).abs()
    k[::32, 0], v[::32] = u, 0.0
    pages = cache_pages(-(-context // page), page, 1, dim)
    slots = torch.arange(context, device="cuda")
    append_tokens(pages, k.cuda(), v.cuda(), slots)
    q = (u * (20.3 * np.log(2) / dim)).to(dtype).expand(new, group, dim).contiguous().cuda()
    got = cache_attention(q, pages, _ints([np.arange(pages.shape[0])]), _ints([0, new]), _ints([context]), scale=1.0)
    keys, values = (x[:, 0].double() for x in read_tokens(pages, slots, dtype=torch.float32))
    scores = q[:, 0].double() @ keys.T
    at = torch.arange(context, device="cuda")
    scores[at[None] > (context - new + torch.arange(new, device="cuda"))[:, None]] = -torch.inf
    weights = torch.softmax(scores, 1)
    want = (weights @ values)[:, None].expand(-1, group, -1)
    # Weights (and of many rows bfloat16 queries) in 11 bits, scores up to 15 of
    # 22 bits or, of those queries, 11; float32 sums of 20000 terms in tiles of 32.
    # Twice the output bounds sum p |v|, whose few negative values are small.
    scores_off = 15 * (2.0 ** -18 if new * group <= 16 or dtype == torch.float16 else 2.0 ** -11)
    share = UNIT[dtype] + 2 * scores_off + 2.0 ** -10 + 2.0 ** -12
    assert (((got.double() - want).abs()) <= share * 2.0 * want.abs().amax(-1, keepdim=True) + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group, new, window", [(3, [3, 1, 4, 2, 0, 5], None), (16, [1, 2, 1, 1, 2, 1], 40), (5, [6, 5, 4, 6, 1, 2], 33),
                                                (4, [8, 3, 60, 1, 7, 8], None)])
def test_blocks_of_eight_rows_of_large_heads(group, new, window, dtype):
    """9 to 32 rows of head dimension 256: tokens whose heads lie in two blocks,
    contexts of the new tokens alone, and beside a chunk of many rows."""
    rng = np.random.default_rng(group)
    lengths = [n + c for n, c in zip(new, (700, 0, 31, 32, 5, 1500))]
    cache = ref.Cache(sum(-(-n // 32) for n in lengths), 32, 2, 256, rng)
    tables = _tables(lengths, 32, 48, cache.shape[0], rng)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.normal(size=(starts[-1], 2 * group, 256)) * 2).to(dtype)
    _check(q, cache, 32, tables, starts, lengths, dtype, window=window, max_new=max(new), group=group)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 4, 70])
def test_long_context_is_split(new):
    rng = np.random.default_rng(new)
    lengths = [9000, 17, 2500]
    starts = np.arange(4) * new
    cache = ref.Cache(sum(-(-n // 256) for n in lengths), 256, 1, 64, rng)
    tables = _tables(lengths, 256, 40, cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(3 * new, 4, 64)) * 4).to(torch.bfloat16)
    a = _check(q, cache, 256, tables, starts, lengths, torch.bfloat16, group=4)
    again = cache_attention(q.cuda(), torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(lengths))
    assert torch.equal(a, again)  # the same sums in the same order


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, group, dim, page, new, context, window", [
    (1, 4, 128, 64, [400, 33, 129], [700, 200, 129], None),     # cut into shares
    (2, 5, 128, 32, [200, 77], [333, 1500], 250),               # rows of a token in two blocks
    (1, 2, 256, 128, [301, 65], [301, 900], None),
    (1, 8, 256, 32, [100], [2000], 600),
    (3, 3, 64, 64, [150, 1, 260], [2100, 40, 260], 1000),
    (16, 4, 64, 256, [3100], [3100], None),                     # enough blocks to be dealt whole
    (16, 2, 128, 64, [2300, 1900], [2350, 1900], 700)])         # and here
def test_many_rows(heads, group, dim, page, new, context, window, dtype):
    """Chunks and prompts whose rows fill workgroups, with ragged ends, rows
    that straddle blocks, windows and the first positions of a context."""
    rng = np.random.default_rng(dim + heads)
    starts = np.concatenate([[0], np.cumsum(new)])
    pages = sum(-(-n // page) for n in context) + 1
    cache = ref.Cache(pages, page, heads, dim, rng)
    tables = _tables(context, page, -(-max(context) // page), pages, rng)
    q = torch.from_numpy(rng.normal(size=(starts[-1], heads * group, dim)) * 2).to(dtype)
    got = cache_attention(q.cuda(), torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints(starts), _ints(context),
                          window=window, max_new=max(new))
    keys, values = (torch.from_numpy(x).cuda() for x in cache.values())
    want, spread, basis, reach = ref.attention_dense(q.cuda(), keys, values, page, tables, starts, context, dim ** -0.5, window)
    off = np.abs(got.cpu().double().numpy() - want)
    few = np.repeat(np.asarray(new) * group <= 16, new)[:, None, None]
    tolerance = np.where(few, _tolerance(want, spread, basis, reach, dtype, True), _tolerance(want, spread, basis, reach, dtype, False))
    assert (off <= tolerance).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_with_holes(dim):
    """NaN in unattended positions and missing pages under blocks of rows."""
    rng = np.random.default_rng(dim)
    page, group, lengths, new = 32, 4, [500, 260], [300, 260]
    starts = np.concatenate([[0], np.cumsum(new)])
    cache = ref.Cache(30, page, 1, dim, rng)
    tables = _tables(lengths, page, 17, 30, rng)
    clean = torch.from_numpy(cache.bytes()).cuda()
    q = torch.from_numpy(rng.normal(size=(starts[-1], group, dim))).half().cuda()
    args = _ints(starts), _ints(lengths)
    want = cache_attention(q, clean, _ints(tables), *args, window=128)
    used = [tables[r][t // page] * page + t % page for r in range(2) for t in range(lengths[r])]
    unused = np.setdiff1d(np.arange(30 * page), used)
    # The first request's window begins at 200 - 127.
    unused = np.concatenate([unused, tables[0][np.arange(64) // page] * page + np.arange(64) % page])
    cache.scales[0][unused], cache.scales[1][unused] = np.nan, np.inf
    dirty = torch.from_numpy(cache.bytes()).cuda()
    assert torch.equal(cache_attention(q, dirty, _ints(tables), *args, window=128), want)
    # One NaN value group, attended by 128 rows of a token; one page missing.
    slot = tables[0][300 // page] * page + 300 % page
    cache.scales[1][slot, 0, 1] = np.nan
    holes = tables.copy()
    holes[1, 2] = -1
    got = cache_attention(q, torch.from_numpy(cache.bytes()).cuda(), _ints(holes), *args, window=128).cpu()
    nan = torch.isnan(got)
    assert nan[100:228, :, 32:64].all() and nan.sum() == 128 * group * 32
    keys, values = cache.values()
    sample = [300, 300 + 64, 300 + 100, 300 + 200, 559]
    for i in sample:
        p = i - 300
        one, *_ = ref.attention(q[i:i + 1].cpu().double().numpy(), keys, values, page, holes[1:], [0, 1], [p + 1], dim ** -0.5, 128)
        # Weights in 11 bits and the result's own rounding.
        assert np.abs(got[i].double().numpy() - one[0]).max() <= 2.0 ** -9 * (np.abs(one).max() + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 6, 80])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_masked_positions_may_hold_anything(new, dim):
    """Positions past a row's own, in unused slots and in pages that the table
    does not name hold NaN and infinities; a NaN that is attended reaches the
    rows and groups it belongs to and no others."""
    rng = np.random.default_rng(dim + new)
    page, group = 32, 2
    lengths = [100, 70, 140]
    starts = np.arange(4) * new
    cache = ref.Cache(16, page, 1, dim, rng)
    tables = _tables(lengths, page, 5, 16, rng)
    used = [tables[r][t // page] * page + t % page for r in range(3) for t in range(lengths[r])]
    unused = np.setdiff1d(np.arange(16 * page), used)
    cache.scales[0][unused] = np.nan
    cache.scales[1][unused] = np.inf
    # The last position of request 1: only its last row attends it. One key of
    # request 2 is NaN from the last but one position on.
    last = tables[1][69 // page] * page + 69 % page
    cache.scales[1][last, 0, 1] = np.nan
    some = tables[2][138 // page] * page + 138 % page
    cache.scales[0][some, 0, 0] = np.nan
    tables[0, 1] = -1            # 32 positions of request 0 are not there
    tables[0, 2] = 1 << 20
    q = torch.from_numpy(rng.normal(size=(3 * new, group, dim))).to(torch.float16)
    got = _check(q, cache, page, tables, starts, lengths, torch.float16, group=group)
    nan = torch.isnan(got.cpu())
    rows = nan[new:2 * new]
    assert rows[-1, :, 32:64].all() and rows.sum() == 32 * group
    assert nan[2 * new:].sum() == min(new, 2) * group * dim and not nan[:new].any()
    window = _check(q, cache, page, tables, starts, lengths, torch.float16, window=1, group=group)
    assert torch.isnan(window.cpu()).sum() == 32 * group + (group * dim if new > 1 else 0)


@pytest.mark.gpu
def test_large_and_small_queries():
    """bfloat16 queries beyond float16's range, tiny ones, and zero rows."""
    rng = np.random.default_rng(8)
    cache = ref.Cache(4, 64, 1, 128, rng)
    tables, lengths = np.array([[2, 0, 3]]), [150]
    q = torch.from_numpy(rng.normal(size=(1, 4, 128)))
    q[0, 0] *= 1e5
    q[0, 1] *= 1e-30
    q[0, 2] = 0
    q = q.to(torch.bfloat16)
    # With scores of thousands the bound on a score passes 1: those rows are
    # compared at a scale that keeps them in range.
    _check(q, cache, 64, tables, [0, 1], lengths, torch.bfloat16, scale=1e-7)
    nan = q.clone()
    nan[0, 0, 3] = float("nan")
    got = cache_attention(nan.cuda(), torch.from_numpy(cache.bytes()).cuda(), _ints(tables), _ints([0, 1]), _ints(lengths))
    assert torch.isnan(got[0, 0]).all() and not torch.isnan(got[0, 1:]).any()


@pytest.mark.gpu
def test_table_values_out_of_range_are_harmless():
    """Lengths past the table, starts past the queries and negative values are
    cut to what the arrays hold."""
    rng = np.random.default_rng(9)
    cache = ref.Cache(3, 32, 1, 64, rng)
    pages = torch.from_numpy(cache.bytes()).cuda()
    q = torch.randn(4, 2, 64, device="cuda", dtype=torch.float16)
    tables = _ints([[0, 1], [2, 5], [1, -3]])
    want = cache_attention(q, pages, tables, _ints([0, 1, 2, 4]), _ints([64, 32, 0]))
    got = cache_attention(q, pages, tables, _ints([-7, 1, 2, 400]), _ints([1 << 30, 40, -5]))
    assert torch.isfinite(got).all() and torch.equal(got[0], want[0]) and not got[2:].any()
    # Requests that claim the same rows, many and few to a kv head.
    for rows in (4, 300):
        many = torch.randn(rows, 2, 64, device="cuda", dtype=torch.float16)
        over = cache_attention(many, pages, tables, _ints([0, rows, 0, rows]), _ints([64, 32, 60]))
        assert over.shape == many.shape
    none = cache_attention(q[:0], pages, tables, _ints([0, 0, 0, 0]), _ints([64, 32, 0]))
    assert none.shape == (0, 2, 64)
    empty = cache_attention(q, pages[:0], tables, _ints([0, 1, 2, 4]), _ints([64, 32, 0]))
    assert not empty.any()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 150])
def test_places_past_32_bits(new):
    """The last pages of a cache of 5.4 GB hold the same tokens as a small
    cache's, and give the same bits; so do queries more than 2^31 bytes in."""
    heads, dim, page, context = 8, 128, 64, 300
    many = 73_000                                        # 73728 bytes each
    g = torch.Generator(device="cuda").manual_seed(new)
    k, v = (torch.randn(context, heads, dim, device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn(new, 2 * heads, dim, device="cuda", generator=g).half()
    order = torch.tensor([2, 4, 0, 3, 1], device="cuda")
    at = torch.arange(context, device="cuda")
    results = []
    for pages in (5, many):
        cache = torch.empty(pages, heads, page // 32, 36 * dim, dtype=torch.uint8, device="cuda")
        cache[-5:] = 0
        table = order + (pages - 5)
        slots = table[at // page] * page + at % page
        append_tokens(cache, k, v, slots)
        rows = q
        if pages == many:
            stride = (2 ** 31 // new + 1024) // 8 * 8    # the last row starts past 2^31 bytes
            wide = torch.empty((new - 1) * stride + 2 * heads * dim + 8, dtype=torch.float16, device="cuda")
            rows = wide.as_strided((new, 2 * heads, dim), (stride, dim, 1))
            rows.copy_(q)
        results.append((*read_tokens(cache, slots), cache_attention(
            rows, cache, table.int()[None], _ints([0, new]), _ints([context]))))
        del cache
    for small, large in zip(*results):
        assert torch.equal(small, large)


@pytest.mark.gpu
def test_other_streams_and_strides():
    rng = np.random.default_rng(10)
    cache = ref.Cache(8, 64, 2, 128, rng)
    pages = torch.from_numpy(cache.bytes()).cuda()
    tables, starts, lengths = _ints([[0, 3], [5, 1]]), _ints([0, 1, 3]), _ints([128, 70])
    x = torch.randn(3, 12, 128, device="cuda", dtype=torch.bfloat16)
    want = cache_attention(x[:, :8].contiguous(), pages, tables, starts, lengths)
    assert torch.equal(want, cache_attention(x[:, :8], pages, tables, starts, lengths))
    odd = torch.randn(3 * 8 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(3, 8, 128).copy_(x[:, :8])
    assert torch.equal(want, cache_attention(odd, pages, tables, starts, lengths))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [cache_attention(x[:, :8], pages, tables, starts, lengths) for _ in range(4)]
    stream.synchronize()
    assert all(torch.equal(want, g) for g in got)


@pytest.mark.gpu
def test_step_in_a_graph():
    """A captured step replays with new lengths, slots and tokens."""
    torch.manual_seed(0)
    requests, heads, dim, page = 3, 2, 64, 32
    pages = cache_pages(20, page, heads, dim)
    tables = torch.full((requests, 6), -1, dtype=torch.int32, device="cuda")
    free, taken = _ints(np.arange(20)), _ints([0])
    cached, new = _ints([0, 0, 0]), _ints([1, 1, 1])
    freq, _ = rotary_frequencies(dim)
    x = torch.randn(requests, 4 + 2 * heads, dim, device="cuda", dtype=torch.bfloat16)

    def step(pages, tables):
        plan = plan_step(cached, new, tables, free, taken, page_size=page, max_tokens=requests)
        q = append_tokens(pages, x[:, 4:6], x[:, 6:], plan.slots, q=x[:, :4], positions=plan.positions, frequencies=freq)
        return cache_attention(q, pages, tables, plan.starts, plan.lengths, max_new=1), plan.taken

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pages.clone(), tables.clone())
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out, after = step(pages, tables)
    pages.zero_(), tables.fill_(-1)
    eager_pages, eager_tables = pages.clone(), tables.clone()
    for i in range(40):
        x.copy_(torch.randn_like(x))
        want, _ = step(eager_pages, eager_tables)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pages, eager_pages), i
        taken.copy_(after)
        cached += 1
    assert int(taken) == 2 * requests


def test_refuses_cpu_tensors_and_shapes():
    pages = cache_pages(2, 32, 1, 64, device="cpu")
    assert pages.shape == (2, 1, 1, 2304)
    k = torch.zeros(1, 1, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        append_tokens(pages, k, k, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        plan_step(*(torch.zeros(1, dtype=torch.int32) for _ in range(2)), torch.zeros(1, 1, dtype=torch.int32),
                  *(torch.zeros(1, dtype=torch.int32) for _ in range(2)), page_size=32, max_tokens=1)
    for bad in ((1, 48, 1, 64), (1, 512, 1, 64), (1, 32, 1, 96), (-1, 32, 1, 64), (1, 32, 0, 64)):
        with pytest.raises(ValueError):
            cache_pages(*bad, device="cpu")


@pytest.mark.gpu
def test_refusals():
    pages = cache_pages(2, 32, 2, 64)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    freq, _ = rotary_frequencies(64)
    at = _ints([0, 1, 2])
    for args, more in (((pages[0], k, k, slots), {}), ((pages.float(), k, k, slots), {}), ((pages[..., :100], k, k, slots), {}),
                       ((pages, k[:, :1], k, slots), {}), ((pages, k, k.float(), slots), {}), ((pages, k, k[:2], slots), {}),
                       ((pages, k, k, slots.int()), {}), ((pages, k, k, slots[:2]), {}), ((pages, k, k.cpu(), slots), {}),
                       ((pages, k, k, slots), dict(q=k)), ((pages, k, k, slots), dict(frequencies=freq)),
                       ((pages, k, k, slots), dict(frequencies=freq[:12], positions=at)),
                       ((pages, k, k, slots), dict(frequencies=freq, positions=at, q=k[:2])),
                       ((pages, k.clone().requires_grad_(), k, slots), {})):
        with pytest.raises(RuntimeError):
            append_tokens(*args, **more)
    with pytest.raises(RuntimeError):
        read_tokens(pages, slots, dtype=torch.int8)
    tables, starts, lengths = _ints([[0, 1]]), _ints([0, 3]), _ints([40])
    for args, more in (((k.float(), pages, tables, starts, lengths), {}), ((k[:, :1], pages, tables, starts, lengths), {}),
                       ((k[..., :32], pages, tables, starts, lengths), {}), ((k, pages, tables.long(), starts, lengths), {}),
                       ((k, pages, tables, starts[:1], lengths), {}), ((k, pages, tables, starts, lengths.long()), {}),
                       ((k, pages, tables, starts, lengths), dict(window=0)), ((k, pages, tables, starts, lengths), dict(max_new=-1)),
                       ((k, pages, _ints(np.zeros((0, 2))), _ints([0]), _ints([])), {}),
                       ((k.clone().requires_grad_(), pages, tables, starts, lengths), {})):
        with pytest.raises(RuntimeError):
            cache_attention(*args, **more)
    big = torch.zeros(4097, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="4096"):
        plan_step(big, big, torch.zeros(4097, 1, dtype=torch.int32, device="cuda"), big, big[:1], page_size=32, max_tokens=1)
    with pytest.raises(RuntimeError, match="page_size"):
        plan_step(at, at, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), at, at[:1], page_size=33, max_tokens=1)


@pytest.mark.gpu
def test_example_serves_quantized_block():
    """Group maxima of 32 normal values are about 2.2 sigma, so codes are 0.31
    sigma apart and off by 0.09 sigma in keys and values both; weights move by
    about as much for scores of order one: 0.13 together."""
    import importlib.util
    from .conftest import REPO_ROOT
    spec = importlib.util.spec_from_file_location("serve_quantized", REPO_ROOT / "examples" / "serve_quantized.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    error = example.serve(tokens=3)
    assert 0.01 < error < 0.2
