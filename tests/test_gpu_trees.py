"""Trees of drafted tokens: plans, attention, what is accepted and kept of them,
against their definitions written token by token."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import _native
from exl3_intel_arc_quantizer_amd.kv_cache import (accept_drafts, append_tokens, cache_attention, cache_pages,
                                                   keep_tokens, plan_step, plan_tree, read_tokens, release_pages)
from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_axes, rotary_frequencies

from . import cache_ref as ref
from .test_gpu_kv_cache import _tables, _tolerance


def _ints(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


def _forest(new, rng, reach=6):
    """Parents of every token: mostly the one before it, some roots."""
    return [-1 if i == 0 or rng.random() < 0.05 else int(rng.integers(max(0, i - reach), i)) if rng.random() < 0.6 else i - 1
            for n in new for i in range(n)]


def _paths(new, parents):
    """Per token its ancestors and itself, ascending."""
    paths, at = [], 0
    for n in new:
        for i in range(n):
            p = parents[at + i]
            paths.append((paths[at + p] if 0 <= p < i else []) + [i])
        at += n
    return paths


def _masks(rows, words):
    """int64 (rows, words) of lists of bits."""
    out = np.zeros((len(rows), 64 * words), np.uint8)
    for t, bits in enumerate(rows):
        out[t, bits] = 1
    return torch.from_numpy(np.packbits(out, axis=1, bitorder="little").view(np.int64).reshape(len(rows), words))


def _attention(q, keys, values, page, tables, starts, lengths, scale, seen):
    """As cache_ref.attention, of the positions that seen(r, i) gives."""
    q = np.asarray(q, np.float64)
    tokens, heads, dim = q.shape
    kv_heads, pages = keys.shape[1], keys.shape[0] // page
    out, spread, basis, reach = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q), np.zeros((tokens, heads, 1))
    for r in range(len(lengths)):
        for i in range(starts[r + 1] - starts[r]):
            t = np.asarray(seen(r, i), np.int64)
            ids = np.asarray(tables[r])[t // page] if len(t) else np.zeros(0, np.int64)
            slots = (ids * page + t % page)[(ids >= 0) & (ids < pages)]
            if not len(slots):
                continue
            row = starts[r] + i
            for h in range(heads):
                k, v = keys[slots, h * kv_heads // heads], values[slots, h * kv_heads // heads]
                with np.errstate(all="ignore"):
                    x = scale * (k @ q[row, h])
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    out[row, h], spread[row, h] = (w[:, None] * v).sum(0), (w[:, None] * np.abs(v)).sum(0)
                    held = np.abs(v.reshape(-1, dim // 32, 32) @ ref.sylvester()) / 8
                    basis[row, h] = np.repeat((w[:, None, None] * held).sum((0, 2)) / 4, 32)
                    reach[row, h] = scale * np.linalg.norm(q[row, h]) * np.linalg.norm(k, axis=1).max()
    return out, spread, basis, reach


def _check(q, cache, page, tables, new, lengths, rows, words, dtype, window=None, max_new=None, group=1):
    """``rows``: per token the new tokens its mask names. Requests of more tokens
    than the masks have bits attend causally."""
    starts = np.concatenate([[0], np.cumsum(new)]).astype(int)

    def seen(r, i):
        n, length = new[r], lengths[r]
        if n > 64 * words:
            whole = range(length - n + i + 1)
        else:
            whole = list(range(length - n)) + [length - n + j for j in rows[starts[r] + i] if j < n]
        return list(whole)[-min(window or 1 << 40, len(whole)):] if len(whole) else []

    keys, values = cache.values()
    pages = torch.from_numpy(cache.bytes()).cuda()
    got = cache_attention(q.cuda(), pages, _ints(tables), _ints(starts), _ints(lengths), window=window, max_new=max_new,
                          trees=_masks(rows, words).cuda())
    want, spread, basis, scores = _attention(q.double().numpy(), keys, values, page, tables, starts, lengths, q.shape[-1] ** -0.5, seen)
    few = max(new) * group <= 16
    got = got.cpu()
    nan = np.isnan(want)
    assert np.array_equal(torch.isnan(got).numpy(), nan)
    off = np.abs(got.double().numpy() - want)
    assert (off <= _tolerance(want, spread, basis, scores, dtype, few))[~nan].all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, group, dim, page, most, window", [
    (2, 4, 128, 64, 1, None), (1, 1, 64, 32, 7, None), (2, 2, 128, 32, 8, 40), (1, 8, 256, 64, 4, None), (1, 4, 64, 128, 30, 100),
    (2, 4, 128, 64, 40, None), (1, 4, 256, 32, 33, 70), (1, 16, 128, 64, 64, None), (1, 8, 64, 32, 64, 3)])
def test_trees_attend_ancestors(heads, group, dim, page, most, window, dtype):
    rng = np.random.default_rng(dim + group + most)
    new = [most, 0, 1, max(1, most // 2), most, max(1, most - 3)]
    lengths = [200 + most, 50, 1, 64, most, 333]
    parents = _forest(new, rng)
    cache = ref.Cache(sum(-(-n // page) for n in lengths) + 1, page, heads, dim, rng)
    tables = _tables(lengths, page, -(-400 // page), cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(sum(new), heads * group, dim)) * 2).to(dtype)
    rows = _paths(new, parents)
    got = _check(q, cache, page, tables, new, lengths, rows, 1, dtype, window=window, max_new=most, group=group)
    _check(q, cache, page, tables, new, lengths, rows, 3, dtype, window=window, group=group)
    # A run is a tree of one branch: as without masks, in rounding.
    runs = _paths(new, [i - 1 for n in new for i in range(n)])
    run = _check(q, cache, page, tables, new, lengths, runs, 1, dtype, window=window, max_new=most, group=group)
    if most > 6:
        assert not torch.equal(run, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, most, words, window", [(64, 130, 3, None), (128, 150, 3, 90), (256, 100, 2, None), (128, 70, 16, 5), (64, 65, 1, None)])
def test_large_trees_and_runs_beside_them(dim, most, words, window, dtype):
    """Trees of several words, and requests that are too long to be one."""
    rng = np.random.default_rng(dim + most)
    new = [most, 64 * words + 5 if words < 4 else 3, 2, 64]
    lengths = [most + 77, 64 * words + 5 + 30, 90, 64]
    parents = _forest(new, rng, 40)
    cache = ref.Cache(sum(-(-n // 32) for n in lengths) + 1, 32, 1, dim, rng)
    tables = _tables(lengths, 32, 40, cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(sum(new), 4, dim)) * 2).to(dtype)
    _check(q, cache, 32, tables, new, lengths, [p if max(p) < 64 * words else [] for p in _paths(new, parents)], words, dtype,
           window=window, group=4)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 40, 90])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_any_mask(dim, new):
    """Masks that name nothing, all, later tokens and not the row's own; rows that
    a window and an empty mask leave with nothing; NaN in places not named."""
    rng = np.random.default_rng(dim + new)
    words = -(-new // 64)
    lengths = [new, new + 40, new + 3]
    rows = [sorted(rng.permutation(new)[:rng.integers(0, new + 1)].tolist()) for _ in range(3 * new)]
    rows[0], rows[new] = [], []
    cache = ref.Cache(16, 32, 1, dim, rng)
    tables = _tables(lengths, 32, 5, 16, rng)
    q = torch.from_numpy(rng.normal(size=(3 * new, 2, dim))).to(torch.float16)
    for window in (None, 1, 30):
        got = _check(q, cache, 32, tables, [new] * 3, lengths, rows, words, torch.float16, window=window, group=2)
        assert not got[0].any() and got[new].any()
    # The last new token of request 1 holds NaN: only rows that name it see it.
    slot = tables[1][(new + 39) // 32] * 32 + (new + 39) % 32
    cache.scales[1][slot, 0, 1] = np.nan
    got = _check(q, cache, 32, tables, [new] * 3, lengths, rows, words, torch.float16, group=2)
    hit = torch.isnan(got).flatten(1).any(1)
    assert hit.tolist() == [new <= t < 2 * new and new - 1 in rows[t] for t in range(3 * new)]
    tables[1, 0] = -1
    _check(q, cache, 32, tables, [new] * 3, lengths, rows, words, torch.float16, group=2)


@pytest.mark.gpu
@pytest.mark.parametrize("most, words, requests", [(1, 1, 1), (13, 1, 5), (64, 1, 9), (65, 2, 3), (200, 4, 4), (1024, 16, 2), (9, 1, 700)])
def test_plan_tree(most, words, requests):
    rng = np.random.default_rng(most + requests)
    new = [most] + [int(n) for n in rng.integers(0, most + 1, size=requests - 1)]
    parents = _forest(new, rng, 50)
    lengths = [n + int(rng.integers(0, 5000)) for n in new]
    starts, pad = np.concatenate([[0], np.cumsum(new)]), 37
    given = parents + [5] * pad
    bad = [t for t in range(len(parents)) if parents[t] == -1]
    for t in bad[::2]:   # whatever is no earlier token counts as none
        given[t] = int(rng.choice([-7, 10 ** 6, 1 << 30]))
    tree = plan_tree(_ints(given), _ints(starts), _ints(lengths), max_new=most)
    paths = _paths(new, parents)
    assert torch.equal(tree.masks.cpu(), torch.cat([_masks(paths, words), torch.zeros(pad, words, dtype=torch.int64)]))
    cached = np.repeat(np.array(lengths) - new, new)
    assert tree.positions.tolist() == [int(c) + len(p) - 1 for c, p in zip(cached, paths)] + [0] * pad
    # Longer than a mask has bits: a run.
    if words > 1:
        tree = plan_tree(_ints(given), _ints(starts), _ints(lengths), max_new=64)
        assert tree.masks.shape == (len(given), 1) and not tree.masks[:most].any()
        assert tree.positions[:most].tolist() == list(range(lengths[0] - most, lengths[0]))


def _accepted(new, lengths, parents, tokens, choices, certain):
    places, kept, after, at = [-1] * len(parents), [], [], 0
    for r, n in enumerate(new):
        path = list(range(min(max(certain[r], 1), n)))
        first = len(path)
        while path:
            child = [c for c in range(first, n) if c > path[-1] and parents[at + c] == path[-1] and tokens[at + c] == choices[at + path[-1]]]
            if not child:
                break
            path.append(child[0])
        for place, i in enumerate(path):
            places[at + i] = place
        kept.append(lengths[r] - n + len(path))
        after.append(choices[at + path[-1]] if n else -1)
        at += n
    return places, kept, after


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("most, requests", [(1, 1), (2, 3), (13, 6), (64, 9), (65, 4), (300, 5), (12, 900)])
def test_accept_drafts(most, requests, dtype):
    rng = np.random.default_rng(most * requests)
    new = [most] + [int(n) for n in rng.integers(0, most + 1, size=requests - 1)]
    parents, total = _forest(new, rng, 30), sum(new)
    lengths = [n + int(rng.integers(0, 99)) for n in new]
    # Few ids, so that siblings are alike and most choices are met.
    tokens, choices = rng.integers(0, 3, total).tolist(), rng.integers(0, 3, total).tolist()
    if dtype == torch.int64:
        tokens, choices = [t + (1 << 40) for t in tokens], [t + (1 << 40) for t in choices]
    certain = [int(c) for c in rng.choice([-1, 0, 1, 2, 5, 1 << 20], requests)]
    starts, pad = _ints(np.concatenate([[0], np.cumsum(new)])), [7] * 5
    args = _ints(tokens + pad, dtype), _ints(choices + pad, dtype), _ints(parents + [0] * 5), starts, _ints(lengths)
    for given in (None, certain):
        got = accept_drafts(*args, certain=None if given is None else _ints(given))
        places, kept, after = _accepted(new, lengths, parents, tokens, choices, given or [1] * requests)
        assert got.places.tolist() == places + [-1] * 5
        assert got.lengths.tolist() == kept and got.next.tolist() == after and got.next.dtype == dtype


@pytest.mark.gpu
@pytest.mark.parametrize("heads, dim, page, most, requests", [(1, 64, 32, 3, 1), (3, 128, 64, 20, 5), (2, 256, 128, 70, 3), (2, 64, 256, 600, 2), (8, 128, 32, 9, 60)])
def test_keep_tokens(heads, dim, page, most, requests):
    """Bytes of kept entries at their places, all others as they were."""
    rng = np.random.default_rng(most + requests)
    new = [most] + [int(n) for n in rng.integers(0, most + 1, size=requests - 1)]
    total = sum(new)
    pages = torch.randint(0, 256, (-(-total // page) + 3, heads, page // 32, 36 * dim), dtype=torch.uint8, device="cuda")
    slots = rng.permutation(pages.shape[0] * page)[:total]
    places, want = [], {}
    for r, n in enumerate(new):
        kept = np.flatnonzero(rng.random(n) < (0.5 if r else 0.95))
        row = np.full(n, -1)
        row[kept] = np.arange(len(kept))
        places += row.tolist()
    starts = np.concatenate([[0], np.cumsum(new)])
    one, other = 3, 4
    hidden = slots.copy()
    if total > 20:   # a slot outside the cache: its moves do nothing
        hidden[one], hidden[other] = -1, pages.shape[0] * page
    for r, n in enumerate(new):
        for i in range(n):
            source, place = hidden[starts[r] + i], places[starts[r] + i]
            if place >= 0 and 0 <= source < pages.shape[0] * page and 0 <= hidden[starts[r] + place] < pages.shape[0] * page:
                want[int(hidden[starts[r] + place])] = int(source)
    every = torch.arange(pages.shape[0] * page, device="cuda")
    before = read_tokens(pages, every, dtype=torch.float32)
    source = every.clone()
    for to, of in want.items():
        source[to] = of
    version = pages._version
    keep_tokens(pages, _ints(hidden, torch.int64), _ints(starts), _ints(places))
    assert pages._version > version
    for x, y in zip(before, read_tokens(pages, every, dtype=torch.float32)):
        assert torch.equal(x[source].view(torch.int32), y.view(torch.int32))
    again = pages.clone()
    keep_tokens(pages, _ints(slots, torch.int64), _ints(starts), _ints(np.full(total, -1)))
    assert torch.equal(again, pages)


@pytest.mark.gpu
@pytest.mark.parametrize("requests, width, page", [(1, 5, 64), (7, 9, 32), (300, 4, 256), (40, 200, 32)])
def test_release_pages(requests, width, page):
    rng = np.random.default_rng(requests + width)
    before = rng.integers(0, width * page + page, requests)          # some past their rows
    after = np.maximum(before - rng.integers(-3, 2 * page, requests), rng.choice([0, -5], requests))
    after[::5] = 0
    tables = rng.permutation(requests * width).reshape(requests, width)
    tables[rng.random(tables.shape) < 0.1] = -1                      # pages that a step did not get
    free = np.arange(requests * width + 50) + 10 ** 6
    taken = requests * width + 20
    want, back = tables.copy(), []
    for r in range(requests):
        for p in range(min(-(-max(after[r], 0) // page), width), min(-(-before[r] // page), width)):
            if tables[r, p] >= 0:
                back.append(tables[r, p])
            want[r, p] = -1
    got_tables, got_free, given = _ints(tables), _ints(free), _ints([taken])
    versions = got_tables._version, got_free._version
    left = release_pages(_ints(before), _ints(after), got_tables, got_free, given, page_size=page)
    assert got_tables._version > versions[0] and got_free._version > versions[1]
    free[taken - len(back):taken] = back
    assert int(left) == taken - len(back) and int(given) == taken
    assert np.array_equal(got_tables.cpu().numpy(), want) and np.array_equal(got_free.cpu().numpy(), free)
    # Fewer taken than come back: what has no place is dropped, in bounds.
    left = release_pages(_ints(before), _ints(np.zeros(requests)), _ints(tables), got_free, _ints([0]), page_size=page)
    assert int(left) == 0 and np.array_equal(got_free.cpu().numpy(), free)


@pytest.mark.gpu
def test_released_pages_are_taken_again():
    tables, free, taken = _ints(np.full((2, 6), -1)), _ints(np.arange(12)), _ints([0])
    plan = plan_step(_ints([0, 0]), _ints([70, 150]), tables, free, taken, page_size=32, max_tokens=256)
    plan.check()
    assert tables.tolist() == [[0, 1, 2, -1, -1, -1], [3, 4, 5, 6, 7, -1]]
    left = release_pages(plan.lengths, _ints([33, 0]), tables, free, plan.taken, page_size=32)
    assert tables.tolist() == [[0, 1] + [-1] * 4, [-1] * 6] and int(left) == 2
    plan = plan_step(_ints([33, 0]), _ints([0, 180]), tables, free, left, page_size=32, max_tokens=256)
    plan.check()
    assert tables.tolist() == [[0, 1] + [-1] * 4, [2, 3, 4, 5, 6, 7]] and int(plan.taken) == 8


def _model(hidden, heads, dim, ids, axes, generator):
    """A random attention layer between an embedding and a choice of ids."""
    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=generator)
    return {"embed": normal(ids, hidden).half(), "qkv": (normal(hidden, 4 * heads * dim) * hidden ** -0.5).half(),
            "out": (normal(2 * heads * dim, ids) * 0.2).half(), "heads": heads, "dim": dim, "axes": axes}


def _layer(model, tokens, plan, positions, pages, tables, frequencies, trees, most):
    heads, dim = model["heads"], model["dim"]
    x = (model["embed"][tokens] @ model["qkv"]).view(-1, 4 * heads, dim)
    at = positions if model["axes"] is None else positions.expand(3, -1).contiguous()
    q = append_tokens(pages, x[:, 2 * heads:3 * heads], x[:, 3 * heads:], plan.slots, q=x[:, :2 * heads], positions=at,
                      frequencies=frequencies, axes=model["axes"])
    out = cache_attention(q, pages, tables, plan.starts, plan.lengths, max_new=most, trees=trees)
    return (out.flatten(1).float() @ model["out"].float()).argmax(1)


@pytest.mark.gpu
@pytest.mark.parametrize("mixed", [False, True])
def test_decoding_with_trees_is_decoding(mixed):
    """Greedy decoding with random trees of drafts, part of which are right,
    makes the tokens that single steps make; pages come and go."""
    generator = torch.Generator(device="cuda").manual_seed(5)
    rng = np.random.default_rng(5)
    requests, ids, page, width, steps = 3, 11, 32, 8, 25
    axes = rotary_axes((12, 10, 10), interleaved=True) if mixed else None
    model = _model(128, 2, 64, ids, axes, generator)
    frequencies, _ = rotary_frequencies(64)

    def start():
        pages = cache_pages(requests * width + 4, page, 2, 64)
        return pages, _ints(np.full((requests, width), -1)), _ints(np.arange(requests * width + 4)), _ints([0])

    # One token a step.
    pages, tables, free, taken = start()
    cached, token, told = _ints([0] * requests), _ints([1, 2, 3], torch.int64), []
    for _ in range(4 * steps):
        plan = plan_step(cached, _ints([1] * requests), tables, free, taken, page_size=page, max_tokens=requests)
        told.append(token.tolist())
        token = _layer(model, token, plan, plan.positions, pages, tables, frequencies, None, 1)
        cached, taken = plan.lengths, plan.taken
    told = np.array(told).T

    # Trees whose tokens are the right ones more often than not.
    pages, tables, free, taken = start()
    cached, held = _ints([0] * requests), [0] * requests
    token = [1, 2, 3]
    wins = 0
    for _ in range(steps):
        new = [int(n) for n in rng.integers(1, 9, requests)]
        parents = _forest(new, rng)
        paths, tokens, at = _paths(new, parents), [], 0
        for r, n in enumerate(new):
            parents[at] = -1
            for i in range(n):
                right = told[r][held[r] + len(paths[at + i]) - 1]
                tokens.append(token[r] if i == 0 else int(right) if rng.random() < 0.7 else int(rng.integers(0, ids)))
            at += n
        pad = -(-len(parents) // 8) * 8 - len(parents)
        given = _ints(tokens + [0] * pad, torch.int64), _ints(parents + [-1] * pad)
        plan = plan_step(cached, _ints(new), tables, free, taken, page_size=page, max_tokens=len(parents) + pad)
        tree = plan_tree(given[1], plan.starts, plan.lengths, max_new=8)
        choices = _layer(model, given[0], plan, tree.positions, pages, tables, frequencies, tree.masks, 8)
        kept = accept_drafts(given[0], choices, given[1], plan.starts, plan.lengths)
        taken = release_pages(plan.lengths, kept.lengths, tables, free, plan.taken, page_size=page)
        keep_tokens(pages, plan.slots, plan.starts, kept.places)
        plan.check()
        places, starts = kept.places.tolist(), plan.starts.tolist()
        for r in range(requests):
            path = [tokens[t] for t in range(starts[r], starts[r + 1]) if places[t] >= 0]
            assert path == told[r][held[r]:held[r] + len(path)].tolist()
            held[r] += len(path)
            wins += len(path) - 1
        cached, token = kept.lengths, kept.next.tolist()
        assert cached.tolist() == held and int(taken) == sum(-(-n // page) for n in held)
        assert token == [told[r][held[r]] for r in range(requests)]
    assert wins > 0


@pytest.mark.gpu
def test_step_of_trees_in_a_graph():
    """A captured step of trees replays with new tokens, parents and lengths; two
    captured steps and eager ones share nothing."""
    torch.manual_seed(1)
    requests, heads, dim, page, new = 3, 2, 128, 32, 6
    total = requests * new
    pages = cache_pages(30, page, heads, dim)
    tables = torch.full((requests, 8), -1, dtype=torch.int32, device="cuda")
    free, taken, cached = _ints(np.arange(30)), _ints([0]), _ints([0] * requests)
    fresh, parents = _ints([new] * requests), _ints([-1, 0, 0, 1, 1, 2] * requests)
    tokens, choices = (torch.zeros(total, dtype=torch.int64, device="cuda") for _ in range(2))
    frequencies, _ = rotary_frequencies(dim)
    x = torch.randn(total, 8 * heads, dim, device="cuda", dtype=torch.bfloat16)

    def step(pages, tables, free):
        plan = plan_step(cached, fresh, tables, free, taken, page_size=page, max_tokens=total)
        tree = plan_tree(parents, plan.starts, plan.lengths, max_new=new)
        q = append_tokens(pages, x[:, 6 * heads:7 * heads], x[:, 7 * heads:], plan.slots, q=x[:, :6 * heads], positions=tree.positions,
                          frequencies=frequencies)
        out = cache_attention(q, pages, tables, plan.starts, plan.lengths, max_new=new, trees=tree.masks)
        kept = accept_drafts(tokens, choices, parents, plan.starts, plan.lengths)
        left = release_pages(plan.lengths, kept.lengths, tables, free, plan.taken, page_size=page)
        keep_tokens(pages, plan.slots, plan.starts, kept.places)
        return out, kept.lengths, left

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pages.clone(), tables.clone(), free.clone())
    torch.cuda.current_stream().wait_stream(side)
    graphs, state, out = [], [], []
    for _ in range(2):
        state.append((pages.clone(), tables.clone(), free.clone()))
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out.append(step(*state[-1]))
    eager = pages.clone(), tables.clone(), free.clone()
    for i in range(12):
        x.copy_(torch.randn_like(x))
        tokens.copy_(torch.randint(0, 2, (total,), device="cuda")), choices.copy_(torch.randint(0, 2, (total,), device="cuda"))
        parents.copy_(_ints([-1, 0, 0, 1, 1 + i % 2, i % 4] * requests))
        want = step(*eager)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, held in zip(out, state):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
            assert all(torch.equal(a, b) for a, b in zip(held, eager)), i
        cached.copy_(want[1]), taken.copy_(want[2])


def test_refuses_cpu_tensors_and_sizes():
    one, many = torch.zeros(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        plan_tree(many, one, one, max_new=4)
    for most in (0, 1025):
        with pytest.raises(ValueError, match="max_new"):
            plan_tree(many, one, one, max_new=most)
    with pytest.raises(RuntimeError, match="GPU"):
        accept_drafts(many, many, many, one, one)
    pages = cache_pages(2, 32, 1, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU"):
        keep_tokens(pages, many.long(), one, many)
    with pytest.raises(RuntimeError, match="GPU"):
        release_pages(one, one, torch.zeros(1, 1, dtype=torch.int32), many, one, page_size=32)
    lib = _native.load_library()
    assert lib.exl3_plan_tree(None, None, None, 0, 4, 1, None, None, None) == 1
    assert lib.exl3_plan_tree(None, None, None, 4097, 4, 1, None, None, None) == 1
    assert lib.exl3_plan_tree(None, None, None, 1, 1 << 40, 1, None, None, None) == 1
    for words in (0, 17):
        assert lib.exl3_plan_tree(None, None, None, 1, 4, words, None, None, None) == 1
    assert lib.exl3_accept_drafts(None, None, 0, None, None, None, None, 0, 4, None, None, None, None) == 1
    assert lib.exl3_cache_keep(None, 4, 33, 1, 64, None, None, None, 1, 4, None) == 1
    assert lib.exl3_cache_keep(None, 4, 32, 1, 65, None, None, None, 1, 4, None) == 1
    assert lib.exl3_cache_keep(None, 4, 32, 1, 64, None, None, None, 0, 4, None) == 1
    assert lib.exl3_release_pages(None, None, 1, None, 4, 31, None, 4, None, None, None) == 1
    assert lib.exl3_release_pages(None, None, 1, None, 0, 32, None, 4, None, None, None) == 1
    assert lib.exl3_release_pages(None, None, 1, None, 1, 32, None, -1, None, None, None) == 1
    for masks_words in (0, 17):
        assert lib.exl3_cache_attention_trees(None, 0, 0, None, 1, 1, 1, None, 1, 32, 1, 64, None, 1, None, None, 1, 64, masks_words,
                                              1.0, 1, 1, None, 1 << 40, None) == 1


@pytest.mark.gpu
def test_refusals():
    parents, starts, lengths = _ints([-1, 0, 0]), _ints([0, 3]), _ints([9])
    for args in ((parents.long(), starts, lengths), (parents, starts.long(), lengths), (parents, starts, lengths.long()),
                 (parents, starts, _ints([9, 9])), (parents.cpu(), starts, lengths), (parents[::2], starts, lengths),
                 (parents, starts[:1], lengths[:0]), (parents, starts.view(1, 2), lengths)):
        with pytest.raises(RuntimeError):
            plan_tree(*args, max_new=4)
    ids = _ints([1, 2, 3])
    for args, more in (((ids, ids.long(), parents, starts, lengths), {}), ((ids.float(), ids.float(), parents, starts, lengths), {}),
                       ((ids[:2], ids, parents, starts, lengths), {}), ((ids, ids[:2], parents, starts, lengths), {}),
                       ((ids, ids, parents.long(), starts, lengths), {}), ((ids, ids, parents, starts, lengths), dict(certain=ids)),
                       ((ids, ids, parents, starts, lengths), dict(certain=lengths.long()))):
        with pytest.raises(RuntimeError):
            accept_drafts(*args, **more)
    pages = cache_pages(2, 32, 2, 64)
    slots = ids.long()
    for args in ((pages[0], slots, starts, parents), (pages, ids, starts, parents), (pages, slots, starts.long(), parents),
                 (pages, slots, starts, parents[:2]), (pages, slots, starts, parents.long()), (pages, slots, starts.cpu(), parents)):
        with pytest.raises(RuntimeError):
            keep_tokens(*args)
    tables = _ints([[0, 1]])
    for args, more in (((lengths, lengths, tables.long(), ids, lengths), {}), ((ids, lengths, tables, ids, lengths), {}),
                       ((lengths, ids, tables, ids, lengths), {}), ((lengths, lengths, tables, slots, lengths), {}),
                       ((lengths, lengths, tables, ids, ids), {}), ((lengths, lengths, tables, ids, lengths), dict(page_size=48))):
        with pytest.raises(RuntimeError):
            release_pages(*args, **{"page_size": 32, **more})
    q = torch.zeros(3, 2, 64, device="cuda", dtype=torch.float16)
    for trees in (ids, ids.long(), torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.zeros(3, 17, dtype=torch.int64, device="cuda"),
                  torch.zeros(3, 0, dtype=torch.int64, device="cuda"), torch.zeros(3, 1, dtype=torch.int64),
                  torch.zeros(3, 2, dtype=torch.int64, device="cuda")[:, :1], torch.zeros(3, 1, dtype=torch.int32, device="cuda")):
        with pytest.raises(RuntimeError, match="trees"):
            cache_attention(q, pages, tables, starts, lengths, trees=trees)


@pytest.mark.gpu
def test_example_decodes_drafted_trees():
    """A step keeps one to three of a tree's five tokens."""
    import importlib.util
    from .conftest import REPO_ROOT
    spec = importlib.util.spec_from_file_location("serve_drafts", REPO_ROOT / "examples" / "serve_drafts.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    answers, steps = example.serve(tokens=10)
    assert len(answers) == 3 and min(map(len, answers)) >= 10
    for answer in answers:
        assert steps < len(answer) <= 3 * steps + 1
        assert all(0 <= token < example.VOCABULARY for token in answer)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, most, requests", [(64, 25, 9), (64, 40, 5), (128, 40, 7), (128, 45, 9), (128, 17, 1), (256, 12, 6), (256, 70, 2)])
def test_ragged_batches(dim, most, requests, dtype):
    """Requests of one token to `most`, four heads to a kv head: waves of 32 rows,
    blocks of which some waves have no rows, and those of few rows beside them; at
    last with a NaN in the first request's newest values."""
    rng = np.random.default_rng(dim + most)
    new = [most, *rng.integers(1, most + 1, requests - 1).tolist()]
    lengths = [int(n + rng.integers(0, 400)) for n in new]
    parents = _forest(new, rng)
    cache = ref.Cache(sum(-(-n // 64) for n in lengths) + 1, 64, 2, dim, rng)
    tables = _tables(lengths, 64, 8, cache.shape[0], rng)
    q = torch.from_numpy(rng.normal(size=(sum(new), 8, dim)) * 2).to(dtype)
    _check(q, cache, 64, tables, new, lengths, _paths(new, parents), 2, dtype, max_new=most, group=4)
    _check(q, cache, 64, tables, new, lengths, _paths(new, parents), 2, dtype, window=100, group=4)
    cache.scales[1][tables[0][(lengths[0] - 1) // 64] * 64 + (lengths[0] - 1) % 64, 1, 0] = np.nan
    got = _check(q, cache, 64, tables, new, lengths, _paths(new, parents), 2, dtype, max_new=most, group=4)
    assert torch.isnan(got).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim, requests, new, hint, heads", [
    (128, 1, 3, 3, 8), (128, 1, 30, 30, 8), (64, 70, 20, 24, 4), (128, 40, 25, 40, 16), (256, 5, 60, 64, 2), (64, 1, 900, 900, 16)])
def test_calls_stay_within_their_workspace(dim, requests, new, hint, heads):
    """Bytes past the asked size keep what they hold, and less is refused."""
    lib = _native.load_library()
    tokens, context, group, words = requests * new, new + 700, 4, -(-hint // 64)
    width = -(-context // 64)
    pages = torch.zeros(requests * width, heads, 2, 36 * dim, dtype=torch.uint8, device="cuda")
    tables = torch.arange(requests * width, dtype=torch.int32, device="cuda").view(requests, width)
    starts = torch.arange(requests + 1, dtype=torch.int32, device="cuda") * new
    lengths = torch.full((requests,), context, dtype=torch.int32, device="cuda")
    masks = torch.full((tokens, words), -1, dtype=torch.int64, device="cuda")
    q = torch.randn(tokens, group * heads, dim, device="cuda").half()
    size = lib.exl3_cache_attention_trees_workspace(tokens, group * heads, heads, dim, requests, hint)
    held = torch.full((size + (1 << 20),), 173, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 3.0)

    def call(bytes_):
        return lib.exl3_cache_attention_trees(
            q.data_ptr(), q.stride(0), dim, out.data_ptr(), tokens, group * heads, 1, pages.data_ptr(), pages.shape[0], 64, heads,
            dim, tables.data_ptr(), width, starts.data_ptr(), lengths.data_ptr(), requests, masks.data_ptr(), words, 1.0,
            2 ** 31 - 1, hint, held.data_ptr(), bytes_, torch.cuda.current_stream().cuda_stream)

    assert call(size) == 0 and (held[size:] == 173).all()
    assert not out.any()  # a cache of zeros
    assert call(size - 1) != 0
