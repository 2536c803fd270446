"""Arguments at the ends of their ranges."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import _native
from exl3_intel_arc_quantizer_amd.kv_cache import append_tokens, cache_attention, cache_pages, read_tokens
from exl3_intel_arc_quantizer_amd.rotary import apply_rotary

from . import cache_ref as ref


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


@pytest.fixture
def much_memory():
    """Frees what a test of many tokens takes."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("pairs, dtype", [(8, torch.float16), (3, torch.bfloat16)])
def test_rotary_of_more_tokens_than_a_launch_has_blocks(pairs, dtype, much_memory):
    tokens = 2 ** 24 + 5
    at = torch.arange(tokens, device="cuda", dtype=torch.int32) % 97
    freq = torch.linspace(0.1, 1.0, pairs, dtype=torch.float64, device="cuda")
    row = torch.randn(1, 1, 16, device="cuda", dtype=dtype)
    few, _ = apply_rotary(row.expand(97, 1, 16), None, at[:97], freq)
    got, more = apply_rotary(row.expand(tokens, 1, 16), row.expand(tokens, 1, 16), at.long(), freq)
    assert torch.equal(got, few[at]) and torch.equal(got, more)


@pytest.mark.gpu
def test_append_and_read_of_more_tokens_than_a_launch_has_blocks(much_memory):
    """All slots but a few lie outside the cache; rows of the others are never
    looked at and hold what they hold."""
    tokens = 2 ** 27 + 9
    some = torch.tensor([0, 2 ** 26 - 1, 2 ** 26, 2 ** 26 + 7, 2 ** 27 - 1, 2 ** 27, 2 ** 27 + 8], device="cuda")
    x = torch.empty(tokens, 1, 64, device="cuda", dtype=torch.float16)
    rows = torch.randn(len(some), 1, 64, device="cuda", dtype=torch.float16)
    x[some] = rows
    slots = torch.full((tokens,), -1, device="cuda")
    slots[some] = torch.tensor([5, 70, 3, 127, 64, 0, 31], device="cuda")
    at = torch.zeros(tokens, device="cuda", dtype=torch.int32)
    at[some] = torch.arange(len(some), device="cuda", dtype=torch.int32) * 11
    freq = torch.linspace(0.1, 1.0, 16, dtype=torch.float64, device="cuda")
    pages, small = cache_pages(2, 64, 1, 64), cache_pages(2, 64, 1, 64)
    turned = append_tokens(pages, x, x, slots, q=x, positions=at, frequencies=freq)[some]
    want = append_tokens(small, rows, rows, slots[some], q=rows, positions=at[some], frequencies=freq)
    assert torch.equal(turned, want) and torch.equal(pages, small)
    del x, at
    many, few = read_tokens(pages, slots), read_tokens(pages, slots[some])
    for a, b in zip(many, few):
        assert torch.equal(a[some], b)
        assert not a[[1, 2 ** 26 - 2, 2 ** 26 + 1, 2 ** 27 + 7]].any()


@pytest.mark.gpu
def test_windows_and_hints_past_64_bits():
    """A window no context reaches is no window, however it is written."""
    rng = np.random.default_rng(2)
    cache = ref.Cache(4, 32, 1, 64, rng)
    args = (torch.from_numpy(cache.bytes()).cuda(), _ints([[3, 0, 1]]), _ints([0, 5]), _ints([90]))
    q = torch.randn(5, 2, 64, device="cuda", dtype=torch.float16)
    want = cache_attention(q, *args)
    for window in (90, 2 ** 31, 2 ** 32 + 1, 2 ** 63, 2 ** 64 + 1, 2 ** 70):
        assert torch.equal(cache_attention(q, *args, window=window), want), window
    for hint in (5, 2 ** 31, 2 ** 32, 2 ** 63, 2 ** 64 + 1):
        assert torch.equal(cache_attention(q, *args, max_new=hint), want), hint


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, requests, tokens, hint, heads", [
    (128, 1, 3000, 3000, 16), (64, 1, 1, 1, 2), (128, 40, 40, 40, 16), (128, 1, 8192, 8192, 16), (128, 70, 70, 70, 16),
    (256, 5, 600, 200, 2), (64, 300, 900, 60, 4)])
def test_calls_stay_within_their_workspace(dim, requests, tokens, hint, heads, dtype):
    """Bytes past the asked size keep what they hold; a step whose blocks are all
    dealt whole has partial results of its few-row requests at most."""
    lib = _native.load_library()
    new = tokens // requests
    context, page, group = new + 40, 64, 2
    width = -(-context // page)
    pages = torch.zeros(requests * width, heads, 2, 36 * dim, dtype=torch.uint8, device="cuda")
    tables = torch.arange(requests * width, dtype=torch.int32, device="cuda").view(requests, width)
    starts = torch.arange(requests + 1, dtype=torch.int32, device="cuda") * new
    lengths = torch.full((requests,), context, dtype=torch.int32, device="cuda")
    q = torch.randn(tokens, group * heads, dim, device="cuda").to(dtype)
    size = lib.exl3_cache_attention_workspace(tokens, group * heads, heads, dim, requests, hint)
    if (tokens, hint) in ((8192, 8192), (70, 70)):  # up to (64 + 1) 16 and (1 + 70) 16 blocks of 256 rows
        assert size <= lib.exl3_cache_attention_workspace(1, group * heads, heads, dim, 1, 1) + 16 * (requests + 2048)
    held = torch.full((size + (1 << 20),), 173, dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, 3.0)
    status = lib.exl3_cache_attention(
        q.data_ptr(), q.stride(0), dim, out.data_ptr(), tokens, group * heads, 1 if dtype == torch.float16 else 2,
        pages.data_ptr(), pages.shape[0], page, heads, dim, tables.data_ptr(), width, starts.data_ptr(),
        lengths.data_ptr(), requests, 1.0, 2 ** 31 - 1, hint, held.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert status == 0 and (held[size:] == 173).all()
    assert not out.any()  # a cache of zeros
    assert lib.exl3_cache_attention(
        q.data_ptr(), q.stride(0), dim, out.data_ptr(), tokens, group * heads, 1, pages.data_ptr(), pages.shape[0], page,
        heads, dim, tables.data_ptr(), width, starts.data_ptr(), lengths.data_ptr(), requests, 1.0, 2 ** 31 - 1, hint,
        held.data_ptr(), size - 1, torch.cuda.current_stream().cuda_stream) != 0
