"""Rotary positions of several axes against their 64-bit definition: forward,
gradient, tangents, into a cache, and refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

from exl3_intel_arc_quantizer_amd.kv_cache import append_tokens, cache_pages, read_tokens
from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_axes, rotary_frequencies

from .test_gpu_rotary import _bound


def _turned(x, positions, axes, frequencies, layout, magnitude=1.0, sign=1.0):
    """float64 (tokens, heads, dim), pair by pair."""
    y = torch.as_tensor(x).double().numpy().copy()
    n = len(frequencies)
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        at = positions[axes[i]].double().numpy() if 0 <= axes[i] < len(positions) else np.zeros(len(y))
        angle = sign * at[:, None] * frequencies[i]
        c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
        u, w = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def test_axes_of_sections():
    assert rotary_axes((2, 1, 3), device="cpu").tolist() == [0, 0, 1, 2, 2, 2]
    assert rotary_axes((2, 1, 3), interleaved=True, device="cpu").tolist() == [0, 1, 2, 0, 2, 2]
    assert rotary_axes([24, 20, 20], interleaved=True, device="cpu").tolist() == [0, 1, 2] * 20 + [0] * 4
    assert rotary_axes((0, 4), device="cpu").tolist() == [1] * 4 and rotary_axes([3], device="cpu").dtype == torch.int32
    for bad in ((), (0, 0), (3, -1)):
        with pytest.raises(ValueError, match="sections"):
            rotary_axes(bad, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens, q_heads, k_heads, dim, sections, mixed, first", [
    (1, 32, 8, 128, (16, 24, 24), False, 4000), (7, 4, 1, 64, (12, 10, 10), True, 999_983), (131, 3, 3, 256, (16, 16), False, 0),
    (5, 2, 2, 80, (40,), False, 17), (3, 1, 2, 10, (1, 1, 1), False, 5), (300, 2, 1, 64, (8, 8, 8, 8), True, 0)])
def test_matches_definition(tokens, q_heads, k_heads, dim, sections, mixed, first, dtype, layout):
    g = torch.Generator().manual_seed(tokens * dim)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dtype) for h in (q_heads, k_heads))
    pairs = sum(sections)
    freq, _ = rotary_frequencies(2 * pairs, base=500000.0, device="cpu")
    axes = rotary_axes(sections, interleaved=mixed, device="cpu")
    positions = torch.randint(0, 5000, (len(sections), tokens), generator=g) + first
    for at in (positions, positions.int()):
        got = apply_rotary(q.cuda(), k.cuda(), at.cuda(), freq.cuda(), layout=layout, magnitude=1.25, axes=axes.cuda())
        for x, y in zip((q, k), got):
            want = _turned(x.double(), positions, axes, freq.numpy(), layout, 1.25)
            off = np.abs(y.cpu().double().numpy() - want)
            assert y.dtype == dtype and (off <= _bound(x.double(), want, dtype, pairs, layout, 1.25)).all()
            assert torch.equal(y.cpu()[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.gpu
def test_one_axis_is_as_before():
    x = torch.randn(9, 6, 64, device="cuda", dtype=torch.bfloat16)
    freq, _ = rotary_frequencies(64)
    at = torch.arange(9, device="cuda") * 1001
    want = apply_rotary(x[:, :4], x[:, 4:], at, freq)
    for axes, positions in (([0] * 32, at[None]), ([1] * 32, torch.stack([at * 3, at])), ([2, 0, 1] * 10 + [2, 0], at.expand(3, 9).contiguous())):
        axes = torch.tensor(axes, dtype=torch.int32, device="cuda")
        got = apply_rotary(x[:, :4], x[:, 4:], positions, freq, axes=axes)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Axes that there are none of do not turn.
    axes = torch.tensor([0] * 16 + [-1] * 8 + [1, 7, 1 << 30, -1 << 31] * 2, dtype=torch.int32, device="cuda")
    got = apply_rotary(x, None, at[None], freq, axes=axes)[0]
    still = [*range(16, 32), *range(48, 64)]
    assert torch.equal(got[..., still], x[..., still]) and torch.equal(got[:, :4, :16], want[0][..., :16])
    y = x.clone()
    apply_rotary(y, None, at[None], freq, axes=axes, out=(y, None))
    assert torch.equal(y, got)
    assert apply_rotary(x[:0], None, at[None, :0], freq, axes=axes)[0].shape == (0, 6, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_and_tangent(layout):
    g = torch.Generator().manual_seed(3)
    q, k, dq, dk = (torch.randn(6, h, 32, generator=g) for h in (3, 1, 3, 1))
    freq, _ = rotary_frequencies(24, device="cpu")
    axes = rotary_axes((5, 4, 3), interleaved=True, device="cpu")
    at = torch.randint(0, 900, (3, 6), generator=g)
    args = at.cuda(), freq.cuda()
    more = dict(layout=layout, magnitude=0.5, axes=axes.cuda())
    a, b = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = apply_rotary(a, b, *args, **more)
    grads = torch.autograd.grad(out, (a, b), (dq.cuda(), dk.cuda()), create_graph=True)
    for x, y in zip((dq, dk), grads):
        want = _turned(x.double(), at, axes, freq.numpy(), layout, 0.5, -1.0)
        assert (np.abs(y.detach().cpu().double().numpy() - want) <= _bound(x, want, torch.float32, 12, layout, 1.0)).all()
    # Differences: the rotation is linear, so (f(q + d) - f(q)) . g = d . grad up
    # to rounding: 6e-7 of |x1| + |x2| in each of two values, over 6 * 3 * 32
    # terms of |g| < 4, |x| + |d| < 8.
    d = torch.randn(6, 3, 32, generator=g).cuda()
    with torch.no_grad():
        moved, _ = apply_rotary(a + d, b, *args, **more)
        still, _ = apply_rotary(a, b, *args, **more)
        left, right = ((moved - still).double() * dq.cuda()).sum(), (d.double() * grads[0]).sum()
    assert abs(float(left - right)) < 6 * 3 * 32 * 2 * 6e-7 * 8 * 4
    with fwd.dual_level():
        dual = fwd.make_dual(q.cuda(), d)
        tangent = fwd.unpack_dual(apply_rotary(dual, b.detach(), *args, **more)[0]).tangent
    assert torch.equal(tangent, apply_rotary(d, None, *args, **more)[0])
    # Axes written to after the forward pass: no gradient of others.
    kept = axes.cuda()
    out = apply_rotary(a, b, *args, layout=layout, axes=kept)
    kept.zero_()
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(out, (a, b), (dq.cuda(), dk.cuda()))


@pytest.mark.gpu
def test_backward_in_a_graph():
    """Forward and backward captured, an eager graph of the same leaves alive."""
    q = torch.randn(40, 4, 64, device="cuda").requires_grad_()
    freq, _ = rotary_frequencies(64)
    axes, at = rotary_axes((12, 10, 10)), torch.randint(0, 99, (3, 40), device="cuda")
    grad = torch.randn_like(q)
    leaf = q.detach().requires_grad_()
    kept = apply_rotary(q, None, at, freq, axes=axes)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(apply_rotary(leaf, None, at, freq, axes=axes)[0], leaf, grad)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(apply_rotary(leaf, None, at, freq, axes=axes)[0], leaf, grad)[0]
    for _ in range(4):
        grad.copy_(torch.randn_like(grad))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(kept, q, grad, retain_graph=True)[0]
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens", [5, 2100])
def test_append_turns_by_axes(tokens, layout):
    """The cache's side of a step: as turning first and appending then. The turned
    keys stay in 32 bits between, as float32 rows do."""
    heads, dim, page = 2, 64, 32
    x = torch.randn(tokens, 5, dim, device="cuda")
    freq, _ = rotary_frequencies(dim)
    axes, at = rotary_axes((12, 10, 10)), torch.randint(0, 9999, (3, tokens), device="cuda", dtype=torch.int32)
    slots = torch.randperm(-(-tokens // page) * page, device="cuda")[:tokens]
    one, other = (cache_pages(-(-tokens // page), page, heads, dim) for _ in range(2))
    q = append_tokens(one, x[:, 1:3], x[:, 3:], slots, q=x[:, :1], positions=at, frequencies=freq, layout=layout, axes=axes)
    turned, keys = apply_rotary(x[:, :1], x[:, 1:3], at, freq, layout=layout, axes=axes)
    append_tokens(other, keys, x[:, 3:], slots)
    assert torch.equal(q, turned) and torch.equal(one, other)
    assert torch.equal(read_tokens(one, slots)[0], read_tokens(other, slots)[0])


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 2, 32, device="cuda")
    freq, _ = rotary_frequencies(32)
    axes, at = rotary_axes((8, 8)), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for positions, given in ((at, None), (at[0], axes), (at, axes.long()), (at, axes[:8]), (at, axes.cpu()), (at.t().contiguous(), axes),
                             (at.float(), axes), (at.cpu(), axes), (at[:0], axes), (at[:, ::2], axes), (at[None], axes),
                             (torch.zeros(8, 2, dtype=torch.int32, device="cuda").t()[:, ::2], axes)):
        with pytest.raises(RuntimeError):
            apply_rotary(x, None, positions, freq, axes=given)
    pages = cache_pages(1, 32, 2, 64)
    k = torch.zeros(4, 2, 64, device="cuda")
    slots = torch.arange(4, device="cuda")
    with pytest.raises(RuntimeError, match="axes"):
        append_tokens(pages, k, k, slots, axes=axes)
    with pytest.raises(RuntimeError):
        append_tokens(pages, k, k, slots, positions=at[0], frequencies=freq, axes=axes)
