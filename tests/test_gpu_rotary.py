"""Rotary positions against their 64-bit definition, with gradient, tangents,
strides and refusals."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd.rotary import apply_rotary, rotary_frequencies

from .cache_ref import turned

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _bound(x, y, dtype, pairs, layout, magnitude):
    """What |turned - y| may be: the angle's fraction of a turn rounded to
    float32 (2^-25 half turns: 9.4e-8 radians) and 2 units in each of sin and
    cos (2.4e-7), two products and a sum (1.8e-7 of each term): under 6e-7 of
    |x1| + |x2|, and the result's own rounding."""
    reach = np.abs(np.asarray(x, np.float64)).copy()
    a, b = (np.s_[..., :pairs], np.s_[..., pairs:2 * pairs]) if layout == "half" else \
        (np.s_[..., 0:2 * pairs:2], np.s_[..., 1:2 * pairs:2])
    both = reach[a] + reach[b]
    reach[a], reach[b] = both, both
    return 6e-7 * reach * max(magnitude, 1.0) + UNIT[dtype] * np.abs(y) + 2.0 ** -25 * (dtype == torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens, q_heads, k_heads, dim, pairs, first", [
    (1, 32, 8, 128, 64, 4000), (7, 4, 1, 64, 32, 999_983), (131, 3, 3, 256, 32, 0),
    (5, 2, 2, 80, 40, 17), (3, 1, 2, 10, 3, 5), (2, 2, 1, 7, 3, 1)])
def test_matches_definition(tokens, q_heads, k_heads, dim, pairs, first, dtype, layout):
    g = torch.Generator().manual_seed(tokens * dim + pairs)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dtype) for h in (q_heads, k_heads))
    freq, _ = rotary_frequencies(2 * pairs, base=500000.0, device="cpu")
    positions = torch.arange(tokens, dtype=torch.int64) * 3 + first
    got = apply_rotary(q.cuda(), k.cuda(), positions.cuda(), freq.cuda(), layout=layout, magnitude=1.25)
    for x, y in zip((q, k), got):
        want = turned(x.double(), positions, freq.numpy(), layout, 1.25)
        off = np.abs(y.cpu().double().numpy() - want)
        assert y.dtype == dtype and (off <= _bound(x.double(), want, dtype, pairs, layout, 1.25)).all()
        assert torch.equal(y.cpu()[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.gpu
def test_strides_out_and_int32_positions():
    x = torch.randn(9, 12, 64, device="cuda", dtype=torch.bfloat16)
    freq, _ = rotary_frequencies(64)
    at = torch.arange(9, device="cuda", dtype=torch.int32) + 100
    q, k = x[:, :8], x[:, 8:12]
    a, b = apply_rotary(q.contiguous(), k.contiguous(), at.long(), freq)
    c, d = apply_rotary(q, k, at, freq)
    assert torch.equal(a, c) and torch.equal(b, d)
    odd = torch.randn(9 * 12 * 65, device="cuda", dtype=torch.bfloat16)[1:9 * 12 * 64 + 1].view(9, 12, 64).copy_(x)
    e, f = apply_rotary(odd[:, :8], odd[:, 8:], at, freq)
    assert torch.equal(a, e) and torch.equal(b, f)
    alone, none = apply_rotary(q, None, at, freq)
    assert none is None and torch.equal(alone, a)
    y = x.clone()
    apply_rotary(y[:, :8], y[:, 8:], at, freq, out=(y[:, :8], y[:, 8:]))
    assert torch.equal(y, torch.cat([a, b], 1))
    empty = apply_rotary(x[:0, :8], x[:0, 8:], at[:0], freq)
    assert empty[0].shape == (0, 8, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_and_tangent(layout):
    g = torch.Generator().manual_seed(3)
    q, k, dq, dk = (torch.randn(6, h, 32, generator=g) for h in (3, 1, 3, 1))
    freq, _ = rotary_frequencies(24, device="cpu")
    at = torch.arange(6) + 50
    args = at.cuda(), freq.cuda()
    a, b = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = apply_rotary(a, b, *args, layout=layout, magnitude=0.5)
    grads = torch.autograd.grad(out, (a, b), (dq.cuda(), dk.cuda()))
    for x, y in zip((dq, dk), grads):
        want = turned(x.double(), at, freq.numpy(), layout, 0.5, -1.0)
        assert (np.abs(y.cpu().double().numpy() - want) <= _bound(x, want, torch.float32, 12, layout, 1.0)).all()
    # Differences: the rotation is linear, so (f(q + d) - f(q)) . g = d . grad up
    # to rounding: 6e-7 of |x1| + |x2| in each of two values, over 6 * 3 * 32
    # terms of |g| < 4, |x| + |d| < 8.
    d = torch.randn(6, 3, 32, generator=g).cuda()
    with torch.no_grad():
        moved, _ = apply_rotary(a + d, b, *args, layout=layout, magnitude=0.5)
        still, _ = apply_rotary(a, b, *args, layout=layout, magnitude=0.5)
    lhs = ((moved.double() - still.double()) * dq.cuda().double()).sum()
    rhs = (d.double() * grads[0].double()).sum()
    assert abs(float(lhs - rhs)) <= 576 * 2 * 6e-7 * 16 * 4
    # Only k, a broadcast gradient, and forward mode.
    only = torch.autograd.grad(apply_rotary(q.cuda(), b, *args, layout=layout)[1].sum(), b)[0]
    want = turned(np.ones(k.shape), at, freq.numpy(), layout, 1.0, -1.0)
    assert (np.abs(only.cpu().double().numpy() - want) <= _bound(np.ones(k.shape), want, torch.float32, 12, layout, 1.0)).all()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        y, _ = apply_rotary(fwd.make_dual(q.cuda(), dq.cuda()), None, *args, layout=layout)
        tangent = fwd.unpack_dual(y).tangent
    assert torch.equal(tangent, apply_rotary(dq.cuda(), None, *args, layout=layout)[0])


def test_frequencies():
    f, m = rotary_frequencies(8, base=10000.0, device="cpu")
    assert m == 1.0 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14)
    assert np.allclose(rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")[0], f / 4, rtol=1e-14)
    b, _ = rotary_frequencies(8, scaling="base", factor=4.0, device="cpu")
    assert np.allclose([b[0], b[-1]], [f[0], f[-1] / 4], rtol=1e-12)
    r, m = rotary_frequencies(128, scaling="ramp", factor=8.0, original_length=4096, device="cpu")
    f, _ = rotary_frequencies(128, device="cpu")
    turns = 4096 * f / (2 * np.pi)
    assert np.array_equal(r[turns > 40], f[turns > 40]) and np.allclose(r[turns < 0.8], f[turns < 0.8] / 8)
    assert ((r <= f) & (r >= f / 8 * (1 - 1e-12))).all() and abs(m - (0.1 * np.log(8.0) + 1)) < 1e-15
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="ramp"), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=2, scaling="base", factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(device="cpu", **bad)


def test_refuses_cpu_tensors_and_layouts():
    q = torch.zeros(2, 1, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        apply_rotary(q, None, torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="layout"):
        apply_rotary(q, None, torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.float64), layout="x")


@pytest.mark.gpu
def test_refusals():
    q, k = torch.zeros(4, 2, 16, device="cuda"), torch.zeros(4, 1, 16, device="cuda")
    at = torch.zeros(4, dtype=torch.int32, device="cuda")
    f = torch.ones(8, dtype=torch.float64, device="cuda")
    for args in ((q[0], k, at, f), (q, k.half(), at, f), (q, k[:3], at, f), (q, k, at[:3], f), (q, k, at.float(), f),
                 (q, k, at, f.float()), (q, k, at, torch.ones(9, dtype=torch.float64, device="cuda")), (q, k, at, f[:0]),
                 (q.transpose(1, 2), None, at, f), (q.double(), None, at, f), (q, k.cpu(), at, f),
                 (q, torch.zeros(4, 1, 8, device="cuda"), at, f)):
        with pytest.raises(RuntimeError):
            apply_rotary(*args)
    with pytest.raises(RuntimeError, match="out"):
        apply_rotary(q.requires_grad_(), k, at, f, out=(torch.empty_like(q), torch.empty_like(k)))


@pytest.mark.gpu
def test_backward_sees_the_positions_of_the_forward_pass():
    q = torch.ones(4, 2, 16, device="cuda", requires_grad=True)
    at = torch.arange(4, device="cuda")
    f = torch.ones(8, dtype=torch.float64, device="cuda")
    y = apply_rotary(q, None, at, f)[0]
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="frequencies"):
        apply_rotary(q, None, at, f.clone().requires_grad_())
