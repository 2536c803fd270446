"""Derivatives of the rotary positions beyond the plain gradient."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

from exl3_intel_arc_quantizer_amd.rotary import apply_rotary

from .cache_ref import turned


def _given():
    g = torch.Generator().manual_seed(11)
    q, k, dq, dk = (torch.randn(5, h, 24, generator=g).cuda() for h in (3, 2, 3, 2))
    at = torch.arange(5, device="cuda") * 7 + 20
    return q, k, dq, dk, at, torch.logspace(0, -3, 8, dtype=torch.float64).cuda()


def _exact(x, at, freq, sign=1.0):
    return turned(x.double().cpu(), at.cpu(), freq.cpu().numpy(), "half", 0.75, sign)


def _bound(x):
    """Angles are taken in 64 bits; cosine and sine rounded to float32 once
    (2^-25 each: at most 1), two products and a sum (2^-24 of each term): under
    3 2^-24 of |x1| + |x2|. Doubled where it is applied twice."""
    return 3 * 2.0 ** -24 * 2 * np.abs(x.cpu().double().numpy()).max()


@pytest.mark.gpu
def test_tangent_of_queries_or_keys_alone():
    q, k, dq, dk, at, freq = _given()
    more = dict(magnitude=0.75)
    for which in (0, 1):
        with fwd.dual_level():
            given = [q, k]
            given[which] = fwd.make_dual(given[which], (dq, dk)[which])
            out = apply_rotary(*given, at, freq, **more)
            tangents = [fwd.unpack_dual(x).tangent for x in out]
            values = [fwd.unpack_dual(x).primal for x in out]
        d = (dq, dk)[which]
        assert np.abs(tangents[which].cpu().double().numpy() - _exact(d, at, freq)).max() <= _bound(d)
        other = tangents[1 - which]
        assert other is None or (other.shape == (q, k)[1 - which].shape and not other.any())
        for value, plain in zip(values, apply_rotary(q, k, at, freq, **more)):
            assert torch.equal(value, plain)


@pytest.mark.gpu
def test_tangent_of_a_gradient_of_queries_alone():
    """Forward over reverse: the gradient is linear in the output's, so its
    tangent is the gradient of the tangent."""
    q, k, dq, _, at, freq = _given()
    with fwd.dual_level():
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        out = apply_rotary(a, b, at, freq, magnitude=0.75)
        grad_q, grad_k = torch.autograd.grad(out, (a, b), (fwd.make_dual(torch.ones_like(q), dq), torch.ones_like(k)))
        tangent, none = fwd.unpack_dual(grad_q).tangent, fwd.unpack_dual(grad_k).tangent
    assert np.abs(tangent.cpu().double().numpy() - _exact(dq, at, freq, -1.0)).max() <= _bound(dq)
    assert none is None or not none.any()


@pytest.mark.gpu
def test_second_derivatives():
    q, k, dq, dk, at, freq = _given()
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    x, y = apply_rotary(a, b, at, freq, magnitude=0.75)
    gq, gk = torch.autograd.grad(((x ** 2).sum() + (y ** 2).sum()) / 2, (a, b), create_graph=True)
    # Of |R x|^2 / 2 the gradient is m^2 x on the turned values, x on the others.
    hq, hk = torch.autograd.grad((gq, gk), (a, b), (dq, dk))
    for d, h in ((dq, hq), (dk, hk)):
        want = d.clone()
        want[..., :16] *= 0.75 ** 2
        assert (h - want).abs().max() <= 2 * _bound(d)
