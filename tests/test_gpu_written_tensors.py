"""Tensors that the operators write in place: what torch records or saves, and
outputs that share memory."""

from __future__ import annotations

import pytest
import torch

from exl3_intel_arc_quantizer_amd.rotary import apply_rotary


def _given(tokens=6, heads=4, dim=32, device="cuda"):
    x = torch.randn(tokens, heads, dim, device=device)
    at = torch.arange(tokens, device=device) + 3
    freq = torch.full((dim // 2,), 0.25, dtype=torch.float64, device=device)
    return x, at, freq


def _refuses_recorded_out(device):
    import torch.autograd.forward_ad as fwd
    q, at, freq = _given(device=device)
    k = q[:, :1].clone()
    leaf = torch.zeros_like(q).requires_grad_()
    of_graph = leaf * 2
    before = of_graph.detach().clone()
    for out in ((leaf, torch.empty_like(k)), (of_graph, torch.empty_like(k)),
                (torch.empty_like(q), torch.zeros_like(k).requires_grad_())):
        with pytest.raises(RuntimeError, match="out cannot be"):
            apply_rotary(q, k, at, freq, out=out)
    with fwd.dual_level():
        dual = fwd.make_dual(torch.zeros_like(q), torch.ones_like(q))
        with pytest.raises(RuntimeError, match="out cannot be"):
            apply_rotary(q, None, at, freq, out=(dual, None))
    assert torch.equal(of_graph, before) and not leaf.any()
    return q, k, at, freq, leaf


def test_recorded_out_is_refused_before_any_device():
    _refuses_recorded_out("cpu")


@pytest.mark.gpu
def test_recorded_out_is_refused():
    q, k, at, freq, leaf = _refuses_recorded_out("cuda")
    with torch.no_grad():  # as torch's own in-place operations
        apply_rotary(q, None, at, freq, out=(leaf, None))
    assert torch.equal(leaf, apply_rotary(q, None, at, freq)[0])
