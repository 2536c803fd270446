"""Tensors that the operators write in place: what torch records or saves, and
outputs that share memory."""

from __future__ import annotations

import pytest
import torch

from exl3_intel_arc_quantizer_amd import _native
from exl3_intel_arc_quantizer_amd.kv_cache import append_tokens, cache_attention, cache_pages, plan_step, read_tokens
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
def test_out_that_is_no_tensor_is_refused():
    q, at, freq = _given()
    with pytest.raises(RuntimeError, match="out"):
        apply_rotary(q, None, at, freq, out=([0.0], None))
    with pytest.raises(RuntimeError, match="out"):
        apply_rotary(q, q[:, :1].clone(), at, freq, out=(torch.empty_like(q), None))


@pytest.mark.gpu
def test_recorded_out_is_refused():
    q, k, at, freq, leaf = _refuses_recorded_out("cuda")
    with torch.no_grad():  # as torch's own in-place operations
        apply_rotary(q, None, at, freq, out=(leaf, None))
    assert torch.equal(leaf, apply_rotary(q, None, at, freq)[0])


@pytest.mark.gpu
def test_backward_refuses_tensors_that_were_turned_in_place():
    q, at, freq = _given()
    k = torch.randn(6, 1, 32, device="cuda")
    w = torch.ones_like(q, requires_grad=True)
    u = torch.ones_like(k, requires_grad=True)
    y, z = (q * w).sum(), (k * u).sum()
    apply_rotary(q, k, at, freq, out=(q, k))
    for result in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            result.backward()
    # A view's write counts for what it is a view of.
    x = torch.randn(6, 5, 32, device="cuda")
    w = torch.ones_like(x, requires_grad=True)
    y = (x * w).sum()
    apply_rotary(x[:, :4], x[:, 4:], at, freq, out=(x[:, :4], x[:, 4:]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_written_caches_and_tables_have_new_versions():
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pages, tables = cache_pages(3, 32, 1, 64), torch.full((1, 2), -1, dtype=torch.int32, device="cuda")
    versions = pages._version, tables._version
    plan = plan_step(ints(0), ints(2), tables, ints(2, 0, 1), ints(0), page_size=32, max_tokens=2)
    k = torch.randn(2, 1, 64, device="cuda")
    append_tokens(pages, k, k, plan.slots)
    assert pages._version > versions[0] and tables._version > versions[1]
    versions = pages._version, tables._version, k._version
    read_tokens(pages, plan.slots)
    cache_attention(k.half(), pages, tables, plan.starts, plan.lengths)
    assert (pages._version, tables._version, k._version) == versions
    # A server's tensors are made in inference mode, and used in it or out of it.
    with torch.inference_mode():
        held, rows, q = pages.clone(), tables.clone(), torch.randn(2, 1, 64, device="cuda")
        at, freq = ints(4, 5), torch.ones(32, dtype=torch.float64, device="cuda")
        plan_step(ints(2), ints(2), rows, ints(2, 0, 1), ints(1), page_size=32, max_tokens=2)
        append_tokens(held, k, k, plan.slots)
        apply_rotary(q, None, at, freq, out=(q, None))
    append_tokens(held, k, k, plan.slots)
    apply_rotary(q, None, at, freq, out=(q, None))
    assert torch.equal(held, pages)


def _brute(a, b):
    """Whether two (address, shape, strides) of bytes have one in common."""
    def places(t):
        base, (n, h, d), (sn, sh) = t
        return {base + i * sn + j * sh + e for i in range(n) for j in range(h) for e in range(d)}
    return bool(places(a) & places(b))


def test_shared_memory_is_found_exactly():
    """Rows of one projection lie between each other and share nothing; against
    every byte's address, for shapes small enough to list them."""
    import random
    rng = random.Random(5)
    both = set()
    for _ in range(400):
        a, b = ((4096 + rng.randrange(40), (rng.randint(1, 4), rng.randint(1, 3), rng.choice([2, 4, 6])),
                 (rng.choice([0, 6, 8, 12, 24, 40]), rng.choice([0, 2, 6, 8, 16]))) for _ in range(2))
        found = _native.shares_memory(a, b)
        assert found == _brute(a, b), (a, b)
        both.add(found)
    assert both == {False, True}
    assert not _native.shares_memory((4096, (0, 3, 4), (12, 4)), (4096, (2, 3, 4), (12, 4)))


def test_rows_that_overlap_themselves():
    for shape, strides, free in (((3, 2, 8), (16, 8), True), ((3, 2, 8), (8, 24), True), ((3, 2, 8), (20, 9), True),
                                 ((3, 2, 8), (0, 8), False), ((3, 2, 8), (16, 0), False), ((3, 2, 8), (15, 8), False),
                                 ((3, 2, 8), (16, 7), False), ((1, 2, 8), (0, 8), True), ((3, 1, 8), (8, 0), True),
                                 ((3, 1, 8), (7, 0), False), ((0, 2, 8), (0, 0), True)):
        assert _native.rows_are_apart(shape, strides) == free, (shape, strides)


@pytest.mark.gpu
def test_out_that_shares_memory_is_refused():
    """Blocks of a launch would write what others read or write. Refused on the
    host, before any launch."""
    x = torch.randn(6, 12, 32, device="cuda")
    _, at, freq = _given()
    before = x.clone()
    q, k = x[:, :4], x[:, 4:8]
    flat = x.view(-1)
    shifted = flat[4:4 + 6 * 12 * 32 - 384].as_strided((6, 4, 32), (384, 32, 1), 4)
    other = torch.empty(6, 4, 32, device="cuda")
    for out in ((k, q),                                             # swapped
                (shifted, other), (other, shifted),                 # a few values on
                (q, q), (other, other),                             # one for both
                (other, other.flip(0).as_strided((6, 4, 32), (0, 32, 1))),  # one row for all tokens
                (torch.empty(6, 1, 32, device="cuda").expand(6, 4, 32), k),
                (torch.empty(1, 4, 32, device="cuda").expand(6, 4, 32), k),
                (x[:, 2:6], other),                                 # half of each
                (x.transpose(0, 1)[:6, :4].as_strided((6, 4, 32), (32, 384, 1)), other)):
        with pytest.raises(RuntimeError, match="out"):
            apply_rotary(q, k, at, freq, out=out)
    with pytest.raises(RuntimeError, match="out"):
        apply_rotary(q[:1].expand(6, 4, 32), None, at, freq, out=(q[:1].expand(6, 4, 32), None))
    assert torch.equal(x, before)


@pytest.mark.gpu
def test_out_between_other_rows_is_taken():
    x = torch.randn(6, 12, 32, device="cuda")
    _, at, freq = _given()
    before = x.clone()
    q, k = x[:, 0:12:3], x[:, 1:12:3]
    want = apply_rotary(q.contiguous(), k.contiguous(), at, freq)
    apply_rotary(q, k, at, freq, out=(x[:, 2:12:3], torch.empty_like(before)[:, :4]))
    assert torch.equal(x[:, 2::3], want[0]) and torch.equal(q, before[:, 0::3])
    apply_rotary(q, k, at, freq, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    alone = before[:, :4]
    apply_rotary(alone, None, at, freq, out=(before[:, 8:], None))
    assert torch.equal(before[:, 8:], apply_rotary(alone.contiguous(), None, at, freq)[0])
    one = torch.randn(1, 4, 32, device="cuda")  # a stride that no step takes
    apply_rotary(one, None, at[:1], freq, out=(one.as_strided((1, 4, 32), (0, 32, 1)), None))
