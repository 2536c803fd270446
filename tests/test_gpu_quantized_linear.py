"""Products with trellis weights as they are stored, against their 64-bit
definition."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from exl3_intel_arc_quantizer_amd import _native
from exl3_intel_arc_quantizer_amd.quantized_linear import quantized_linear
from exl3_intel_arc_quantizer_amd.serialization import decode_weight_from_storage
from oracle import trellis_format_ref as fmt

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _sylvester() -> np.ndarray:
    h = np.ones((1, 1))
    while h.shape[0] < 128:
        h = np.block([[h, h], [h, -h]])
    return h / np.sqrt(128.0)


def _blocks(x: np.ndarray) -> np.ndarray:
    return (x.reshape(*x.shape[:-1], -1, 128) @ _sylvester()).reshape(x.shape)


def _tiles(words: np.ndarray, K: int, cb: int) -> np.ndarray:
    """float64 (in, out) values of (in / 16, out / 16, 16 K) words, state by
    state: the 16 bits that end with bit (i + 1) K of the tile's ring."""
    tk, tn, _ = words.shape
    halves = words.view(np.uint16).astype(np.int64).reshape(tk, tn, -1, 2)[..., ::-1].reshape(tk, tn, -1)
    bits = (halves[..., None] >> np.arange(15, -1, -1)) & 1
    bits = bits.reshape(tk, tn, 256 * K)
    state = np.zeros((tk, tn, 256), np.int64)
    for b in range(16):
        state = 2 * state + bits[..., (np.arange(1, 257) * K - 16 + b) % (256 * K)]
    values = fmt.codebook_lut(cb).astype(np.float64)[state]
    tiles = np.empty_like(values)
    tiles[..., fmt.tensor_core_perm()] = values
    return tiles.reshape(tk, tn, 16, 16).transpose(0, 2, 1, 3).reshape(16 * tk, 16 * tn)


def _given(rows, k, n, K, dtype, seed=0, scales=torch.float16):
    rng = np.random.default_rng(seed + rows * 7 + k + n + K)
    words = torch.from_numpy(rng.integers(-32768, 32768, size=(k // 16, n // 16, 16 * K)).astype(np.int16))
    su = torch.from_numpy(rng.choice([-1.0, 1.0], k) * np.exp(rng.normal(size=k) * 0.3) * k ** -0.5).to(scales)
    sv = torch.from_numpy(rng.choice([-1.0, 1.0], n) * np.exp(rng.normal(size=n) * 0.3)).to(scales)
    x = torch.from_numpy(rng.normal(size=(rows, k)))
    x[:, 3::41] *= 9
    return x.to(dtype), words, su, sv


def _want(x, words, su, sv, K, cb):
    """(y, what |y' - y| may be before y' is rounded), float64, with the row's
    values counting with 22 bits; the second also for 11.

    The scaled row's products and seven levels of sums are each off by 2^-24 of
    what they add, sum |x su| / sqrt(128) of a block at most, ten times; a value
    of z then by 2^-22 of itself (two float16 parts) or 2^-11 (one). The 2 k
    products of an output are exact, their sums off by 2^-24 of sum |z w| each;
    the output's transform by 2^-24 of what it adds, ten times."""
    given = x.double().numpy() * su.double().numpy()
    z, w = _blocks(given), _tiles(words.numpy(), K, cb)
    reach = np.abs(given).reshape(*given.shape[:-1], -1, 128).sum(-1, keepdims=True) / np.sqrt(128.0)
    reach = np.broadcast_to(reach, (*reach.shape[:-1], 128)).reshape(given.shape)
    u, weights, scale = z @ w, np.abs(w), np.abs(sv.double().numpy())

    def spread(off):
        total = off.reshape(*off.shape[:-1], -1, 128).sum(-1, keepdims=True) / np.sqrt(128.0)
        return np.broadcast_to(total, (*total.shape[:-1], 128)).reshape(off.shape) * scale

    def bound(bits):
        off = (10 * 2.0 ** -24 * reach + bits * np.abs(z)) @ weights + 2 * x.shape[-1] * 2.0 ** -24 * (np.abs(z) @ weights)
        return spread(off + 10 * 2.0 ** -24 * np.abs(u))

    return _blocks(u) * sv.double().numpy(), bound(2.0 ** -22), bound(2.0 ** -11)


def _check(rows, k, n, K, cb, dtype, seed=0, scales=torch.float16):
    x, words, su, sv = _given(rows, k, n, K, dtype, seed, scales)
    got = quantized_linear(x.cuda(), words.cuda(), su.cuda(), sv.cuda(), K, cb)
    want, fine, coarse = _want(x, words, su, sv, K, cb)
    bound = coarse if dtype == torch.bfloat16 and rows > 64 else fine
    off = np.abs(got.double().cpu().numpy() - want)
    assert got.dtype == dtype and got.shape == (rows, n)
    assert (off <= bound + UNIT[dtype] * (np.abs(want) + bound) + 2.0 ** -25).all(), float((off / (bound + UNIT[dtype] * np.abs(want))).max())
    # All in all no more than the rounding of the output (an element is off by half
    # a place, UNIT of itself, at most) and what one part leaves of z, whose errors
    # of 2^-11 at most are of both signs.
    part = 2.0 ** -11 if bound is coarse else 0.0
    assert np.linalg.norm(off) <= (UNIT[dtype] + part + 2.0 ** -16) * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("cb", [0, 1, 2])
@pytest.mark.parametrize("K", range(1, 9))
def test_every_rate_and_codebook(K, cb):
    for rows in (3, 11, 20, 40, 70):
        _check(rows, 256, 384, K, cb, torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_rows(rows, dtype):
    _check(rows, 384, 640, 4, 2, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, k, n, K", [
    (1, 128, 128, 3), (1, 2176, 128, 4), (2, 128, 1920, 5), (8, 1152, 256, 2), (30, 128, 128, 8), (64, 1408, 128, 6),
    (65, 128, 128, 4), (200, 128, 2304, 1), (520, 256, 1152, 7), (3, 9088, 128, 4), (1, 33024, 128, 2), (70, 17408, 128, 3)])
def test_sizes(rows, k, n, K):
    for dtype in (torch.float16, torch.bfloat16):
        _check(rows, k, n, K, K % 3, dtype)


@pytest.mark.gpu
def test_is_the_decoded_weight():
    """The product with the weight that the storage decodes to, in float64; its
    elements are float32 roundings of the definition."""
    x, words, su, sv = (t.cuda() for t in _given(24, 512, 256, 4, torch.float16))
    w = decode_weight_from_storage(words, su, sv, 4)
    want = x.double() @ w.double()
    got = quantized_linear(x, words, su, sv, 4)
    # 16 roundings of 2^-24 in each element of w, 512 of them a sum.
    spread = x.double().abs() @ w.double().abs() * 512 * 2.0 ** -20
    assert ((got.double() - want).abs() <= UNIT[torch.float16] * want.abs() + spread).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 12, 50, 90])
def test_shapes_strides_and_scale_types(rows):
    x, words, su, sv = (t.cuda() for t in _given(rows, 256, 256, 4, torch.bfloat16))
    want = quantized_linear(x, words, su, sv, 4)
    wide = torch.zeros(rows, 2, 264, dtype=x.dtype, device="cuda")
    wide[:, 1, 8:] = x
    assert torch.equal(want, quantized_linear(wide[:, 1, 8:], words, su, sv, 4))
    odd = torch.empty(rows * 256 + 1, dtype=x.dtype, device="cuda")[1:].view(rows, 256).copy_(x)
    assert torch.equal(want, quantized_linear(odd, words, su, sv, 4))
    assert torch.equal(want, quantized_linear(x.t().contiguous().t(), words, su, sv, 4))
    assert torch.equal(want, quantized_linear(x.view(1, rows, 1, 256), words, su, sv, 4).view(rows, 256))
    assert torch.equal(want[0], quantized_linear(x[0], words, su, sv, 4)) or rows > 1
    assert torch.equal(want, quantized_linear(x, words, su.float(), sv.float(), 4))
    assert torch.equal(want, quantized_linear(x, words, su.float(), sv, 4))
    assert torch.equal(want, quantized_linear(x, words, su[:, None], sv[None], 4))
    same = quantized_linear(x[:1].expand(rows, 256), words, su, sv, 4)
    assert torch.equal(same, same[:1].expand(rows, 256))
    assert quantized_linear(x[:0], words, su, sv, 4).shape == (0, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 6, 14, 40, 130])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_do_not_touch_each_other(rows, dtype):
    """Rows of any size, and rows that are not finite, beside ordinary ones."""
    x, words, su, sv = (t.cuda() for t in _given(rows, 384, 256, 4, dtype))
    want = quantized_linear(x, words, su, sv, 4)
    y = x.clone()
    y[0, 200] = float("nan")
    got = quantized_linear(y, words, su, sv, 4)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], want[1:])
    y[0, 200] = -float("inf")
    got = quantized_linear(y, words, su, sv, 4)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], want[1:])
    # Powers of two scale a row's result exactly while it has its places.
    power = 2.0 ** -8 if dtype == torch.float16 else 2.0 ** 70
    scaled = x.clone()
    scaled[-1] = scaled[-1].double().mul(power).to(dtype)
    if torch.equal(scaled[-1].double(), x[-1].double() * power):
        got = quantized_linear(scaled, words, su, sv, 4)
        assert torch.equal(got[:-1], want[:-1])
        # A float16 result 256 times smaller may lose places: half of one, 2^-25, and
        # half of one of the larger result, 2^-12 of a value under 2^-14.
        off = (got[-1].double() - want[-1].double() * power).abs()
        assert (off <= (1.5 * 2.0 ** -25 if dtype == torch.float16 else 0.0)).all()
    zero = quantized_linear(torch.zeros_like(x), words, su, sv, 4)
    assert not zero.any()


@pytest.mark.gpu
def test_results_past_the_type_are_infinite():
    x, words, su, sv = (t.cuda() for t in _given(2, 128, 128, 4, torch.float16))
    big = quantized_linear(x, words, su, sv.float() * 1e7, 4)
    want = _want(x.cpu(), words.cpu(), su.cpu(), (sv.float() * 1e7).cpu(), 4, 2)[0]
    assert np.array_equal(np.isinf(big.cpu().numpy()), np.abs(want) >= 65520)


@pytest.mark.gpu
def test_words_past_32_bits():
    """A weight of 4.3 GB: input channels of its last block alone."""
    k = n = 65536
    words = torch.randint(-32768, 32768, (k // 16, n // 16, 128), device="cuda", dtype=torch.int16)
    su, sv = torch.ones(k, device="cuda"), torch.ones(n, device="cuda")
    for rows in (1, 20, 66):
        x = torch.zeros(rows, k, device="cuda", dtype=torch.float16)
        x[:, -128:] = torch.randn(rows, 128, device="cuda")
        got = quantized_linear(x, words, su, sv, 8)
        want = quantized_linear(x[:, -128:].contiguous(), words[-8:].contiguous(), su[-128:], sv, 8)
        # Both sum the same 128 products in float32, in orders of their own.
        assert ((got.double() - want.double()).abs() <= 2.0 ** -10 * want.double().abs() + 2.0 ** -8).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 13, 40, 150])
def test_in_a_graph_and_on_another_stream(rows):
    x, words, su, sv = (t.cuda() for t in _given(rows, 512, 256, 4, torch.bfloat16))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = quantized_linear(x, words, su, sv, 4)
    with torch.cuda.stream(side):
        assert torch.equal(quantized_linear(x, words, su, sv, 4), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = quantized_linear(x, words, su, sv, 4)
    for i in range(5):
        x.copy_(torch.randn_like(x))
        want = quantized_linear(x, words, su, sv, 4)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


@pytest.mark.gpu
def test_refusals():
    x, words, su, sv = (t.cuda() for t in _given(4, 256, 128, 4, torch.float16))
    for args in ((x.float(), words, su, sv, 4), (x.cpu(), words, su, sv, 4), (x, words.cpu(), su, sv, 4), (x, words.int(), su, sv, 4),
                 (x, words[:, ::2], su, sv, 4), (x, words, su[:-1], sv, 4), (x, words, su, sv[:-1], 4), (x, words, su.double(), sv, 4),
                 (x, words, su, sv.cpu(), 4), (x.clone().requires_grad_(), words, su, sv, 4),
                 (x, words, su.clone().requires_grad_(), sv, 4)):
        with pytest.raises(RuntimeError):
            quantized_linear(*args)
    for args in ((x[:, :128], words, su, sv, 4), (x, words, su, sv, 5), (x, words, su, sv, 9), (x, words, su, sv, 4, 3),
                 (x[:, :240], words[:15].contiguous(), su[:240], sv, 4)):
        with pytest.raises(ValueError):
            quantized_linear(*args)


def test_refuses_cpu_tensors_and_sizes():
    x, words, su, sv = _given(4, 256, 128, 4, torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        quantized_linear(x, words, su, sv, 4)
    lib = _native.load_library()
    assert lib.exl3_linear_workspace(4, 256, 128, 1) > 0 and lib.exl3_linear_workspace(0, 256, 128, 2) == 0
    assert lib.exl3_linear(None, 256, 0, 1, None, None, None, 0, 256, 128, 4, 2, None, None, 0, None) == 0
    for rows, k, n in ((-1, 128, 128), (4, 100, 128), (4, 128, 0), (4, 128, 192), ((1 << 22) + 1, 128, 128)):
        assert lib.exl3_linear_workspace(rows, k, n, 1) == -1
        assert lib.exl3_linear(None, k, rows, 1, None, None, None, 0, k, n, 4, 2, None, None, 1 << 40, None) == 1
    for K, cb, kind in ((0, 2, 1), (9, 2, 1), (4, 3, 1), (4, 2, 0), (4, 2, 3)):
        assert lib.exl3_linear(None, 128, 4, kind, None, None, None, 0, 128, 128, K, cb, None, None, 1 << 40, None) == 1
    assert lib.exl3_linear(None, 128, 4, 1, None, None, None, 0, 128, 128, 4, 2, None, None, 16, None) == 1
    assert b"too small" in lib.exl3_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 7, 30, 45, 100, 140])
def test_weights_that_start_anywhere(rows):
    """Words and scales that begin inside another tensor."""
    x, words, su, sv = (t.cuda() for t in _given(rows, 256, 384, 3, torch.bfloat16))
    want = quantized_linear(x, words, su, sv, 3)

    def moved(t, by):
        return torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")[by:].view(t.shape).copy_(t)

    for by in (1, 2, 4):
        assert torch.equal(want, quantized_linear(x, moved(words, by), su, sv, 3))
        assert torch.equal(want, quantized_linear(x, words, moved(su, by), moved(sv, by), 3))
        assert torch.equal(want, quantized_linear(x, words, moved(su.float(), by), moved(sv.float(), by), 3))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 3, 4, 48, 100])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_row_that_is_not_finite_is_alone(rows, dtype):
    x, words, su, sv = (t.cuda() for t in _given(rows, 640, 256, 5, dtype))
    want = quantized_linear(x, words, su, sv, 5)
    for value in (float("nan"), float("inf")):
        y = x.clone()
        y[1, 637] = value
        got = quantized_linear(y, words, su, sv, 5)
        assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows, k, n", [(4, 4096, 1408), (13, 4224, 256), (33, 2176, 768), (48, 1408, 4096), (128, 1152, 640),
                                        (257, 640, 1280), (1024, 256, 512)])
def test_more_sizes(rows, k, n):
    for dtype in (torch.float16, torch.bfloat16):
        _check(rows, k, n, 1 + rows % 8, rows % 3, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, k, n, K", [(200, 128, 33024, 5), (200, 1920, 16384, 2), (170, 256, 512, 8), (450, 640, 256, 4), (250, 1280, 384, 3)])
def test_blocks_of_many_rows(rows, k, n, K):
    """Blocks of 256, 224 and 192 rows, in one share and in more."""
    for dtype in (torch.bfloat16, torch.float16):
        _check(rows, k, n, K, 2 - K % 3, dtype)
