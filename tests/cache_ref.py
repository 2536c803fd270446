"""Plain 64-bit forms of the attention cache's operators, for the tests: the
definitions written token by token, on the CPU."""

from __future__ import annotations

import numpy as np
import torch

GROUP = 32


def sylvester() -> np.ndarray:
    h = np.ones((1, 1))
    while h.shape[0] < GROUP:
        h = np.block([[h, h], [h, -h]])
    return h


def turned(x, positions, frequencies, layout, magnitude=1.0, sign=1.0) -> np.ndarray:
    """float64 (tokens, heads, dim) turned by position * frequency."""
    y = torch.as_tensor(x).double().numpy().copy()
    n = len(frequencies)
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        angle = sign * torch.as_tensor(positions).double().numpy()[:, None] * frequencies[i]
        c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
        u, w = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def scale_of(most: np.ndarray) -> np.ndarray:
    """The float16 scale of a group whose largest transformed magnitude is
    `most` (float32)."""
    wanted = np.minimum(most.astype(np.float32) * np.float32(1.0 / 7.0), np.float32(9344.0))
    rounded = torch.from_numpy(wanted).to(torch.bfloat16).to(torch.float16).numpy()
    return np.where(np.isfinite(most), rounded, np.float16(np.nan)).astype(np.float16)


def butterfly32(x: np.ndarray) -> np.ndarray:
    """H x over the last axis (32) in x's type, levels of 1, 2, 4, 8, 16."""
    for h in (1, 2, 4, 8, 16):
        x = x.reshape(*x.shape[:-1], 16 // h, 2, h)
        x = np.stack([x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]], -2)
        x = x.reshape(*x.shape[:-3], GROUP)
    return x


def encode(x: np.ndarray):
    """(codes - 8, scales) of float32 values (..., dim), the definition's own
    float32 steps: bit for bit what the cache holds for them."""
    with np.errstate(all="ignore"):
        y = butterfly32(x.astype(np.float32).reshape(*x.shape[:-1], -1, GROUP)) * np.float32(0.125)
        most = np.abs(y).max(-1, keepdims=True)
        most = np.where(np.isfinite(y).all(-1, keepdims=True), most, np.float32(np.inf))
        scale = scale_of(most)
        s = scale.astype(np.float32)
        inverse = np.where(s > 0, np.float32(1.0) / np.where(s > 0, s, np.float32(1)), np.float32(0))
        codes = np.clip(np.rint(y * inverse.astype(np.float32)), -7, 7)
        codes = np.where(np.isnan(scale), 0, codes)
    return codes.astype(np.int32), scale


def decode(codes: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 values (..., dim) of codes - 8 (..., groups, 32) and scales
    (..., groups, 1)."""
    y = codes.astype(np.float64) * scale.astype(np.float64)
    return ((y @ sylvester()) / 4).reshape(*codes.shape[:-2], -1)


class Cache:
    """A cache in its logical form, and the bytes of it."""

    def __init__(self, pages, page, heads, dim, rng):
        self.shape = (pages, page, heads, dim)
        shape = (2, pages * page, heads, dim // GROUP, GROUP)
        self.codes = rng.integers(-8, 8, size=shape)
        scale = np.exp(rng.normal(size=shape[:-1] + (1,)) * 0.3) * 0.2
        self.scales = torch.from_numpy(scale.astype(np.float32)).to(torch.bfloat16).to(torch.float16).numpy()

    def values(self):
        """float64 keys and values (slots, heads, dim)."""
        return decode(self.codes[0], self.scales[0]), decode(self.codes[1], self.scales[1])

    def bytes(self) -> np.ndarray:
        pages, page, heads, dim = self.shape
        out = np.zeros((pages, heads, page // 32, 36 * dim), np.uint8)
        groups = dim // GROUP
        slot = np.arange(pages * page)
        p, tile, t = slot // page, slot % page // 32, slot % 32
        nibbles = (self.codes + 8).astype(np.uint32)
        for head in range(heads):
            for d in range(0, dim, 8):
                g, j, r = d // 32, d % 32 // 8, d // 8
                eight = nibbles[:, :, head, g, d % 32:d % 32 + 8]
                key = sum(eight[0][:, u] << (4 * (u // 2 + 4 * (u % 2))) for u in range(8))
                value = sum(eight[1][:, u] << (4 * u) for u in range(8))
                k_at = 4 * (t * (dim // 8) + j * groups + g)
                v_at = 16 * dim + 4 * ((t // 8 * (dim // 8) + r) * 8 + t % 8)
                for b in range(4):
                    out[p, head, tile, k_at + b] = key >> (8 * b) & 255
                    out[p, head, tile, v_at + b] = value >> (8 * b) & 255
            for g in range(groups):
                ks, vs = (self.scales[i][:, head, g, 0].view(np.uint16) for i in (0, 1))
                k_at = 32 * dim + 2 * (t * groups + g)
                v_at = 34 * dim + 2 * ((t // 8 * groups + g) * 8 + t % 8)
                for b in range(2):
                    out[p, head, tile, k_at + b] = ks >> (8 * b) & 255
                    out[p, head, tile, v_at + b] = vs >> (8 * b) & 255
        return out


def attention(q, keys, values, page, tables, starts, lengths, scale, window):
    """(out, sum p |v|, the same of the transformed values and taken back
    without cancellation, largest |q| |k|) in float64, row by row. keys and
    values are by slot; table entries outside the cache hide their page."""
    q = np.asarray(q, np.float64)
    tokens, heads, dim = q.shape
    kv_heads = keys.shape[1]
    out, spread, basis, reach = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q), np.zeros((tokens, heads, 1))
    pages = keys.shape[0] // page
    for r in range(len(lengths)):
        n = starts[r + 1] - starts[r]
        for i in range(n):
            p = lengths[r] - n + i
            t = np.arange(max(0, p - (window or 1 << 40) + 1), p + 1)
            ids = tables[r][t // page] if len(t) else np.zeros(0, np.int64)
            there = (ids >= 0) & (ids < pages)
            slots = (ids * page + t % page)[there]
            if not len(slots):
                continue
            for h in range(heads):
                k, v = keys[slots, h * kv_heads // heads], values[slots, h * kv_heads // heads]
                row = q[starts[r] + i, h]
                with np.errstate(all="ignore"):
                    x = scale * (k @ row)
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    out[starts[r] + i, h] = (w[:, None] * v).sum(0)
                    spread[starts[r] + i, h] = (w[:, None] * np.abs(v)).sum(0)
                    held = np.abs(v.reshape(-1, dim // GROUP, GROUP) @ sylvester()) / 8
                    held = (w[:, None, None] * held).sum((0, 2)) / 4
                    basis[starts[r] + i, h] = np.repeat(held, GROUP)
                    reach[starts[r] + i, h] = scale * np.linalg.norm(row) * np.linalg.norm(k, axis=1).max()
    return out, spread, basis, reach


def plan(cached, new, tables, free, taken, page, max_tokens):
    """The step plan, request by request and token by token."""
    tables = np.array(tables)
    width, status, at = tables.shape[1], 0, taken
    slots = np.full(max_tokens, -1, np.int64)
    positions = np.zeros(max_tokens, np.int32)
    starts = [0]
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        if c + n > width * page:
            status |= 2
        for p in range(min(-(-c // page), width), min(-(-(c + n) // page), width)):
            tables[r, p] = free[at] if at < len(free) else -1
            at += 1
        for i in range(n):
            t = starts[-1] + i
            if t < max_tokens:
                positions[t] = c + i
                if (c + i) // page < width and tables[r, (c + i) // page] >= 0:
                    slots[t] = tables[r, (c + i) // page] * page + (c + i) % page
        starts.append(starts[-1] + n)
    if at > len(free):
        status |= 1
    if starts[-1] > max_tokens:
        status |= 4
    lengths = [max(c, 0) + max(n, 0) for c, n in zip(cached, new)]
    return slots, positions, np.array(starts), np.array(lengths), min(at, max(len(free), taken)), status, tables


def attention_dense(q, keys, values, page, tables, starts, lengths, scale, window):
    """As `attention`, in float64 products over whole requests (on the tensors'
    device), for sizes that row by row would take too long."""
    tokens, heads, dim = q.shape
    kv_heads, dev = keys.shape[1], q.device
    outs = [torch.zeros(tokens, heads, dim, dtype=torch.float64, device=dev) for _ in range(3)]
    reach = torch.zeros(tokens, heads, 1, dtype=torch.float64, device=dev)
    turn = torch.from_numpy(sylvester()).to(dev)
    for r in range(len(lengths)):
        a, b, n = starts[r], starts[r + 1], lengths[r]
        t = torch.arange(n, device=dev)
        slots = torch.as_tensor(tables[r], device=dev).long()[t // page] * page + t % page
        at = torch.arange(n - (b - a), n, device=dev)[:, None]
        seen = (t[None] <= at) & (t[None] > at - (window or 1 << 40))
        for h in range(heads):
            k, v = keys[slots, h * kv_heads // heads], values[slots, h * kv_heads // heads]
            row = q[a:b, h].double()
            x = (row @ k.T * scale).masked_fill(~seen, float("-inf"))
            w = torch.softmax(x, 1)
            outs[0][a:b, h], outs[1][a:b, h] = w @ v, w @ v.abs()
            held = (v.reshape(n, dim // GROUP, GROUP) @ turn).abs().sum(2) / 32
            outs[2][a:b, h] = (w @ held).repeat_interleave(GROUP, 1)
            reach[a:b, h, 0] = scale * row.norm(dim=1) * k.norm(dim=1).max()
    return (*(o.cpu().numpy() for o in outs), reach.cpu().numpy())
