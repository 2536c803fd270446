"""Cases of the operators around a 4-bit attention cache: rotary positions,
the step plan (block tables and slot maps), appending to and reading from the
cache, and attention over it.

``listed()`` names representative sizes, ``draw(rng)`` gives more of the same
ranges, ``prepare`` makes what a serving (or training) program holds before
the call, ``run`` makes one pass: in plain torch operations where ``own`` is
false, through the package where it is true. ``work`` says what a pass cannot
do without, ``exact`` evaluates the definitions in float64.

The cache. ``pages`` is uint8 (pages, kv heads, P / 32, 36 D): tiles of 32
tokens of one head, each 16 D bytes of key codes, 16 D of value codes, then
2 D bytes of key scales and 2 D of value scales (float16). D is split in
groups of 32 with one scale each; a group x is held as y = H x / 8 (H the
Sylvester matrix of order 32), s = float16(bfloat16(max|y| / 7)) and 4-bit
codes c = clamp(rint(y / s), -7, 7) + 8, so it stands for H ((c - 8) s) / 4.

  key codes    [token 32][j 4][group D / 32] dwords of dims 32 group + 8 j ..
               + 7; nibble u of a dword is dim 2 u (u < 4) or 2 (u - 4) + 1
  value codes  [octet 4][D / 8][token 8] dwords of dims 8 r .. 8 r + 7 in
               nibble order; token 8 octet + token
  key scales   [token 32][D / 32]
  value scales [octet 4][D / 32][token 8]
"""

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
TILE = 32


def listed():
    return [
        # One request, one token: the rotary step of a single decoded token.
        {"name": "rotary_token", "op": "rotary", "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "layout": "half", "dtype": "float16", "first": 4000, "base": 10000.0, "grad": False},
        # A prompt batch of 8192 tokens at long positions.
        {"name": "rotary_prompt", "op": "rotary", "tokens": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "layout": "half", "dtype": "bfloat16", "first": 120000, "base": 500000.0, "grad": False},
        # A training step's forward and backward: adjacent pairs, a quarter of
        # the head, an odd number of tokens, float32.
        {"name": "rotary_grad", "op": "rotary", "tokens": 4099, "q_heads": 16, "kv_heads": 16, "dim": 64,
         "rotary": 16, "layout": "interleaved", "dtype": "float32", "first": 0, "base": 10000.0, "grad": True},
        # Every request of a serving batch decodes one token.
        {"name": "plan_decode", "op": "plan", "requests": 256, "context": 8192, "new": 1, "page": 64, "mix": 1},
        # Chunks of many prompts, ragged, some requests with nothing new.
        {"name": "plan_prompts", "op": "plan", "requests": 1531, "context": 2048, "new": 96, "page": 32, "mix": 2},
        # A decode step of 64 requests: q and k rotated, k and v written.
        {"name": "append_decode", "op": "append", "tokens": 64, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "layout": "half", "dtype": "bfloat16", "first": 4000, "page": 64},
        # A prompt batch, odd length, small heads without grouping.
        {"name": "append_prompt", "op": "append", "tokens": 8191, "q_heads": 16, "kv_heads": 16, "dim": 64,
         "layout": "interleaved", "dtype": "float16", "first": 0, "page": 128},
        # One request decodes one token: latency.
        {"name": "attend_token", "op": "attend", "requests": 1, "context": 4097, "new": 1, "even": True,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "dtype": "float16", "mix": 1},
        # A ragged serving batch, contexts from one token to 8192.
        {"name": "attend_batch", "op": "attend", "requests": 128, "context": 8192, "new": 1, "even": False,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "dtype": "bfloat16", "mix": 2},
        # Few requests with very long contexts and four drafted tokens each.
        {"name": "attend_drafts", "op": "attend", "requests": 3, "context": 131072, "new": 4, "even": False,
         "q_heads": 32, "kv_heads": 4, "dim": 128, "page": 256, "window": 0, "dtype": "bfloat16", "mix": 3},
        # Ragged prompt chunks on top of cached contexts, a sliding window.
        {"name": "attend_chunks", "op": "attend", "requests": 7, "context": 4500, "new": 1000, "even": False,
         "q_heads": 16, "kv_heads": 4, "dim": 256, "page": 32, "window": 2048, "dtype": "float16", "mix": 4},
        # A whole prompt of 8192 tokens.
        {"name": "attend_prompt", "op": "attend", "requests": 1, "context": 8192, "new": 8192, "even": True,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "dtype": "bfloat16", "mix": 5},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["rotary", "plan", "append", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = {"q_heads": kv * rng.choice([1, 2, 4, 5, 8, 16] if kv < 8 else [1, 2, 4]), "kv_heads": kv, "dim": dim}
    page = rng.choice([32, 64, 128, 256])
    if op == "rotary":
        tokens = _log(rng, 1, 16384)
        tokens = max(1, min(tokens, 335_000_000 // (4 * dim * (heads["q_heads"] + kv))))
        return {"op": op, "tokens": tokens, **heads, "rotary": rng.choice([dim, dim, dim // 2, dim // 4]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(sorted(TYPES)),
                "first": rng.choice([0, _log(rng, 1, 1_000_000)]), "base": rng.choice([10000.0, 500000.0]),
                "grad": rng.random() < 0.4}
    if op == "plan":
        requests = _log(rng, 1, 4096)
        return {"op": op, "requests": requests, "context": _log(rng, 1, 16384),
                "new": rng.choice([1, _log(rng, 1, max(1, 200_000 // requests))]), "page": page,
                "mix": rng.randrange(1 << 20)}
    if op == "append":
        tokens = _log(rng, 1, 16384)
        tokens = max(1, min(tokens, 80_000_000 // (dim * (heads["q_heads"] + 4 * kv))))
        return {"op": op, "tokens": tokens, **heads, "layout": rng.choice(["half", "interleaved"]),
                "dtype": rng.choice(["float16", "bfloat16"]), "first": rng.choice([0, _log(rng, 1, 1_000_000)]),
                "page": page}
    new = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 4096)])
    requests = _log(rng, 1, 128 if new < 16 else 12)
    # No more cached values and products than the largest listed cases have.
    most = min(400_000_000 // (requests * kv * dim), 130_000_000_000 // (requests * heads["q_heads"] * new * dim))
    context = max(1, min(_log(rng, 1, 131072), most))
    return {"op": op, "requests": requests, "context": context, "new": min(new, context), "even": rng.random() < 0.3,
            **heads, "page": page, "window": rng.choice([0, 0, _log(rng, 1, 8192)]),
            "dtype": rng.choice(["float16", "bfloat16"]), "mix": rng.randrange(1 << 20)}


# ------------------------------------------------------------- inputs

def _lengths(case):
    """(tokens held before the step, new tokens) of every request."""
    rng = random.Random(case["mix"])
    cached, fresh = [], []
    for i in range(case["requests"]):
        if case["op"] == "plan":
            new = case["new"] if case["new"] == 1 else rng.choice([0, rng.randint(1, case["new"]), rng.randint(1, case["new"])])
            cached.append(rng.randint(0, case["context"]))
        else:
            # The longest first, so that every case holds its full context.
            short = rng.random() < 0.25
            total = _log(rng, 1, case["context"]) if short else rng.randint(1, case["context"])
            total = case["context"] if case["even"] or i == 0 else total
            new = min(total, case["new"] if case["new"] <= 4 or case["even"] or i == 0 else rng.randint(1, case["new"]))
            cached.append(total - new)
        fresh.append(new)
    return cached, fresh


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device=DEVICE, generator=g) * scale).to(dtype)


def _frequencies(rotary, base):
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEVICE)
    return torch.pow(torch.full_like(i, base), -2.0 * i / rotary)


def _tables(held, page, width, g):
    """Pages of a shuffled pool for every request's ``held`` tokens, the rest
    of each row -1, and the pages that are left."""
    pages = [-(-n // page) for n in held]
    total = sum(pages)
    pool = torch.randperm(total + 64, device=DEVICE, generator=g).to(torch.int32)
    used = torch.tensor(pages, device=DEVICE)
    at = torch.arange(width, device=DEVICE)[None, :]
    first = (torch.cumsum(used, 0) - used)[:, None]
    rows = torch.where(at < used[:, None], pool[(first + at).clamp(max=total + 63)], torch.full_like(pool[:1], -1))
    return rows.contiguous(), total + 64, pool[total:]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cache(pages, kv_heads, page, dim, g):
    """A filled cache: rotated groups are close to normal, so codes are
    rounded normal values; positions past a request's end hold old tokens."""
    tiles = page // TILE
    shape = (pages, kv_heads, tiles, 32 * dim)
    nibbles = [torch.randn(shape, device=DEVICE, dtype=torch.float16, generator=g).mul_(2.6).round_().clamp_(-7, 7)
               .add_(8).to(torch.uint8) for _ in range(2)]
    codes = nibbles[0] | (nibbles[1] << 4)
    scales = torch.randn((pages, kv_heads, tiles, 2 * dim), device=DEVICE, generator=g).mul_(0.2).exp_().mul_(0.27)
    scales = scales.to(torch.bfloat16).to(torch.float16)
    return torch.cat([codes, scales.view(torch.uint8)], 3)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = dict(case)
    if op == "plan":
        cached, fresh = _lengths(case)
        order = np.random.RandomState(seed % (1 << 31)).permutation(len(cached))
        cached, fresh = [cached[i] for i in order], [fresh[i] for i in order]
        page = case["page"]
        width = -(-(case["context"] + case["new"]) // page)
        rows, pool, _ = _tables(cached, page, width, g)
        wanted = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, fresh))
        free = torch.randperm(wanted + 100, device=DEVICE, generator=g).to(torch.int32) + pool
        # The free list is a stack that earlier steps have taken 17 pages of;
        # the program pads its token buffers to a multiple of 64.
        state.update(cached=_ints(cached), fresh=_ints(fresh), tables=rows, free=free, taken=_ints([17]),
                     max_tokens=max(64, -(-sum(fresh) // 64) * 64))
        return state
    dtype = TYPES[case["dtype"]]
    dim, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    if op in ("rotary", "append"):
        t = case["tokens"]
        # q, k (and v) are slices of one projection's output.
        parts = hq + hk * (2 if op == "append" else 1)
        x = _normal((t, parts, dim), dtype, g)
        x[:, hq:hq + hk, ::17] *= 6
        state.update(q=x[:, :hq], k=x[:, hq:hq + hk], positions=torch.arange(t, device=DEVICE, dtype=torch.int32) + case["first"])
        if op == "rotary":
            state["frequencies"] = _frequencies(case["rotary"], case["base"])
            if case["grad"]:
                state["q"], state["k"] = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
                state["dq"], state["dk"] = _normal((t, hq, dim), dtype, g), _normal((t, hk, dim), dtype, g)
        else:
            page = case["page"]
            pages = -(-t // page) + 8
            slots = torch.arange(t, device=DEVICE)
            order = torch.randperm(pages, device=DEVICE, generator=g)
            state.update(v=x[:, hq + hk:], frequencies=_frequencies(dim, 10000.0), slots=order[slots // page] * page + slots % page,
                         pages=_cache(pages, hk, page, dim, g))
        return state
    cached, fresh = _lengths(case)
    order = np.random.RandomState(seed % (1 << 31)).permutation(len(cached))
    cached, fresh = [cached[i] for i in order], [fresh[i] for i in order]
    held = [c + n for c, n in zip(cached, fresh)]
    page = case["page"]
    rows, pool, _ = _tables(held, page, -(-max(held) // page), g)
    state.update(pages=_cache(pool, hk, page, dim, g), tables=rows, starts=_ints([0] + np.cumsum(fresh).tolist()),
                 lengths=_ints(held), q=_normal((sum(fresh), hq, dim), dtype, g, 2.0), most=max(fresh), longest=max(held))
    return state


# ------------------------------------------------------------- plain forms

def _turn(x, angles, layout, magnitude=1.0):
    """x (tokens, heads, dim) in float32, rotated by angles (tokens, rotary / 2)."""
    x = x.float()
    cos, sin = (angles.cos() * magnitude).float()[:, None], (angles.sin() * magnitude).float()[:, None]
    half = angles.shape[1]
    if layout == "half":
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b, rest = x[..., 0:2 * half:2], x[..., 1:2 * half:2], x[..., 2 * half:]
    pairs = torch.stack([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([pairs.flatten(-2), rest], -1)


def _angles(positions, frequencies):
    return positions.double()[:, None] * frequencies[None]


def _run_rotary(s):
    angles = _angles(s["positions"], s["frequencies"])
    dtype = s["q"].dtype
    q, k = (_turn(x.detach(), angles, s["layout"]).to(dtype) for x in (s["q"], s["k"]))
    if not s["grad"]:
        return {"q": q, "k": k}
    dq, dk = (_turn(x, -angles, s["layout"]).to(dtype) for x in (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _run_plan(s):
    page, tables = s["page"], s["tables"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    width = tables.shape[1]
    lengths = cached + fresh
    have = (cached + page - 1) // page
    need = ((lengths + page - 1) // page).clamp(max=width) - have.clamp(max=width)
    base = torch.cumsum(need, 0) - need
    at = torch.arange(width, device=DEVICE)[None, :] - have[:, None]
    taken = s["taken"].long()
    place = taken + base[:, None] + at
    count = s["free"].shape[0]
    page_of = torch.where(place < count, s["free"][place.clamp(0, count - 1)].long(), -1)
    rows = torch.where((at >= 0) & (at < need[:, None]), page_of, tables.long())
    starts = torch.cat([torch.zeros_like(fresh[:1]), torch.cumsum(fresh, 0)])
    t = torch.arange(s["max_tokens"], device=DEVICE)
    inside = t < starts[-1]
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=len(fresh) - 1)
    position = torch.where(inside, cached[r] + t - starts[r], 0)
    slot_page = rows[r, (position // page).clamp(max=width - 1)]
    good = inside & (position < width * page) & (slot_page >= 0)
    slots = torch.where(good, slot_page * page + position % page, -1)
    wanted = taken + need.sum()
    status = (wanted > count).int() + 2 * (lengths > width * page).any().int() + 4 * (starts[-1:] > s["max_tokens"]).int()
    return {"slots": slots, "positions": position.int(), "starts": starts.int(), "lengths": lengths.int(),
            "tables": rows.int(), "taken": wanted.clamp(max=count).int(), "status": status.int()}


def _sums(x):
    """H x over the last axis (32), H the Sylvester matrix, as five levels of
    sums and differences."""
    shape = x.shape
    for h in (1, 2, 4, 8, 16):
        x = x.reshape(*shape[:-1], 16 // h, 2, h)
        x = torch.stack([x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]], -2)
    return x.reshape(shape)


def _quantised(x):
    """float32 (tokens, heads, dim) to the values that its cache entry stands for."""
    y = _sums(x.unflatten(-1, (-1, TILE))) * 0.125
    most = y.abs().amax(-1, keepdim=True)
    scale = torch.clamp(most * (1.0 / 7.0), max=9344.0).to(torch.bfloat16).to(torch.float16).float()
    scale = torch.where(torch.isfinite(most), scale, float("nan"))
    codes = torch.clamp(torch.round(y * torch.where(scale > 0, 1.0 / scale, 0.0)), -7, 7)
    return (_sums(codes * scale) * 0.25).flatten(-2)


def _run_append(s):
    angles = _angles(s["positions"], s["frequencies"])
    dtype = s["q"].dtype
    q = _turn(s["q"], angles, s["layout"]).to(dtype)
    k = _quantised(_turn(s["k"], angles, s["layout"])).to(dtype)
    v = _quantised(s["v"].float()).to(dtype)
    return {"q": q, "k": k, "v": v}


def _held(pages, dim):
    """Keys and values (pages, heads, tokens, dim) in float32 of whole pages."""
    n, heads, tiles, _ = pages.shape
    groups = dim // TILE
    codes = pages[..., :32 * dim].reshape(n, heads, tiles, 2, 16 * dim)
    scales = pages[..., 32 * dim:].contiguous().view(torch.float16).reshape(n, heads, tiles, 2, dim)
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.float16) - 8
    k, v = nibbles[..., 0, :], nibbles[..., 1, :]
    k = k.reshape(n, heads, tiles, TILE, 4, groups, 8)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    k = k.transpose(-3, -2).reshape(n, heads, tiles * TILE, groups, TILE).float()
    k = k * scales[..., 0, :].reshape(n, heads, tiles * TILE, groups, 1).float()
    v = v.reshape(n, heads, tiles, 4, dim // 8, 8, 8).transpose(-3, -2)
    v = v.reshape(n, heads, tiles * TILE, groups, TILE).float()
    scale = scales[..., 1, :].reshape(n, heads, tiles, 4, groups, 8).transpose(-2, -1)
    v = v * scale.reshape(n, heads, tiles * TILE, groups, 1).float()
    turn = _sums(torch.eye(TILE, device=DEVICE)) * 0.25
    return (k @ turn).flatten(-2), (v @ turn).flatten(-2)


def _run_attend(s):
    q, dim, page, most, longest = s["q"], s["dim"], s["page"], s["most"], s["longest"]
    hk, group = s["kv_heads"], s["q_heads"] // s["kv_heads"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    requests, width = s["tables"].shape
    k, v = _held(s["pages"][s["tables"].clamp(min=0).long().flatten()], dim)
    k, v = (x.reshape(requests, width, hk, page, dim).transpose(1, 2).reshape(requests, hk, width * page, dim)[:, :, :longest]
            for x in (k, v))
    fresh = starts[1:] - starts[:-1]
    i = torch.arange(most, device=DEVICE)[None]
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    padded = q[rows].float().reshape(requests, most, hk, group, dim).permute(0, 2, 1, 3, 4)
    padded = padded.reshape(requests, hk, most * group, dim)
    scores = torch.matmul(padded, k.transpose(-1, -2).contiguous()) * dim ** -0.5
    at = (lengths - fresh)[:, None] + i
    t = torch.arange(longest, device=DEVICE)
    seen = t <= at[:, :, None]
    if s["window"]:
        seen = seen & (t > at[:, :, None] - s["window"])
    seen = seen[:, None, :, None, :]
    scores = scores.view(requests, hk, most, group, longest).masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp_(scores.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = weights.sum(-1, keepdim=True)
    v = torch.where((t < lengths[:, None])[:, None, :, None], v, 0.0)
    out = torch.matmul(weights.reshape(requests, hk, most * group, longest), v).view(requests, hk, most, group, dim)
    out = torch.where(total > 0, out / total, 0.0)
    inside = i < fresh[:, None]
    return out.permute(0, 2, 1, 3, 4).reshape(requests, most, hk * group, dim)[inside].to(q.dtype)


# ------------------------------------------------------------- the framework's operators

def _own_rotary(s):
    from exl3_intel_arc_quantizer_amd.rotary import apply_rotary
    q, k = apply_rotary(s["q"], s["k"], s["positions"], s["frequencies"], layout=s["layout"])
    if not s["grad"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _own_plan(s):
    from exl3_intel_arc_quantizer_amd.kv_cache import plan_step
    plan = plan_step(s["cached"], s["fresh"], s["tables"], s["free"], s["taken"], page_size=s["page"],
                     max_tokens=s["max_tokens"])
    return {"slots": plan.slots, "positions": plan.positions, "starts": plan.starts, "lengths": plan.lengths,
            "tables": s["tables"], "taken": plan.taken, "status": plan.status}


def _own_append(s):
    from exl3_intel_arc_quantizer_amd.kv_cache import append_tokens, read_tokens
    q = append_tokens(s["pages"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"],
                      frequencies=s["frequencies"], layout=s["layout"])
    k, v = read_tokens(s["pages"], s["slots"], dtype=s["k"].dtype)
    return {"q": q, "k": k, "v": v}


def _own_attend(s):
    from exl3_intel_arc_quantizer_amd.kv_cache import cache_attention
    return cache_attention(s["q"], s["pages"], s["tables"], s["starts"], s["lengths"], window=s["window"] or None,
                           max_new=s["most"])


_PLAIN = {"rotary": _run_rotary, "plan": _run_plan, "append": _run_append, "attend": _run_attend}
_OWN = {"rotary": _own_rotary, "plan": _own_plan, "append": _own_append, "attend": _own_attend}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------------- what a pass needs

def work(case):
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        page = case["page"]
        tokens = max(64, -(-sum(fresh) // 64) * 64)
        # Table entries: those that new tokens' slots come from are read, or
        # read from the free list and written.
        held = sum(-(-(c + n) // page) - c // page for c, n in zip(cached, fresh) if n)
        added = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, fresh))
        return {"bytes": 4 * (4 * len(cached) + held + added) + 12 * tokens, "flops": 0}
    size = TYPES[case["dtype"]].itemsize
    dim, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    if op == "rotary":
        values = case["tokens"] * (hq + hk) * dim * (2 if case["grad"] else 1)
        return {"bytes": 2 * values * size + 4 * case["tokens"], "flops": 3 * values * case["rotary"] // dim}
    if op == "append":
        t, cell = case["tokens"], dim * 9 // 8
        return {"bytes": t * (2 * hq * dim * size + 4 * hk * dim * size + 2 * hk * cell + 12 + 8),
                "flops": t * dim * (3 * (hq + hk) + 24 * hk)}
    cached, fresh = _lengths(case)
    window = case["window"] or 1 << 60
    pairs = tokens = 0
    for c, n in zip(cached, fresh):
        # Position p sees min(p + 1, window) positions.
        full = max(0, min(c + n, window) - c)
        pairs += full * c + full * (full + 1) // 2 + (n - full) * window
        tokens += min(c + n, window + n - 1)
    return {"bytes": tokens * hk * dim * 9 // 8 + 2 * sum(fresh) * hq * dim * size, "flops": 4 * dim * hq * pairs}


# ------------------------------------------------------------- the definitions in float64

def _turn64(x, positions, frequencies, layout, sign):
    x = x.detach().double().clone()
    r = 2 * len(frequencies)
    first = torch.arange(len(frequencies), device=DEVICE) * (2 if layout == "interleaved" else 1)
    second = first + (1 if layout == "interleaved" else r // 2)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                       sign * positions.double()[:, None, None] * frequencies)
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _sylvester():
    i = torch.arange(TILE, device=DEVICE)
    both = i[:, None] & i
    odd = sum((both >> b) & 1 for b in range(5)) % 2
    return (1 - 2 * odd).double()


def _quantised64(x):
    h = _sylvester()
    y = x.unflatten(-1, (-1, TILE)) @ h / 8
    scale = (y.abs().amax(-1, keepdim=True) / 7).clamp(max=9344)
    # To eight significant bits, and to the places that float16 has.
    power = torch.exp2(torch.floor(torch.log2(scale.clamp(min=2.0 ** -60))) - 7).clamp(min=2.0 ** -24)
    scale = torch.round(scale / power) * power
    codes = torch.round(y / scale.clamp(min=2.0 ** -30)).clamp(-7, 7)
    return ((codes * scale) @ h / 4).flatten(-2)


def _request64(s, r, head):
    """Keys and values (tokens, dim) in float64 of one head of a request, from
    the byte and nibble each value sits at."""
    dim, n = s["dim"], int(s["lengths"][r])
    groups = dim // TILE
    t = torch.arange(n, device=DEVICE)
    rows = s["pages"][s["tables"][r, t // s["page"]].long(), head, t % s["page"] // TILE]
    t, d = (t % TILE)[:, None], torch.arange(dim, device=DEVICE)[None]
    u = d % 8
    nibble = 8 * (t * dim // 8 + d % TILE // 8 * groups + d // TILE) + u // 2 + 4 * (u % 2)
    k = (rows.gather(1, nibble // 2) >> (4 * (nibble % 2)).to(torch.uint8)) & 15
    nibble = 8 * ((t // 8 * (dim // 8) + d // 8) * 8 + t % 8) + u
    v = (rows.gather(1, 16 * dim + nibble // 2) >> (4 * (nibble % 2)).to(torch.uint8)) & 15
    scales = rows[:, 32 * dim:].contiguous().view(torch.float16).double()
    ks = scales.gather(1, (t * groups + d // TILE))
    vs = scales.gather(1, dim + (t // 8 * groups + d // TILE) * 8 + t % 8)
    h = _sylvester() / 4
    return tuple((((c.double() - 8) * x).unflatten(-1, (-1, TILE)) @ h).flatten(-2) for c, x in ((k, ks), (v, vs)))


def _attend64(s):
    group = s["q_heads"] // s["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    starts = s["starts"].tolist()
    for r, length in enumerate(s["lengths"].tolist()):
        a, b = starts[r], starts[r + 1]
        at = torch.arange(length - (b - a), length, device=DEVICE)[:, None]
        t = torch.arange(length, device=DEVICE)[None]
        hidden = (t > at) | (t <= at - (s["window"] or 1 << 60))
        for h in range(s["kv_heads"]):
            k, v = _request64(s, r, h)
            for g in range(h * group, (h + 1) * group):
                scores = s["q"][a:b, g].double() @ k.T / math.sqrt(s["dim"])
                out[a:b, g] = torch.softmax(scores.masked_fill(hidden, float("-inf")), -1) @ v
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers, which have to be equal
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _attend64(s)
    turn = lambda x, sign: _turn64(x, s["positions"], s["frequencies"], s["layout"], sign)  # noqa: E731
    if case["op"] == "append":
        return {"q": turn(s["q"], 1), "k": _quantised64(turn(s["k"], 1)), "v": _quantised64(s["v"].double())}
    out = {"q": turn(s["q"], 1), "k": turn(s["k"], 1)}
    return {**out, "dq": turn(s["dq"], -1), "dk": turn(s["dk"], -1)} if case["grad"] else out
