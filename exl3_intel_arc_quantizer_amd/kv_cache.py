"""A 4-bit attention cache on the GPU, and the operators of a serving step
around it (HIP kernels; ``include/exl3_layer.h``).

Keys and values get the treatment that the weights get: groups of 32 values
are rotated by a Hadamard transform, which spreads a large channel over its
group, and stored as 4-bit codes with one scale, 4.5 bits a value. A step of a
served model is

    plan = plan_step(cached, new, tables, free_pages, taken, page_size=64,
                     max_tokens=tokens)               # once a step
    q = append_tokens(pages, k, v, plan.slots, q=q, positions=plan.positions,
                      frequencies=frequencies)        # every layer
    out = cache_attention(q, pages, tables, plan.starts, plan.lengths,
                          max_new=most)               # most new tokens of a request

with no host synchronisation in it. The cache of a layer is one uint8 tensor
(``cache_pages``); tables, slots and lengths serve all layers. The functions
enqueue work on the current stream of the tensors' device and keep nothing
between calls. None of them has a gradient except the rotary step, which is
``rotary.apply_rotary`` on its own.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native
from .hadamard import records
from .rotary import layout_code

TILE = 32
MAX_REQUESTS = 4096
PAGE_SIZES = (32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)

PAGES_RAN_OUT, ROW_TOO_SHORT, TOO_MANY_TOKENS = 1, 2, 4


def cache_pages(num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                device="cuda") -> torch.Tensor:
    """An empty cache of ``num_pages`` pages of ``page_size`` tokens: uint8
    (num_pages, kv_heads, page_size / 32, 36 * head_dim). The other functions
    take its sizes from this shape."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if num_pages < 0 or kv_heads < 1:
        raise ValueError(f"bad cache shape: {num_pages} pages of {kv_heads} heads")
    return torch.zeros((num_pages, kv_heads, page_size // TILE, 36 * head_dim),
                       dtype=torch.uint8, device=device)


class StepPlan(NamedTuple):
    """What a step's layers share, all on the GPU."""

    slots: torch.Tensor      # int64 (max_tokens,): place of each token in the cache, -1 for none
    positions: torch.Tensor  # int32 (max_tokens,): its position in the request
    starts: torch.Tensor     # int32 (requests + 1,): first token of each request
    lengths: torch.Tensor    # int32 (requests,): tokens held after the step
    taken: torch.Tensor      # int32 (1,): entries of free_pages used so far
    status: torch.Tensor     # int32 (1,): 0, or a sum of the reasons that check() names

    def check(self) -> None:
        """Raise RuntimeError if the step does not fit (waits for the GPU)."""
        status = int(self.status)
        if status:
            reasons = [text for bit, text in (
                (PAGES_RAN_OUT, "the free pages ran out"),
                (ROW_TOO_SHORT, "a request outgrew its row of the table"),
                (TOO_MANY_TOKENS, "more new tokens than max_tokens")) if status & bit]
            raise RuntimeError("plan_step: " + ", ".join(reasons))


def plan_step(cached: torch.Tensor, new: torch.Tensor, tables: torch.Tensor,
              free_pages: torch.Tensor, taken: torch.Tensor, *, page_size: int,
              max_tokens: int) -> StepPlan:
    """Block tables, slots and positions of one step, from the requests'
    lengths alone and without a host round trip.

    ``cached`` and ``new`` (int32, (requests,), at most 4096) are the tokens
    each request holds and the ones it adds; ``tables`` (int32, (requests,
    width)) names the pages of each request and gets, in place, the pages that
    the new tokens need, taken from ``free_pages`` (int32) in order from entry
    ``taken`` (int32, (1,)) on. ``taken`` itself is not changed: the next step
    passes the plan's, so that a step can be planned again. Slots past the last
    new token are -1, and so are those of tokens that have no page, in this step
    or because an earlier one ran out of them (``status``, ``StepPlan.check``)."""
    return StepPlan(*_native.plan_step(cached, new, tables, free_pages, taken, page_size,
                                       max_tokens))


def _unrecorded(what: str, *tensors) -> None:
    if any(t is not None and records(t) for t in tensors):
        raise RuntimeError(f"{what} has no gradient: detach its inputs")


def append_tokens(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
                  q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                  frequencies: Optional[torch.Tensor] = None, layout: str = "half",
                  magnitude: float = 1.0) -> Optional[torch.Tensor]:
    """Write keys and values (tokens, kv_heads, head_dim) to their slots
    (int64), in place; tokens with a slot outside the cache are skipped.

    With ``frequencies`` (a multiple of 8 pairs) and ``positions`` the keys
    first turn as in ``rotary.apply_rotary``, and so do the queries ``q``
    (tokens, q_heads, head_dim) if given, which are returned: the cache's side
    of a step is then one launch that reads the projection once. No slot may
    be given twice in a call."""
    _unrecorded("append_tokens", k, v, q, frequencies)
    return _native.cache_append(pages, k, v, slots, q, positions, frequencies,
                                layout_code(layout), magnitude)


def read_tokens(pages: torch.Tensor, slots: torch.Tensor, *,
                dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (tokens, kv_heads, head_dim) that the cache holds at
    ``slots`` (int64), zeros for slots outside it."""
    return _native.cache_read(pages, slots, dtype)


def cache_attention(q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor,
                    starts: torch.Tensor, lengths: torch.Tensor, *,
                    scale: Optional[float] = None, window: Optional[int] = None,
                    max_new: Optional[int] = None) -> torch.Tensor:
    """Attention of a step's new tokens over the cache, with its new tokens
    appended already; (tokens, q_heads, head_dim) like ``q`` (float16 or
    bfloat16), which may have more query heads than the cache has kv heads (a
    multiple). Single tokens, drafted tokens, prompt chunks and whole prompts
    may be mixed.

    Request r's queries are rows starts[r] .. starts[r + 1] - 1 and the last
    of its lengths[r] positions; each attends its own position and those
    before it, the last ``window`` of them if given. Positions in pages that
    ``tables`` does not name are not attended; rows that attend nothing, and
    rows of no request, are 0. ``scale`` defaults to head_dim ** -0.5.
    ``max_new``, the most new tokens of any request or a bound of them, chooses
    kernels; results depend on it in rounding at most. Left out, a request may
    have all of q's rows: a batch of single tokens then pays for a kernel of many
    rows beside its own (128 requests of 4096 positions: 134 us with
    ``max_new=1``, 178 without).

    Queries count with 22 bits, and so do the weights of requests of up to 16
    rows to a kv head (32 of head_dim 256); beyond, weights count with 11 bits, as
    in products of 16-bit operands. Scores, maxima and sums are float32."""
    _unrecorded("cache_attention", q)
    return _native.cache_attention(q, pages, tables, starts, lengths, scale, window, max_new)
