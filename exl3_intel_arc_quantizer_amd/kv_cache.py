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

with no host synchronisation in it. Drafted tokens of a request may be a tree:

    tree = plan_tree(parents, plan.starts, plan.lengths, max_new=most)
    q = append_tokens(..., positions=tree.positions, ...)
    out = cache_attention(..., trees=tree.masks)
    ...                                               # the model's choice after every token
    kept = accept_drafts(tokens, choices, parents, plan.starts, plan.lengths, max_new=most)
    taken = release_pages(plan.lengths, kept.lengths, tables, free_pages, plan.taken,
                          page_size=64)
    keep_tokens(pages, plan.slots, plan.starts, kept.places)     # every layer

after which the requests hold ``kept.lengths`` tokens, and ``kept.next`` follows.
The cache of a layer is one uint8 tensor
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
    for t in tensors:
        if t is not None and records(t):
            raise RuntimeError(f"{what} has no gradient: detach its inputs")


def append_tokens(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
                  q: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                  frequencies: Optional[torch.Tensor] = None, layout: str = "half",
                  magnitude: float = 1.0, axes: Optional[torch.Tensor] = None
                  ) -> Optional[torch.Tensor]:
    """Write keys and values (tokens, kv_heads, head_dim) to their slots
    (int64), in place; tokens with a slot outside the cache are skipped.

    With ``frequencies`` (a multiple of 8 pairs) and ``positions`` the keys
    first turn as in ``rotary.apply_rotary`` (with ``axes`` too), and so do the queries ``q``
    (tokens, q_heads, head_dim) if given, which are returned: the cache's side
    of a step is then one launch that reads the projection once. No slot may
    be given twice in a call."""
    _unrecorded("append_tokens", k, v, q, frequencies)
    return _native.cache_append(pages, k, v, slots, q, positions, frequencies,
                                layout_code(layout), magnitude, axes)


def read_tokens(pages: torch.Tensor, slots: torch.Tensor, *,
                dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (tokens, kv_heads, head_dim) that the cache holds at
    ``slots`` (int64), zeros for slots outside it."""
    return _native.cache_read(pages, slots, dtype)


def cache_attention(q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor,
                    starts: torch.Tensor, lengths: torch.Tensor, *,
                    scale: Optional[float] = None, window: Optional[int] = None,
                    max_new: Optional[int] = None,
                    trees: Optional[torch.Tensor] = None) -> torch.Tensor:
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

    ``trees`` (int64, (tokens or more, words), ``plan_tree``) are masks of the new
    tokens: of a request with up to 64 * words of them, row i attends the positions
    before the request's new tokens and its new token j where bit j of the row's
    mask is set (bit j % 64 of word j // 64), of this sequence the last ``window``.
    Any mask may be given; a row that it leaves empty is 0. Requests with more new
    tokens attend as without.

    Queries count with 22 bits, and so do the weights of requests of up to 16
    rows to a kv head (32 of head_dim 256); beyond, weights count with 11 bits, as
    in products of 16-bit operands. Scores, maxima and sums are float32."""
    _unrecorded("cache_attention", q)
    return _native.cache_attention(q, pages, tables, starts, lengths, scale, window, max_new, trees)


class TreePlan(NamedTuple):
    """What a step's layers share of the trees of drafted tokens, on the GPU."""

    masks: torch.Tensor      # int64 (tokens, words): a token's ancestors and itself
    positions: torch.Tensor  # int32 (tokens,): its position, one more than its parent's


def plan_tree(parents: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor, *,
              max_new: int) -> TreePlan:
    """Masks and positions of a step whose new tokens are trees.

    ``parents`` (int32, (tokens,), as many as the step's slots) gives, for each new
    token of a request (rows starts[r] .. starts[r + 1] - 1, the last of its
    lengths[r] tokens), the place among them of the token it follows, counted from
    0 and less than its own, or -1 if it follows the cached ones; any other number
    counts as -1. ``max_new`` (at most 1024) bounds the tokens of a tree: masks
    have ceil(max_new / 64) words, and a request of more tokens than they have bits
    is no tree but a run: its positions count up. Tokens of no request get 0."""
    return TreePlan(*_native.plan_tree(parents, starts, lengths, _tree_words(max_new)))


def _tree_words(max_new: int) -> int:
    """Words of a mask for trees of up to ``max_new`` tokens."""
    if not 1 <= max_new <= 64 * _native.MAX_TREE_WORDS:
        raise ValueError(f"max_new must be in 1..{64 * _native.MAX_TREE_WORDS}, got {max_new}")
    return -(-max_new // 64)


class Accepted(NamedTuple):
    """What a step keeps of its drafted tokens, on the GPU."""

    places: torch.Tensor     # int32 (tokens,): place among the request's kept tokens, or -1
    lengths: torch.Tensor    # int32 (requests,): tokens held, those kept among them
    next: torch.Tensor       # (requests,): the token chosen after the last kept one


def accept_drafts(tokens: torch.Tensor, choices: torch.Tensor, parents: torch.Tensor,
                  starts: torch.Tensor, lengths: torch.Tensor, *,
                  certain: Optional[torch.Tensor] = None,
                  max_new: Optional[int] = None) -> Accepted:
    """The drafted tokens that the model would have chosen itself.

    ``tokens`` are the step's token ids and ``choices`` the model's choice after
    each of them (int32 or int64, (tokens,)); ``parents``, ``starts`` and
    ``lengths`` as in ``plan_tree``. Of every request the first ``certain`` tokens
    (int32, (requests,); at least, and if left out, the first: the one that the
    last step chose) are kept, then from the last of them down, as long as there is
    one, the first token after those whose parent is the last kept and which is the
    choice after it. ``next`` is -1 for requests without new tokens.

    ``max_new`` is the bound that ``plan_tree`` was given (1024 if left out).
    Requests of more tokens than its masks have bits attended as a run, whatever
    their parents say, and are accepted as one: of each token the next one follows."""
    words = _native.MAX_TREE_WORDS if max_new is None else _tree_words(max_new)
    return Accepted(*_native.accept_drafts(tokens, choices, parents, starts, lengths, certain, words))


def keep_tokens(pages: torch.Tensor, slots: torch.Tensor, starts: torch.Tensor,
                places: torch.Tensor) -> None:
    """Move the entries of kept tokens together, in place: a token goes to the slot
    of its request's token number ``places`` (int32, as ``accept_drafts`` gives
    them: growing along a request, -1 for tokens that stay where they are, and no
    larger than its own number). ``slots`` and ``starts`` are the step's; moves from
    or to a slot outside the cache are skipped."""
    _native.cache_keep(pages, slots, starts, places)


def release_pages(before: torch.Tensor, after: torch.Tensor, tables: torch.Tensor,
                  free_pages: torch.Tensor, taken: torch.Tensor, *, page_size: int) -> torch.Tensor:
    """Give back the pages of requests that held ``before`` tokens and keep
    ``after`` of them (int32, (requests,); 0 ends a request): their entries of
    ``tables`` become -1 and the pages, in order, the last of ``free_pages`` before
    entry ``taken``, both in place. Returns the new ``taken``; the step plans'
    ``free_pages`` are thus a stack, from which the next ``plan_step`` takes.

    Only as many pages as were taken from it have a place on the stack. Of more (pages
    that a caller put into the tables from elsewhere) the first ones stay in their
    rows, where the caller finds them: entries past the kept tokens that are not -1,
    to be read before the next ``plan_step``, which writes over those it needs."""
    return _native.release_pages(before, after, tables, free_pages, taken, page_size)
