"""Serving from a paged cache held in 8 bits: block tables, append, and stick-breaking attention of new tokens over cached ones.

A model that was trained with ``sb_attn_varlen`` answers token by token with these.  Once per step, whatever the number of layers::

    step = sb_cache_blocks(lengths, new_tokens, tables, free_pages, free_count, page_tokens, tokens)

once per layer::

    sb_cache_append(k, v, cache, step.pieces)                                            # k, v: [heads, tokens, head_dim]
    out, rem = sb_attn_cached(q, cache, tables, step.lengths, step.ends, v=v)            # out = o + rem * v

and at the end of the step::

    lengths.copy_(step.lengths), free_count.copy_(step.free_count)

Everything stays on the GPU: no call waits for it, and a step can be captured into a CUDA graph.  No counterpart in the reference, which has no
serving path."""
import math
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _lib
from ..ops import OP_NAMESPACE, _empty_like_rows, _unit_inner


class SbCache(NamedTuple):
    """Keys and values of one layer.  Token t of a request lies in page ``tables[request, t // page_tokens]``, place ``t % page_tokens``; its key is
    ``k[page, head, place, :head_dim].float() * k_scale[page, head]``.  k and v may be views with a larger step from page to page, such as
    the two halves of [pages, 2, heads, page_tokens, row]; a page itself is contiguous."""
    k: torch.Tensor        # float8_e4m3fn [pages, heads, page_tokens, row], row = 32, 64 or 128: the smallest that holds head_dim
    v: torch.Tensor
    k_scale: torch.Tensor  # float32 [pages, heads]
    v_scale: torch.Tensor


class SbBlocks(NamedTuple):
    """What a step does to the block tables (see sb_cache_blocks); int32 tensors."""
    lengths: torch.Tensor     # [requests] tokens after the step
    free_count: torch.Tensor  # [1] free pages after the step
    ends: torch.Tensor        # [requests] cumulative ends of the new tokens, packed one request behind the other
    slots: torch.Tensor       # [tokens] page * page_tokens + place of every new token, -1 behind the last one
    pieces: torch.Tensor      # [n, 4] (page, first new token, tokens there before, new tokens) of every page that is written, page -1 behind the last


# ---------------------------------------------------------------------------------------------- registered operators
# What a program that torch.compile traces calls in place of the binding: "cache_blocks", "cache_append", "attn_cached", beside the operators of
# ops.py.  They write tables and caches in place, as the functions do.
T = torch.Tensor


@torch.library.custom_op(f"{OP_NAMESPACE}::cache_blocks", mutates_args={"tables", "free_pages"}, device_types="cuda")
def _blocks_op(lengths: T, new_tokens: T, tables: T, free_pages: T, free_count: T, page_tokens: int, tokens: int) -> Tuple[T, T, T, T, T]:
    # an operator's results may not share their memory
    return tuple(x.clone() for x in _lib.binding().cache_blocks(lengths, new_tokens, tables, free_pages, free_count, page_tokens, tokens))


@_blocks_op.register_fake
def _(lengths, new_tokens, tables, free_pages, free_count, page_tokens, tokens):
    requests = lengths.size(0)
    m = min(requests, tokens)
    pieces = m + min(m, tokens - m) + max(0, tokens - 2 * m) // page_tokens  # sbattn_cache_pieces
    return tuple(lengths.new_empty(shape) for shape in ((requests,), (1,), (requests,), (tokens,), (pieces, 4)))


@torch.library.custom_op(f"{OP_NAMESPACE}::cache_append", mutates_args={"k_codes", "v_codes", "k_scale", "v_scale"}, device_types="cuda")
def _append_op(k: T, v: T, k_codes: T, v_codes: T, k_scale: T, v_scale: T, pieces: T) -> None:
    _lib.binding().cache_append(k, v, k_codes, v_codes, k_scale, v_scale, pieces)


@torch.library.custom_op(f"{OP_NAMESPACE}::attn_cached", mutates_args=(), device_types="cuda")
def _attend_op(q: T, k_codes: T, v_codes: T, k_scale: T, v_scale: T, tables: T, lengths: T, ends: Optional[T], inv_temp: float, attend_current: bool,
               v: Optional[T]) -> Tuple[T, T]:
    return _lib.binding().attend_cached(q, k_codes, v_codes, k_scale, v_scale, tables, lengths, ends, inv_temp, attend_current, v)


@_attend_op.register_fake
def _(q, k_codes, v_codes, k_scale, v_scale, tables, lengths, ends, inv_temp, attend_current, v):
    q = _unit_inner(q)
    return _empty_like_rows(q), torch.empty(q.shape[:-1], dtype=q.dtype, device=q.device)


def sb_cache(pages, heads, head_dim, page_tokens=64, device="cuda"):
    """An empty cache of one layer: 2 * pages * heads * page_tokens * row bytes of codes.  Pages of 64 tokens cost the fewest table
    entries and scales; small ones leave less of a request's last page unused and give each few tokens a scale of their own."""
    if not 1 <= head_dim <= 128:
        raise ValueError("head_dim must be between 1 and 128")
    if page_tokens not in (16, 32, 64, 128):
        raise ValueError("page_tokens must be 16, 32, 64 or 128")
    row = 32 if head_dim <= 32 else 64 if head_dim <= 64 else 128
    codes = [torch.zeros(pages, heads, page_tokens, row, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(pages, heads, dtype=torch.float32, device=device) for _ in range(2)]
    return SbCache(*codes, *scales)


def sb_cache_blocks(lengths, new_tokens, tables, free_pages, free_count, page_tokens, tokens):
    """One step of the block tables.  All tensors are int32 on the GPU:

    lengths [requests]: tokens that every request has; new_tokens [requests]: tokens that it takes (negative: gives up, from its end; a request that
    ends gives up all).  tables [requests, width]: pages of every request.  free_pages [pages]: a stack of free pages, of which
    free_count [1] are there.  tokens: rows that q, k, v of this step have, at least the sum of the positive new_tokens.

    Pages that no longer hold a token go onto the stack, pages that are needed come off it: entries of tables are written in place, and
    free_pages above free_count.  lengths and free_count stay as they are; copy SbBlocks.lengths and .free_count over them when the
    step is done (the same call before that gives the same answer).  Each page is held by one request.

    Refused steps change nothing, have no new tokens and are reported by check_status(): more pages wanted than there are, a length
    outside [0, width * page_tokens], more new tokens than ``tokens``."""
    if torch.compiler.is_compiling():
        return SbBlocks(*_blocks_op(lengths, new_tokens, tables, free_pages, free_count, int(page_tokens), int(tokens)))
    return SbBlocks(*_lib.binding().cache_blocks(lengths, new_tokens, tables, free_pages, free_count, int(page_tokens), int(tokens)))


def sb_cache_append(k, v, cache, pieces):
    """New keys and values k, v ([heads, tokens, head_dim]; bfloat16, float16 or float32) into the cache, in place.  The scale of a page and
    head is the smallest power of two that keeps its largest finite value within 448; it grows when a larger value comes, and the codes of the tokens that are
    there are rounded to the new one.  Infinities and NaN are stored as NaN.  A page is in at most one of the pieces.  No gradients."""
    if torch.compiler.is_compiling():
        if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):  # as the binding; a traced call does not come there in grad mode
            raise RuntimeError("appending to the cache has no backward: call it under torch.no_grad() or with tensors that need no gradient")
        _append_op(k, v, *cache, pieces)
    else:
        _lib.binding().cache_append(k, v, *cache, pieces)


def sb_attn_cached(q, cache, tables, lengths, ends=None, inv_temp=None, attend_current=False, v=None):
    """Attention of new tokens over the cache; their own keys and values have been appended.

    q: [H, T, D], H a multiple of the cache's heads (head h reads cache head h // (H / heads)).  lengths [requests]: tokens of every request, the new ones
    included; ends [requests]: cumulative ends of its rows of q, which are its last tokens in order.  Without ends, row r of q is
    the last token of request r.  A token sees the keys before it, and its own with ``attend_current``.

    Returns (o, rem) as sb_attn_varlen does; with ``v``, the new tokens' values [heads, T, D], the first is o + rem[..., None] * v.  A token that sees no
    key has o = 0 and rem = 1.  Rows behind the last end, and rows of requests of length 0 (without ends), have rem = 0 and an o that is left
    as it was allocated.  No gradients."""
    if inv_temp is None:
        inv_temp = 1 / math.sqrt(q.size(-1))
    attend = _attend_op if torch.compiler.is_compiling() else _lib.binding().attend_cached
    return attend(q, *cache, tables, lengths, ends, float(inv_temp), bool(attend_current), v)
