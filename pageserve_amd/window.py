"""Long texts in a bounded cache, on the GPU.

The reference's attention reads every cached token of a sequence
(engine/paged_attention.py:16-50), and a sequence keeps all of them.  Here a
request may be cut in two ways, over the same paged cache, tables and ragged
batches as in :mod:`pageserve_amd.paged`:

* :func:`window_attention` (and :func:`window_attention4` over a cache in 4 bits,
  :mod:`pageserve_amd.cache4`) reads the tokens of a sliding window and the
  first few, the sinks, which every later token leans on.  It serves single tokens
  and prompts of any length alike; without a window it is plain causal attention;
* :func:`accumulate_weights` adds up what attention each cached token gets, and
  :func:`evict_tokens` cuts requests to the tokens that got most, moved together at
  the front; :func:`truncate_blocks` then gives their last blocks back.

A step: ``append_blocks`` -> per layer ``write_kv`` (or ``write_kv4``),
``window_attention`` with ``return_lse``, ``accumulate_weights`` -> where a
request has outgrown its budget, ``evict_tokens`` for all layers and
``truncate_blocks``.  Lengths, tables and budgets are read on the device: nothing
waits for the host, and a step can be one captured HIP graph.

Prompts and single tokens may be in one call, but the kernels are chosen for the
whole batch by its bounds: a long prompt among single tokens makes them cost several
times what they cost alone.  Two calls over slices of ``lens``, ``block_tables`` and
``offsets`` (``offsets[b0 : b1 + 1]``, the rows where they are), into one ``out``, give
each kind its own.

The rows ``offsets[b] .. offsets[b + 1] - 1`` are request ``b``'s newest tokens, in
order, and ``lens[b]`` counts them: their keys and values are in the cache when the
call runs.  Row ``t`` of ``n`` stands at ``p = lens[b] - n + t`` and sees token
``j`` if ``j <= p`` and (``j > p - window`` or ``j < sinks``).

Everything runs on the current stream of the tensors' device, asynchronously; CPU
tensors are refused.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native
from .cache4 import KVCache4

__all__ = ["window_attention", "window_attention4", "accumulate_weights", "evict_tokens"]


def window_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     lens: torch.Tensor, offsets: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     max_tokens: int | None = None, max_context: int | None = None, scale: float | None = None,
                     return_lse: bool = False, out: torch.Tensor | None = None
                     ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of the requests' newest rows over their cached tokens.

    q: (rows, q_heads, head_dim); the caches (blocks, block_size, kv_heads, head_dim)
    as for :func:`write_kv`, q_heads a multiple of kv_heads; bf16 or fp16, head_dim 64
    or 128, block_size a multiple of 16.  ``window``: how many tokens back a row sees,
    itself included (None: all); ``sinks``: how many of the first tokens it sees
    whatever the window.  ``block_tables`` (int32 [requests, columns]), ``lens``
    (int32 [requests], the rows' own tokens among them) and ``offsets`` (int32
    [requests + 1]) as in :func:`append_blocks`; the blocks of tokens that no row sees
    are not read, and their columns may be absent (-1).

    ``max_tokens`` bounds the rows of a request (default: the rows there are; a
    request's rows beyond it are not computed) and ``max_context`` its tokens
    (default: what the tables can hold).  The kernels and the split of long contexts
    are chosen by them, so a step of single tokens says ``max_tokens=1``; max_context
    never changes what is computed.  ``scale``: of q . k, head_dim ** -0.5 by default.

    Returns (rows, q_heads, head_dim), or writes to ``out`` (contiguous; it may be q
    itself); with ``return_lse`` also the natural logarithm of each row's sum of
    e^score, fp32 (rows, q_heads).  A row that sees no token gets zeros and -inf.  Rows that belong to no
    request are not written: in a new tensor they hold anything, in ``out`` what they
    held.  Softmax and sums are fp32; the weights are rounded to the tensors' dtype
    before they multiply v.  A key or value that is not finite reaches only the rows
    that see it."""
    r = _native.load_host().window_attention(q, [k_cache, v_cache], block_tables, lens, offsets, window, sinks, max_tokens,
                                             max_context, scale, return_lse, out)
    return (r[0], r[1]) if return_lse else r[0]


def window_attention4(q: torch.Tensor, cache: KVCache4, block_tables: torch.Tensor, lens: torch.Tensor,
                      offsets: torch.Tensor, *, window: int | None = None, sinks: int = 0, max_tokens: int | None = None,
                      max_context: int | None = None, scale: float | None = None, return_lse: bool = False,
                      out: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """:func:`window_attention` over a cache in 4 bits; q and the result are bf16 or
    fp16, whatever rows the cache was written from (with fp16, cached values beyond
    its range may count as infinite).  Of a value that is not finite, all dims of its
    group of 32 are not finite in the rows that see it: it is the group's scale."""
    r = _native.load_host().window_attention(q, cache.parts, block_tables, lens, offsets, window, sinks, max_tokens,
                                             max_context, scale, return_lse, out)
    return (r[0], r[1]) if return_lse else r[0]


def accumulate_weights(q: torch.Tensor, k_cache: torch.Tensor | KVCache4, block_tables: torch.Tensor, lens: torch.Tensor,
                       offsets: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor, *,
                       new_lens: torch.Tensor | None = None, window: int | None = None, sinks: int = 0,
                       max_tokens: int | None = None, max_context: int | None = None,
                       scale: float | None = None) -> None:
    """Adds to ``weights`` (fp32 (blocks, block_size), a number for each slot of the
    cache) what attention the rows paid to each token that they see: the sum over
    rows and query heads of e^(score - lse).

    ``lse`` is what :func:`window_attention` returned for the same rows, and the other
    arguments are those of that call; ``k_cache`` may be a :class:`KVCache4` (with fp16
    rows, cached keys beyond its range may count as infinite).  With
    ``new_lens`` (int32 [requests], as :func:`append_blocks` took it) that many last
    tokens of a request start from nothing: their slots hold what an earlier owner
    left there.  One ``weights`` for each layer, or one for all of them.  No block may
    be in two requests' tables, or twice in one: of the additions to a slot that two
    reach, one may be lost.

    Sums are fp32 in a fixed order: the same call gives the same bits."""
    cache = k_cache.parts if isinstance(k_cache, KVCache4) else [k_cache]
    _native.load_host().accumulate_weights(q, cache, block_tables, lens, offsets, lse, weights, new_lens, window, sinks,
                                           max_tokens, max_context, scale)


def evict_tokens(weights: torch.Tensor, lens: torch.Tensor, budget: torch.Tensor, block_tables: torch.Tensor,
                 caches: Sequence[KVCache4 | tuple[torch.Tensor, torch.Tensor]], *, sinks: int = 0, recent: int = 0,
                 max_context: int | None = None) -> torch.Tensor:
    """Cuts every request of more than ``budget[b]`` tokens to as many, and returns
    how many each keeps (int32 [requests]).

    The first ``sinks`` and the last ``recent`` tokens stay (sinks first, where the
    budget does not hold both), and of those between the ones of largest ``weights``
    (fp32 (blocks, block_size); of equal ones the first, a NaN before all, a token in
    an absent block last).  What stays keeps its order and moves to the front of the
    request's blocks, in place, in ``weights`` and in every one of ``caches``: pairs
    (k_cache, v_cache) or :class:`KVCache4`, of as many layers as share the tables.
    ``lens`` and the tables are left: ``truncate_blocks(lens, kept, ...)`` shortens
    them and gives the blocks back.  The keys keep the positions that they were
    rotated for.

    ``budget``: int32 [requests] (below 0 counts as 0).  ``max_context`` bounds the
    requests' tokens (default: what the tables can hold) and sizes the workspace; a
    longer request is left as it is.  The 16-bit caches agree in their sizes with one
    another, and so do the 4-bit ones; no block may be in two requests' tables, and no
    two caches may share an element."""
    parts = [c.parts if isinstance(c, KVCache4) else list(c) for c in caches]
    for p in parts:
        if len(p) not in (2, 4):
            raise ValueError("evict_tokens: a cache is a pair (k_cache, v_cache) or a KVCache4")
    return _native.load_host().evict_tokens(weights, lens, budget, block_tables, parts, sinks, recent, max_context)
