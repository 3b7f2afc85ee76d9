"""The paged cache of keys and values, on the GPU.

The reference keeps its cache in blocks of a fixed number of tokens
(engine/block_allocator.py:13-34, engine/paged_attention.py:62-132): a request's
block table names the blocks that hold its tokens.  There the tables live in
Python and attention gathers the cache one sequence at a time.  Here a batch of
requests is served by kernels that read lengths and tables on the device, so a
whole step, with lengths that change from step to step, can be one captured HIP
graph:

* :func:`append_blocks` extends the requests' tables by the blocks their new
  tokens need and gives every row its slot; :func:`truncate_blocks` shortens
  requests and gives their blocks back;
* :func:`write_kv` stores key and value rows at their slots;
* :func:`tree_attention` lets drafted tokens attend to a request's cached
  tokens and to their own ancestors.

A batch is ragged: the rows ``offsets[b] .. offsets[b + 1] - 1`` of its tensors
belong to request ``b`` (int32, one more entry than requests); rows behind the
last offset belong to none, so a captured batch may be padded.  The caches are
``(blocks, block_size, kv_heads, head_dim)``, with any strides whose last is 1
(halves of one tensor, or heads in front of slots, as permuted views).

A step that verifies drafted tokens needs no room in the cache for them:
:func:`tree_attention` takes their keys and values as rows, and once it is known
which are accepted, ``append_blocks(..., index=)`` gives those their slots (the
others get -1) and ``write_kv`` stores them, layer by layer.

Everything runs on the current stream of the tensors' device, asynchronously;
CPU tensors are refused.
"""

from __future__ import annotations

import torch

from . import _native

__all__ = ["append_blocks", "truncate_blocks", "write_kv", "tree_attention"]


def append_blocks(lens: torch.Tensor, new_lens: torch.Tensor, offsets: torch.Tensor, block_tables: torch.Tensor,
                  free_blocks: torch.Tensor, free_count: torch.Tensor, block_size: int, rows: int,
                  index: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Extends request ``b`` by ``new_lens[b]`` tokens and returns ``(slots,
    status)``.

    In place, in request order: the blocks a request needs beyond those it has
    are taken from the top of the stack ``free_blocks[:free_count]`` into the next
    columns of its row of ``block_tables``; ``lens`` and ``free_count`` are
    updated.  ``status[b]`` (int32) is 0 if the request was served, 1 if the
    requests up to it need more blocks than are free, 2 if its table has too few
    columns (or its length is negative); a request that was not served is left
    as it was.

    ``slots`` (int64, one per row of the batch) holds ``block * block_size +
    place in the block``, i.e. indexes ``k_cache.flatten(0, 1)``.  Row ``i`` of
    the batch is its request's ``n``-th new token, ``n = index[i]``, or ``i -
    offsets[b]`` without an index; its slot is -1 where ``n`` is not in
    ``0 .. new_lens[b] - 1``, the request was not served, the row belongs to
    none or its block was absent (negative) in the table already.  Rows of a
    request with the same index get the same slot.

    All tensors int32 and on one GPU: ``lens`` and ``new_lens`` [requests],
    ``offsets`` [requests + 1], ``block_tables`` [requests, columns],
    ``free_blocks`` [any], ``free_count`` [1], ``index`` [rows].  At most 4096
    requests per call.  Those that are changed may be parts of one buffer, but
    share no element with one another nor with those that are read."""
    slots, status = _native.load_host().append_blocks(lens, new_lens, offsets, block_tables, free_blocks, free_count,
                                                      block_size, rows, index)
    return slots, status


def truncate_blocks(lens: torch.Tensor, keep: torch.Tensor, block_tables: torch.Tensor, free_blocks: torch.Tensor,
                    free_count: torch.Tensor, block_size: int) -> None:
    """Shortens request ``b`` to ``keep[b]`` tokens, in place: 0 for one that is
    finished, any count from its length on to leave it (a negative length becomes
    0).  The blocks it no longer
    needs go back to the stack and their table columns become -1; a negative
    column (an absent block) gives nothing back.  Undoes :func:`append_blocks`
    exactly.  Tensors as there, ``keep`` int32 [requests]."""
    _native.load_host().truncate_blocks(lens, keep, block_tables, free_blocks, free_count, block_size)


def write_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slots: torch.Tensor) -> None:
    """Stores the rows of ``k`` and ``v`` (rows, kv_heads, head_dim) at their
    slots of the caches (the reference's write_kv, engine/paged_attention.py:62-79,
    for a whole batch).  A row whose slot (int64) is outside the cache, as -1 is,
    is left out.  No two rows may have the same slot (:func:`append_blocks` gives
    none twice, unless ``index`` names a token twice): of two that do, pieces of
    either may stay.  Rows that are views of the caches themselves are copied
    first, so rows can be moved to other slots, also of one another.  bf16 or fp16,
    the rows in any strides whose last is 1; no two elements of a cache may share a
    place (an expanded one is refused)."""
    _native.load_host().write_kv(k, v, k_cache, v_cache, slots)


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_tables: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor,
                   parents: torch.Tensor | None = None, *, max_tokens: int = 64, max_context: int | None = None,
                   scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted tokens over the paged cache
    (engine/paged_attention.py:16-50 for a batch of trees).

    Row ``offsets[b] + t`` is token ``t`` of request ``b``.  It attends to the
    request's ``lens[b]`` cached tokens, to itself and to its ancestors among the
    drafted tokens: ``parents`` (int32, per row) names the token of the same
    request that it follows, which must come before it; any other value (-1) means
    that it follows the cached text directly.  Without ``parents`` every token
    follows the one before it, so one token per request is plain decoding and
    several are a drafted chain.

    q: (rows, q_heads, head_dim); k, v: the drafted tokens' own keys and values,
    (rows, kv_heads, head_dim), q_heads a multiple of kv_heads; bf16 or fp16, as
    the caches; head_dim 64 or 128; the caches' block_size a multiple of 16.
    ``max_tokens`` bounds the rows of a request (1..64; a request's rows beyond it
    are not computed).  The kernels are chosen by it, or by the number of rows if
    that is less: plain decoding of a batch gives 1.  ``max_context`` bounds its
    cached tokens: it sizes the split of long contexts over the GPU, never the
    result (default: what the tables can hold).  ``scale``: of q . k, head_dim ** -0.5 by default.

    Returns (rows, q_heads, head_dim), or writes to ``out`` (contiguous; it may be
    q itself).  Rows that belong to no request are not written: in a new tensor
    they hold anything, in ``out`` what they held.  Softmax and sums are fp32; the
    weights are rounded to the tensors' dtype before they multiply v, and divided
    by the sum of the rounded ones.  A value row that is not finite reaches only
    the tokens that attend to it."""
    return _native.load_host().tree_attention(q, k, v, k_cache, v_cache, block_tables, lens, offsets, parents,
                                              max_tokens, -1 if max_context is None else max(int(max_context), 0),
                                              scale, out)
