"""Decode over a paged KV cache: block tables and slots, append, attention.

The cache of one layer is two tensors ``k_pages`` and ``v_pages`` of
``[pages, kv_heads, page_size, head_dim]`` (bf16 or fp16, head_dim 64 or 128,
any page size that is a multiple of 16). A request's row of the block table
lists its pages in the order of its positions; the slot of a position is
``page * page_size + position % page_size``. One step of a batch whose
requests have different lengths is::

    step = assign_pages(cached, block_tables, free_pages, taken, page_size)
    for each layer:
        q = rope_append_paged(qkv, cos, sin, step.positions, step.slots, k_pages, v_pages, q_heads)
        attn = paged_attention(q, k_pages, v_pages, block_tables, step.lengths)
    cached, taken = step.lengths, step.taken

Lengths, tables and the free list are read on the device: nothing
synchronises, and a captured CUDA graph replays at any lengths. The operators
are for inference: a tensor that requires a gradient, or carries a
forward-mode tangent, is refused. They are functions of the extension module
and not ``torch.ops``: dispatch modes, ``torch.export`` and the like do not see
them, and fake, batched or wrapped tensors are refused. A tensor that a call
writes must not share memory with another one of the call.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _ext
from .errors import after_launch


class PageSlots(NamedTuple):
    """What :func:`assign_pages` gives for one step.

    All four lie in one allocation, which lives as long as any of them: clone
    what is to be kept when the slots of a long prompt are not.
    """

    positions: torch.Tensor  # int32 [tokens]: position in its request
    slots: torch.Tensor      # int64 [tokens]: slot in the cache, -1 where there is none
    lengths: torch.Tensor    # int32 [requests]: positions held after the step
    taken: torch.Tensor      # int32 [1]: entries of the free list used


def assign_pages(cached: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor, taken: torch.Tensor,
                 page_size: int, query_start: torch.Tensor | None = None,
                 num_tokens: int | None = None) -> PageSlots:
    """Gives the new tokens of a step their pages, in one launch.

    ``cached[b]`` positions of request ``b`` are in the cache already. Its new
    tokens are rows ``query_start[b]`` to ``query_start[b + 1]`` of the step
    (int32, starting at 0), or row ``b`` alone without ``query_start``. Pages
    that a request needs beyond those it has come from ``free_pages`` (int32),
    from entry ``taken`` on, in the order of the requests; they are written
    into ``block_tables`` (int32 ``[requests, pages]``) in place, and its
    other entries are left as they are.

    ``num_tokens`` is the number of rows (needed with ``query_start``): rows
    past the last request's, the padding of a batch, get position 0 and slot
    -1. Tokens past ``num_tokens`` get their pages and count in ``lengths``,
    but no position and slot: append them before attending. Where the free list or the table's width runs out, tokens get slot -1
    and the table -1, and ``lengths`` counts only positions that have a page:
    ``lengths[b] < cached[b] + new tokens`` tells it. ``cached`` and ``taken``
    are not changed.
    """
    native = _ext.native()
    if num_tokens is None:
        if query_start is not None:
            raise ValueError("assign_pages needs num_tokens with query_start")
        num_tokens = cached.shape[0]
    r = PageSlots._make(native.assign_pages(cached, query_start, block_tables, free_pages, taken, page_size,
                                            num_tokens))
    if native.check_requested():
        after_launch(cached.device)
    return r


def rope_append_paged(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                      slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, q_heads: int,
                      q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-5,
                      interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Norm and rotation of q and k, and append of k and v to the cache, in one launch.

    ``qkv`` is ``[tokens, (q_heads + 2 * kv_heads) * head_dim]``: q, k and v
    heads side by side (rows may be further apart than that). With ``q_norm``
    or ``k_norm`` (``[head_dim]``) each head of q or k is first divided by its
    root mean square over the head and multiplied by the weight. Then its
    first ``2 * cos.shape[1]`` dims are rotated by the angles of row
    ``positions[t]`` of ``cos`` and ``sin`` (:func:`rope_tables`): pairs
    ``(i, i + rotary_dim / 2)``, or ``(2i, 2i + 1)`` with ``interleaved``.
    All of it in fp32, rounded once.

    k and v of token ``t`` go to slot ``slots[t]``; slots must be distinct,
    and a token with slot -1 is not stored. A token with a slot past the cache
    is not stored either, and a position outside the tables is clamped to
    them; both (the latter for tokens with a slot) are recorded
    (:func:`~numa_allreduce_b200.check_kernels`). Returns q as
    ``[tokens, q_heads, head_dim]``.
    """
    native = _ext.native()
    q = native.rope_append_paged(qkv, cos, sin, positions, slots, k_pages, v_pages, q_heads, q_norm, k_norm, eps,
                                 interleaved, out)
    if native.check_requested():
        after_launch(qkv.device)
    return q


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_tables: torch.Tensor,
                    lengths: torch.Tensor, scale: float | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per request over its pages.

    ``q`` is ``[requests, q_heads, head_dim]`` (consecutive query heads share a
    kv head; rows may be further apart), ``lengths[b]`` the positions that
    request ``b`` attends to, the new token's own among them (append it
    first). ``scale`` defaults to ``1 / sqrt(head_dim)``. Scores, softmax and
    sums are in fp32 (a probability enters its product with v as two 16-bit
    values), with one rounding at the end. A request of length
    0 gives zeros; rows of its pages past a request's length are never used,
    whatever they hold. A length past the table's width is cut to it, and a
    page id outside the cache reads as zeros; both are recorded
    (:func:`~numa_allreduce_b200.check_kernels`).

    Long and short requests may be mixed. The width of the table, which bounds
    the lengths, decides how the work is dealt out: a cluster of CTAs per
    request and kv head for few or short ones; whole requests for many short
    ones; otherwise all positions split evenly over the GPU, and the parts of a
    request joined in a second launch. A table no wider than the step
    needs is the fastest.
    """
    native = _ext.native()
    out = native.paged_attention(q, k_pages, v_pages, block_tables, lengths, scale, out)
    if native.check_requested():
        after_launch(q.device)
    return out


def rope_tables(max_positions: int, rotary_dim: int, theta: float = 10000.0, scale: float = 1.0,
                original_positions: int | None = None, low: float = 1.0, high: float = 4.0,
                device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """``cos`` and ``sin`` of ``[max_positions, rotary_dim / 2]`` for :func:`rope_append_paged`.

    Angle ``i`` of position ``p`` is ``p * theta ** (-2 i / rotary_dim)``,
    computed in 64 bits. ``scale`` stretches the positions for longer contexts
    than the model was trained on: every frequency is divided by it, or, with
    ``original_positions`` (the trained length), only those whose wavelength
    exceeds ``original_positions / low``; wavelengths below
    ``original_positions / high`` keep theirs, and the ones between go over
    from one to the other linearly in ``original_positions / wavelength``.
    """
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rope_tables needs positions and an even rotary_dim")
    if scale <= 0 or theta <= 0 or (original_positions is not None and not 0 < low < high):
        raise ValueError("rope_tables needs theta > 0, scale > 0 and 0 < low < high")
    inv = 1.0 / (theta ** (torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim))
    if original_positions is None:
        inv = inv / scale
    else:
        turns = original_positions * inv / (2 * math.pi)  # over the trained length
        kept = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * (kept + (1 - kept) / scale)
    ang = torch.arange(max_positions, device=device, dtype=torch.float64)[:, None] * inv[None, :]
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()
