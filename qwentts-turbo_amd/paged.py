"""Paged key-value cache: operators that serve many streams from one pool of pages.

A layer's cache is two tensors ``[pages, kv_heads, page_size, head_dim]`` (bf16 or fp16);
``block_table[r, i]`` is the page of request r's tokens ``i * page_size ..`` and a token's slot is
``page * page_size + place in the page``. The reference has one contiguous cache for one stream
(megakernel_backbone.py:156-159). ``csrc/qtts_paged.hip`` and ``csrc/qtts_paged_attn.hip`` hold the kernels.

A step of a batch is ``paged_plan`` once, then per layer ``qk_norm_rope_store`` and
``paged_attention_decode`` (one new token per request) or ``paged_attention_prefill`` (any number).
Every call queues on the current stream, reads lengths and tables on the device, keeps no state and may be
captured into a graph (the shapes are then fixed, the lengths are not).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from . import _ext


class PagedPlan(NamedTuple):
    """Where the new tokens of a batch go (device int32 tensors)."""
    slots: torch.Tensor       # [total_tokens] slot of each token, -1 where it has none
    positions: torch.Tensor   # [total_tokens] position of each token in its request
    cu_tokens: torch.Tensor   # [requests + 1] first token of each request
    kv_lens: torch.Tensor     # [requests] tokens held with the new ones; 0 where refused
    status: torch.Tensor      # [requests] 0 granted, 1 pool short, 2 table row full, 3 past total_tokens


def paged_plan(new_tokens: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, total_tokens: int, *, lengths_out: Optional[torch.Tensor] = None,
               free_count_out: Optional[torch.Tensor] = None) -> PagedPlan:
    """Pages, slots and positions for ``new_tokens[r]`` more tokens of every request r, which holds
    ``lengths[r]`` (both int32 [requests]). Pages come from the top of the stack ``free_pages[:free_count]``
    (int32; ``free_count`` int32 [1]) in request order, and go into ``block_table`` (int32
    [requests, width]); a request that finds too few pages is refused, and so is every later one that
    needs a page. ``lengths`` and ``free_count`` are updated, or ``lengths_out`` / ``free_count_out`` written
    instead. ``total_tokens``: entries of the packed token arrays (at least the sum of the new tokens; a
    padded batch may have more, which get slot -1)."""
    return PagedPlan(*_ext.load().paged_plan(new_tokens, lengths, block_table, free_pages, free_count, int(page_size),
                                             int(total_tokens), lengths_out, free_count_out))


def paged_release(release: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                  free_count: torch.Tensor, page_size: int) -> None:
    """Gives the pages of every request r with ``release[r] != 0`` (int32 [requests]) back to the stack; its
    length becomes 0 and its table entries -1."""
    _ext.load().paged_release(release, lengths, block_table, free_pages, free_count, int(page_size))


def qk_norm_rope_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
                       k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                       slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *, eps: float = 1e-6,
                       mrope_section: Sequence[int] = (24, 20, 20), out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMSNorm of every query and key head (gains ``q_weight`` / ``k_weight`` [head_dim], None: no norm),
    rotation by the rows ``positions`` of the tables ``cos`` / ``sin`` (``rope_tables``: [rows, head_dim], both
    halves alike; the cache's type or f32), and K and V into their slots. Computed in f32, rounded once.
    ``q`` [tokens, heads, head_dim] and ``k``, ``v`` [tokens, kv_heads, head_dim] may be views of one
    projection's output. ``positions``: int32 [tokens], or [3, tokens] (t, h, w) with interleaved
    ``mrope_section``; clamped into the tables. A token with a slot below 0 or past the pages is skipped:
    nothing of it is written. Returns the rotated queries (``out``, which may be ``q``, or a new tensor)."""
    return _ext.load().qk_norm_rope_store(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, float(eps),
                                          [int(x) for x in mrope_section], out)


def paged_attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           kv_lens: torch.Tensor, *, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                           max_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per request (``q`` [requests, heads, head_dim], at position
    ``kv_lens[r] - 1``) over its pages. ``window`` > 0 keeps the last ``window`` keys and the first ``sinks``.
    ``scale`` defaults to head_dim ** -0.5. ``max_len``: the longest request as far as the host knows (default:
    what a table row holds); it decides how the keys are split over the GPU, not what is computed. A request
    of length 0 gets zeros; what pages hold past a request's length does not matter."""
    return _ext.load().paged_attention_decode(q, k_cache, v_cache, block_table, kv_lens, _scale(scale, q), int(window),
                                              int(sinks), _max_len(max_len, block_table, k_cache), out)


def paged_attention_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                            kv_lens: torch.Tensor, cu_tokens: torch.Tensor, *, scale: Optional[float] = None, window: int = 0,
                            sinks: int = 0, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new tokens of every request: ``q`` [tokens, heads, head_dim] packs them, request
    r's at ``cu_tokens[r] .. cu_tokens[r + 1]``, the last at position ``kv_lens[r] - 1``; their K and V are in
    the cache already. Otherwise as ``paged_attention_decode``; rows past the last request's tokens are left as
    they are in ``out``."""
    return _ext.load().paged_attention_prefill(q, k_cache, v_cache, block_table, kv_lens, cu_tokens, _scale(scale, q),
                                               int(window), int(sinks), _max_len(max_len, block_table, k_cache), out)


def _scale(scale, q):
    return float(scale) if scale is not None else float(q.shape[-1]) ** -0.5


def _max_len(max_len, block_table, k_cache):
    return int(max_len) if max_len is not None else max(1, block_table.shape[-1] * k_cache.shape[-2])
