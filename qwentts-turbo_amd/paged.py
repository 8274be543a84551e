"""Paged key-value cache: operators that serve many streams from one pool of pages.

A layer's cache is two tensors ``[pages, kv_heads, page_size, head_dim]`` (bf16 or fp16);
``block_table[r, i]`` is the page of request r's tokens ``i * page_size ..`` and a token's slot is
``page * page_size + place in the page``. The reference has one contiguous cache for one stream
(megakernel_backbone.py:156-159). ``csrc/qtts_paged.hip`` and ``csrc/qtts_paged_attn.hip`` hold the kernels.

``BatchedTTSDecoder(mode="paged")`` serves any number of streams this way (``PagedBackbone`` below). By hand, a
step of a batch is ``paged_plan`` once, then per layer ``qk_norm_rope_store`` and
``paged_attention_decode`` (one new token per request) or ``paged_attention_prefill`` (any number).
Every call queues on the current stream, reads lengths and tables on the device, keeps no state and may be
captured into a graph (the shapes are then fixed, the lengths are not).
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import torch

from . import _ext
from .weights import HEAD_DIM, HIDDEN_SIZE, NUM_KV_HEADS


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


class PagedBackbone:
    """The backbone's streams over one pool of pages: ``BatchedTTSDecoder``'s ``mode="paged"``.

    All streams' new tokens go through the layers in one call (``qtts_backbone_paged``: the MFMA projections of the
    prompt prefill around the operators above), whether they are prompts or single tokens. Pages are taken as
    streams grow, so a pool may be smaller than ``n_streams * max_seq_len``; when it runs out, the streams that
    found no page are noted on the device and ``check_error`` raises. ``window`` > 0 bounds what a token attends
    (its last ``window`` keys and the first ``sinks``); pages behind the window stay with their stream."""

    def __init__(self, model, n_streams: int, max_seq_len: int = 4096, page_size: int = 64, num_pages: Optional[int] = None,
                 window: int = 0, sinks: int = 0, device="cuda"):
        from .megakernel_backbone import _extract_tts_backbone_weights
        if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two in [16, 65536], got {page_size}")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must be >= 0")
        self.width = -(-max_seq_len // page_size)
        self.num_pages = n_streams * self.width if num_pages is None else int(num_pages)
        if self.num_pages < 1:
            raise ValueError("num_pages must be >= 1")
        w = _extract_tts_backbone_weights(model, max_seq_len, device=device)
        self.kernel = _ext.load().PagedTTSBackbone(w["layer_weights"], w["final_norm_weight"], w["codec_head_weight"], w["cos_table"],
                                                   w["sin_table"], w["num_layers"])
        self.vocab_size, self.num_layers = w["vocab_size"], w["num_layers"]
        self.n_streams, self.max_seq_len, self.page_size = n_streams, max_seq_len, page_size
        self.window, self.sinks = int(window), int(sinks)
        self.device = torch.device(device)
        pool = (self.num_layers, self.num_pages, NUM_KV_HEADS, page_size, HEAD_DIM)
        self.k_pool = torch.empty(pool, dtype=torch.bfloat16, device=device)
        self.v_pool = torch.empty(pool, dtype=torch.bfloat16, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((n_streams, self.width), -1, **i32)
        self.lengths = torch.zeros(n_streams, **i32)
        self.free_pages = torch.arange(self.num_pages, **i32)
        self.free_count = torch.full((1,), self.num_pages, **i32)
        self.failed = torch.zeros(n_streams, **i32)        # largest plan status of each stream
        self._ones = torch.ones(n_streams, **i32)
        self.positions: List[int] = [0] * n_streams        # tokens asked for, by the host's count

    def reset(self, streams: Optional[Sequence[int]] = None) -> None:
        """Gives the pages of ``streams`` (default: all) back; they start again at position 0."""
        which = range(self.n_streams) if streams is None else streams
        flags = [0] * self.n_streams
        for s in which:
            flags[s] = 1
            self.positions[s] = 0
        mask = torch.tensor(flags, dtype=torch.int32, device=self.device)
        paged_release(mask, self.lengths, self.block_table, self.free_pages, self.free_count, self.page_size)
        self.failed.masked_fill_(mask != 0, 0)

    def _plan(self, counts: Sequence[int], off: Optional[torch.Tensor] = None) -> PagedPlan:
        """``counts[s]`` more tokens of every stream s; none for those that the mask ``off`` marks."""
        if len(counts) != self.n_streams or any(n < 0 for n in counts):
            raise ValueError(f"counts must hold a number of tokens for each of {self.n_streams} streams, got {list(counts)}")
        for s, n in enumerate(counts):
            if self.positions[s] + n > self.max_seq_len:
                raise RuntimeError(f"stream {s}: position {self.positions[s]} + {n} tokens exceeds max_seq_len {self.max_seq_len} "
                                   "(KV cache full)")
        if off is not None:
            new = (~off).to(torch.int32)
        else:
            new = self._ones if all(n == 1 for n in counts) else torch.tensor(list(counts), dtype=torch.int32, device=self.device)
        plan = paged_plan(new, self.lengths, self.block_table, self.free_pages, self.free_count, self.page_size, sum(counts))
        torch.maximum(self.failed, plan.status, out=self.failed)
        for s, n in enumerate(counts):
            self.positions[s] += n
        return plan

    def set_kv_cache(self, stream: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Prefix K and V ([layers, 8, S, 128]) of one stream, which continues at position S."""
        shape = (self.num_layers, NUM_KV_HEADS, k.shape[2] if k.dim() == 4 else -1, HEAD_DIM)
        if tuple(k.shape) != shape or v.shape != k.shape:
            raise ValueError(f"k and v must be [{self.num_layers}, {NUM_KV_HEADS}, S, {HEAD_DIM}], got {tuple(k.shape)} and {tuple(v.shape)}")
        self.reset([stream])
        counts = [0] * self.n_streams
        counts[stream] = int(k.shape[2])
        slots = self._plan(counts).slots.long()
        if not bool((slots >= 0).all()):
            self.reset([stream])
            raise RuntimeError(f"stream {stream}: the pool has too few free pages for {counts[stream]} tokens")
        page, place = slots // self.page_size, slots % self.page_size
        for pool, x in ((self.k_pool, k), (self.v_pool, v)):
            pool[:, page, :, place] = x.to(self.device, torch.bfloat16).permute(2, 0, 1, 3)

    def forward(self, embeds: torch.Tensor, counts: Sequence[int], out_tokens: Optional[torch.Tensor] = None,
                skip: Optional[torch.Tensor] = None, **select) -> torch.Tensor:
        """``counts[s]`` new tokens of every stream s, their embeddings packed in ``embeds`` (bf16 [sum, 1024]), through
        all layers. Returns the final-norm hidden of each stream's last token (f32 [n_streams, 1024]; zeros for a
        stream without tokens or skipped). With ``out_tokens`` each stream's token is selected (``select``: the
        arguments of ``step_select``). ``skip`` needs one token for every stream."""
        single = all(n == 1 for n in counts)
        if skip is not None and not single:
            raise ValueError("skip needs one token for every stream")
        if embeds.shape != (sum(counts), HIDDEN_SIZE) or sum(counts) < 1:
            raise ValueError(f"embeds must be [{sum(counts)}, {HIDDEN_SIZE}] with at least one token, got {tuple(embeds.shape)}")
        # whatever the call refuses, it refuses before a page is taken
        embeds = embeds.to(self.device, torch.bfloat16).contiguous()
        for name, x, size in (("out_tokens", out_tokens, self.n_streams), ("skip", skip, self.n_streams),
                              ("history", select.get("history"), 0), ("n_history", select.get("n_history"), self.n_streams)):
            if x is not None and (x.dtype != torch.int32 or x.device != self.lengths.device or not x.is_contiguous() or x.numel() < size):
                raise ValueError(f"{name} must be a contiguous int32 tensor on {self.lengths.device} with an entry for each stream")
        if select.get("do_sample") and not select.get("temperature", 1.0) > 0:
            raise ValueError("temperature must be > 0")
        off = skip[:self.n_streams] != 0 if skip is not None else None
        plan = self._plan(counts, off)
        slots, positions, lens = plan.slots, plan.positions, plan.kv_lens
        if off is not None:             # a finished stream takes no page, stores and attends nothing; rows stay in stream order
            first = plan.cu_tokens[:-1]
            slots = torch.where(off, -1, slots.index_select(0, first))
            positions = positions.index_select(0, first)
            lens = torch.where(off, 0, lens)
        return self.kernel.forward(embeds, self.k_pool, self.v_pool, self.block_table, slots, positions,
                                   None if single else plan.cu_tokens, lens, max(self.positions), self.window, self.sinks,
                                   out_tokens=out_tokens, skip=skip, **select)

    def check_error(self) -> None:
        """Raises if the pool had no page for some stream since its last reset (synchronises)."""
        bad = [s for s, x in enumerate(self.failed.tolist()) if x]
        if bad:
            raise RuntimeError(f"paged cache: no free page for streams {bad} (pool of {self.num_pages} pages); reset them")
