"""A paged KV cache for requests of different lengths, and the steps of a decoder over it.

The reference holds one row of positions per sequence (``model/transformer_model.py:674``) and has no counterpart to any of this.  Here a request's tokens lie
in pages of a pool, and the new tokens of all requests lie one after another, whatever their number: one each when decoding, a tree of drafted tokens
to verify, a prompt.  A step is

    plan = cache.plan(new_lens, total, parents=parents, max_new=n)                  # pages, positions, slots, masks
    q = rope_paged(q, k, v, plan.positions, plan.slots, frequencies, k_pages, v_pages)      # per layer
    out = paged_attention(q, k_pages, v_pages, cache.tables, cache.lens, plan.starts, masks=plan.masks)
    cache.keep(paths)                                                               # the accepted path of each tree, or cache.append(new_lens)

with nothing read back to the host, so it can be captured into a graph.  Kernels: ``csrc/paged_ops.cu``, ``csrc/rope.cu``, ``csrc/paged_attention.cu``.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _native

_LAYOUTS = {"half": 0, "interleaved": 1, "split": 2}


class PagedPlan(NamedTuple):
    """What ``paged_plan`` says of the new tokens."""
    starts: torch.Tensor             # int32 [requests + 1]: rows [starts[i], starts[i + 1]) are request i's
    positions: torch.Tensor          # int64 [total]
    slots: torch.Tensor              # int64 [total]: page * page_size + row in it; -1 where there is none
    masks: Optional[torch.Tensor]    # int32 [total, words]: bit j says that new token j is an ancestor or the token itself
    held: torch.Tensor               # int32 [requests]: pages that each now holds
    free_count: torch.Tensor         # int32 [2]: pages left on the list, and pages that were missing


def paged_plan(lens: torch.Tensor, new_lens: torch.Tensor, tables: torch.Tensor, held: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, page_size: int, total: int, *,
               parents: Optional[torch.Tensor] = None, max_new: int = 0, held_out: Optional[torch.Tensor] = None,
               free_count_out: Optional[torch.Tensor] = None) -> PagedPlan:
    """Makes the block ``tables`` [requests, width] fit ``lens`` cached and ``new_lens`` new tokens, and places the new ones.

    All int32 CUDA tensors; ``free[:free_count[0]]`` are the free pages.  Pages that a request holds beyond its need go onto the list (all of them for one with no tokens
    left), then those that are missing come from its top, both in the order of requests.  ``tables`` and ``free`` are changed in place; ``held`` and ``free_count`` are
    not, unless they are given as ``held_out`` and ``free_count_out``.  ``total`` is the number of token rows, at least the sum of ``new_lens``: rows behind have position and
    slot -1.  Where pages run out, tokens have slot -1 and ``free_count[1]`` says how many pages were missing.

    ``parents`` [total] makes trees of the new tokens: the index, in its request, of the earlier token that a token continues, or -1 for the cached tokens.  Its position is
    then ``lens`` plus its depth, and ``masks`` names its ancestors; ``max_new`` (at most 256) bounds the new tokens of a request.  At most 4096 requests; pages of
    a power of two."""
    return PagedPlan(*_native.paged_plan(lens, new_lens, tables, held, free, free_count, page_size, total, parents, max_new, held_out, free_count_out))


class RopeFrequencies(NamedTuple):
    """Rotary frequencies as ``rope`` takes them: one per pair, in turns a position as fractions of 2^64, and the factor of cosines and sines."""
    turns: torch.Tensor              # int64 [rotary / 2]
    amplitude: float = 1.0


def scaled_frequencies(rotary: int, theta: float = 10000.0, scaling: Optional[dict] = None):
    """Radians a position of each pair (float64, on the host) and the amplitude: ``theta ** (-2 i / rotary)``, scaled for contexts longer than the trained one.

    ``scaling`` is None or a dict with a ``kind`` and a ``factor``: ``"linear"`` divides all frequencies by the factor; ``"base"`` grows theta so that the slowest pair slows down
    by the factor; ``"bands"`` divides those of pairs that turn fewer than ``low`` times over the ``original`` context, leaves those that turn more than ``high`` times, and
    goes over linearly in between; ``"yarn"`` does the same along the index of the pair (Peng et al., YaRN: efficient context window extension of large language
    models, 2023) and raises the amplitude to 0.1 ln(factor) + 1, for factors above 1."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64)
    f = theta ** (-i / rotary)
    if scaling is None:
        return f, 1.0
    kind, factor = scaling["kind"], float(scaling["factor"])
    if not factor > 0:
        raise ValueError(f"gpuk: rotary scaling by {factor}")
    if kind == "linear":
        return f / factor, 1.0
    if kind == "base":
        if rotary <= 2:
            raise ValueError("gpuk: one pair has no base to scale")
        return (theta * factor ** (rotary / (rotary - 2))) ** (-i / rotary), 1.0
    if kind not in ("bands", "yarn"):
        raise ValueError(f"gpuk: unknown rotary scaling {kind!r}; choose from linear, base, bands, yarn")
    low, high, original = float(scaling["low"]), float(scaling["high"]), float(scaling["original"])
    if not 0 < low < high or not original > 0:
        raise ValueError("gpuk: rotary scaling needs 0 < low < high and an original context")
    if kind == "bands":
        stay = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f / factor * (1 - stay) + f * stay, 1.0
    # the ramp may end beyond the last pair, where all turn more than `low` times: none of them is divided by the whole factor then
    first = max(math.floor(rotary * math.log(original / (high * 2 * math.pi)) / (2 * math.log(theta))), 0)
    last = min(math.ceil(rotary * math.log(original / (low * 2 * math.pi)) / (2 * math.log(theta))), rotary - 1)
    slow = ((i / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
    return f / factor * slow + f * (1 - slow), 0.1 * math.log(max(factor, 1.0)) + 1.0


def rope_frequencies(rotary: int, theta: float = 10000.0, *, scaling: Optional[dict] = None, device=None) -> RopeFrequencies:
    """The frequencies of ``scaled_frequencies`` in fixed point, for ``rope`` and ``rope_paged``: made once per model."""
    if rotary <= 0 or rotary % 2:
        raise ValueError(f"gpuk: {rotary} rotated values are no pairs")
    f, amplitude = scaled_frequencies(rotary, theta, scaling)
    turns = [round(math.ldexp(v / (2 * math.pi), 64)) % (1 << 64) for v in f.tolist()]
    return RopeFrequencies(torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64).to(device), amplitude)


def _layout(name: str) -> int:
    if name not in _LAYOUTS:
        raise ValueError(f"gpuk: unknown order of rotary pairs {name!r}; choose from {sorted(_LAYOUTS)}")
    return _LAYOUTS[name]


def rope(x: torch.Tensor, positions: torch.Tensor, frequencies: RopeFrequencies, *, layout: str = "half", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of ``x`` [tokens, heads, head_dim] (bf16 or fp16, any strides of tokens and heads) at ``positions`` (int64): the first ``2 * len(turns)`` values of each head
    are rotated in fp32 and rounded once, the others copied.  Pairs are (i, i + rotary / 2) for ``"half"``, (2 i, 2 i + 1) for ``"interleaved"``, and for ``"split"`` (2 i, 2 i + 1)
    that come out as (i, i + rotary / 2), as this library's decoder has them.  ``out`` may be ``x``, but for ``"split"``.  Head sizes in multiples of 16, at most 256 rotated."""
    return _native.rope(x, positions, frequencies.turns, frequencies.amplitude, _layout(layout), out)


def rope_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, frequencies: RopeFrequencies, k_pages: torch.Tensor,
               v_pages: torch.Tensor, *, layout: str = "half", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``rope`` of the queries, and of the keys into their ``slots`` of ``k_pages`` [pages, kv_heads, page_size, head_dim]; the values go to ``v_pages`` as they are.  Returns the
    queries.  A token whose slot is negative or outside the pages writes neither, and its queries are NaN; ``gpuk_fp8_linear_status`` reports one outside.
    No two tokens may have one slot.  The pages may be views with other orders of their first three dimensions."""
    return _native.rope_paged(q, k, v, positions, slots, frequencies.turns, frequencies.amplitude, _layout(layout), k_pages, v_pages, out)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, starts: torch.Tensor, *,
                    masks: Optional[torch.Tensor] = None, max_len: Optional[int] = None, max_new: Optional[int] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens ``q`` [tokens, heads, head_dim] over their requests' pages, in which their own keys and values are already, behind ``lens`` cached ones.

    A token sees the cached ones and, of its request's new ones, those up to itself, or with ``masks`` (``PagedPlan.masks``, or any words [tokens, words <= 8]) those whose bits are
    set.  One that sees no key gets zeros; what it does not see does not reach it, be it infinite or NaN.  Rows behind ``starts[-1]`` are left as they are in
    ``out``.  ``max_len`` bounds cached plus new tokens of a request (default: what the table holds), ``max_new`` the new tokens of
    one (default: 1 in calls with no more tokens than requests): speed hints, which change no more than the order of sums.  ``scale`` defaults to
    1 / sqrt(head_dim).  Heads of 64 or 128, bf16 or fp16, pages of 8 tokens or more; the same inputs give the same bits."""
    if scale is not None and not 0.0 < scale < math.inf:
        raise ValueError(f"gpuk: a scale of {scale} is no positive number")
    if max_new is not None and max_new < 1:
        raise ValueError(f"gpuk: at most {max_new} new tokens of a request")
    return _native.paged_attention(q, k_pages, v_pages, tables, lens, starts, masks, -1 if max_len is None else max_len, 0 if max_new is None else max_new,
                                   0.0 if scale is None else scale, out)


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, paths: torch.Tensor, *, held: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Makes the accepted path of each request's tree its next cached tokens: new token ``paths[i, j]`` moves to ``lens[i] + j``, in ``k_pages`` and ``v_pages`` of one layer or
    [layers, pages, kv_heads, page_size, head_dim] of all.  A path ascends and ends at its first entry that does not (-1); it names
    tokens of the last plan only, for only they have pages.  ``held`` (``PagedPlan.held``) ends a path at the first token for which no page was to be had: what was never written does
    not become cached.  Returns the new lengths."""
    return _native.paged_keep(k_pages, v_pages, tables, lens, paths, held, out)


class PagedKVCache:
    """Pages of all layers, the block tables of ``requests`` requests, and the list of free pages; every tensor stays where it is, so a captured step can be replayed.

    Where the pool or a row of the table runs out, tokens of a plan have no slot and NaN logits.  ``append`` and ``keep`` leave them out: a request's cached tokens end in front of the
    first of them, which can be given again once there are pages."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, requests: int, pages_per_request: int, *, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        # what the calls of a step would refuse is refused before there is one
        for name, size, least in (("layers", layers, 1), ("pages", pages, 1), ("kv_heads", kv_heads, 1), ("requests", requests, 0), ("pages_per_request", pages_per_request, 1)):
            if size < least:
                raise ValueError(f"gpuk: a paged cache with {name}={size}")
        if not 8 <= page_size <= 65536 or page_size & (page_size - 1):
            raise ValueError(f"gpuk: pages of {page_size} tokens; attention is built for powers of two from 8 to 65536")
        if head_dim not in (64, 128):
            raise ValueError(f"gpuk: heads of {head_dim}; attention over pages is built for 64 and 128")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"gpuk: a paged cache of {dtype}; it is bfloat16 or float16")
        if requests > 4096:
            raise ValueError(f"gpuk: {requests} requests; a plan is built for at most 4096")
        if pages_per_request * page_size > 0x7fffff00 or requests * pages_per_request > 0x7fffffff:
            raise ValueError(f"gpuk: tables of {requests} requests with pages_per_request={pages_per_request} are too large")
        self.page_size = page_size
        self.k, self.v = (torch.zeros(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        ints = {"dtype": torch.int32, "device": device}
        self.tables = torch.full((requests, pages_per_request), -1, **ints)
        self.lens, self.held = torch.zeros(requests, **ints), torch.zeros(requests, **ints)
        self.free, self.free_count = torch.arange(pages, **ints), torch.tensor([pages, 0], **ints)

    def plan(self, new_lens: torch.Tensor, total: int, *, parents: Optional[torch.Tensor] = None, max_new: int = 0) -> PagedPlan:
        """``paged_plan`` for the cached tokens and ``new_lens`` more; tables and list are advanced."""
        return paged_plan(self.lens, new_lens, self.tables, self.held, self.free, self.free_count, self.page_size, total, parents=parents, max_new=max_new, held_out=self.held,
                          free_count_out=self.free_count)

    def append(self, new_lens: torch.Tensor) -> None:
        """All new tokens of the last plan that have a page are cached from here on."""
        torch.clamp(self.lens + new_lens, self.lens, self.held * self.page_size, out=self.lens)      # the upper bound wins

    def keep(self, paths: torch.Tensor) -> None:
        """Of the last plan's trees, the paths [requests, depth] are cached from here on (``paged_keep``); what else the pages hold is given back by the next plan."""
        self.lens.copy_(paged_keep(self.k, self.v, self.tables, self.lens, paths, held=self.held))

    def release(self, requests) -> None:
        """Ends requests: their pages go back to the list with the next plan, in which they have no new tokens."""
        self.lens[requests] = 0
