"""A key / value cache of pages, held in 8 bits, and attention over it.

What the reference's decoding loop (functs/benchmark/simpleops/attention/attention.py:38-58) does with two fp32
tensors of one length, for many requests of any length: requests share a pool of pages, a table names each one's
pages, keys and values are codes of one byte (float8_e4m3fn or int8) under a scale for each page and head.

    cache = KvCache.empty(pages, heads, page_size, depth)
    step = cache.plan(past_lens, new_lens, block_table, free_pages, max_tokens)   # once a step
    cache.store(k, v, step.slots)                                                 # in every layer
    q = cache.append(q, k, v, step.slots, step.positions, frequencies)            # (the same for a model with rotary positions)
    out, lse = cache.attention(q, block_table, step.lens, step.starts)
    k, v = cache.read(slots, torch.bfloat16)                                      # the numbers again
    fork = cache.fork(parents, lens, block_table, free_pages)                     # beams: behind their selection (functs_amd.beam)
    copy_pages(layers, fork.copies)                                               # in all layers at once

The same calls are TorchScript operators on the cache's tensors: torch.ops.functs.kv_plan, kv_store, kv_append, kv_read,
kv_attention, kv_fork, kv_copy.  Lengths, tables and slots are read on the device and nothing waits for it: a step captured into a graph
serves any lengths that fit its tensors.  include/fxhip.h defines the layout, the codes and every rule.

GPU tensors only: there is no host fallback, and no backward pass (codes are steps).
"""
from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _C  # noqa: F401  (registers the operators)
from . import _lib
from ._lib import C

PAGE_SIZES = (16, 32, 64, 128, 256)
MAX_DEPTH = C["FX_KV_MAX_DEPTH"]


class Step(NamedTuple):
    """Where the tokens of a step go.  slots [tokens] int64 and positions [tokens] int32: -1 for tokens of requests that
    were not granted, and behind the last token; starts [requests + 1]; lens [requests]: tokens after the step, 0 for requests that were
    not granted; taken [1]: how many of the free pages were given out."""
    slots: Tensor
    positions: Tensor
    starts: Tensor
    lens: Tensor
    taken: Tensor


class Fork(NamedTuple):
    """What KvCache.fork says.  lens [rows]: tokens of the new rows, 0 where a row continues none or got no page; copies [rows, 3]: (page, to page, tokens) for copy_pages,
    -1, -1, 0 where nothing is to be copied; taken [1]: how many of the free pages were given out; freed [rows * columns]: pages that no row has any more, the first
    n_freed[0] of them, -1 behind."""
    lens: Tensor
    copies: Tensor
    taken: Tensor
    freed: Tensor
    n_freed: Tensor


def copy_pages(caches: Sequence["KvCache"], copies: Tensor) -> None:
    """Copies pages as Fork.copies says, in all caches (layers of a model, of the same sizes) at once."""
    torch.ops.functs.kv_copy([c.k for c in caches], [c.v for c in caches], [c.k_scale for c in caches], [c.v_scale for c in caches], copies)


class KvCache:
    """The four tensors of a cache: k [pages, heads, page_size, depth], v [pages, heads, page_size / 16, depth, 16],
    k_scale and v_scale [pages, heads]."""

    def __init__(self, k: Tensor, v: Tensor, k_scale: Tensor, v_scale: Tensor):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int, depth: int, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> "KvCache":
        """Memory for `pages` pages; nothing is expected in it (a page starts anew with its first token)."""
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise _lib.FxError(C["FX_E_UNSUPPORTED"], "a cache holds float8_e4m3fn or int8, not %s" % dtype)
        if page_size not in PAGE_SIZES:
            raise _lib.FxError(C["FX_E_UNSUPPORTED"], "page_size must be one of %s, got %s" % (PAGE_SIZES, page_size))
        if depth % 16 != 0 or not 16 <= depth <= MAX_DEPTH:
            raise _lib.FxError(C["FX_E_UNSUPPORTED"], "depth must be a multiple of 16 up to %d, got %s" % (MAX_DEPTH, depth))
        if pages < 1 or heads < 1:
            raise _lib.FxError(C["FX_E_INVALID"], "a cache has at least one page and one head")
        k = torch.empty(pages, heads, page_size, depth, dtype=dtype, device=device)
        v = torch.empty(pages, heads, page_size // 16, depth, 16, dtype=dtype, device=device)
        return cls(k, v, torch.empty(pages, heads, device=device), torch.empty(pages, heads, device=device))

    @property
    def page_size(self) -> int:
        return self.k.size(2)

    def plan(self, past_lens: Tensor, new_lens: Tensor, block_table: Tensor, free_pages: Tensor, max_tokens: int,
             free_start: Optional[Tensor] = None) -> Step:
        """Pages and slots for new_lens[b] more tokens of each request (int32, on the GPU), whose rows lie one request behind the
        other in arrays of max_tokens rows.  New pages come from free_pages (from free_pages[free_start[0]] on), request by request,
        and are entered in block_table [requests, columns]; a request that does not fit gets nothing."""
        return Step(*torch.ops.functs.kv_plan(past_lens, new_lens, block_table, free_pages, self.page_size, max_tokens, free_start))

    def fork(self, parents: Tensor, lens: Tensor, block_table: Tensor, free_pages: Tensor, free_start: Optional[Tensor] = None) -> Fork:
        """The tables of beams behind a selection: row g * beams + j of block_table [groups * beams, columns] continues row g * beams + parents[g, j] (int32 [groups, beams], as
        beam.select() gives them) with its lens[] tokens.  Full pages are shared; a partly filled one has one owner, the other rows that continue it get pages of rows that
        nobody continues, or free ones, and are to be copied.  Call it once a step, and copy_pages() for all layers before anything is stored."""
        return Fork(*torch.ops.functs.kv_fork(parents, lens, block_table, free_pages, self.page_size, free_start))

    def store(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Writes rows k, v [tokens, heads, depth] to `slots`.  The rows of one page are neighbours, as plan() lays them; a page
        starts anew where the first of them is its first token."""
        torch.ops.functs.kv_store(k, v, self.k, self.v, self.k_scale, self.v_scale, slots)

    def append(self, q: Tensor, k: Tensor, v: Tensor, slots: Tensor, positions: Tensor, frequencies: Tensor, magnitude: float = 1.0,
               interleaved: bool = False) -> Tensor:
        """store() of keys that turn by their tokens' positions on the way (functs_amd.rotary), in fp32 and rounded once, to their codes.  Returns
        the queries q [tokens, query heads, depth] turned, as rotary.rotary() gives them; one launch for all."""
        return torch.ops.functs.kv_append(q, k, v, self.k, self.v, self.k_scale, self.v_scale, slots, positions, frequencies, magnitude, interleaved)

    def read(self, slots: Tensor, dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor]:
        """Keys and values [tokens, heads, depth] at `slots`, as numbers; zeros for slots outside the cache."""
        return torch.ops.functs.kv_read(self.k, self.v, self.k_scale, self.v_scale, slots, dtype)

    def attention(self, q: Tensor, block_table: Tensor, lens: Tensor, starts: Tensor, scale: Optional[float] = None, window: int = 0,
                  max_new: int = 0, out: Optional[Tensor] = None, lse: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """Rows starts[b] to starts[b + 1] of q [tokens, query heads, depth] are the last tokens of request b's lens[b]; each sees
        the tokens up to its own (the last `window` of them, if not 0).  Returns the weighted values (type of q) and the logarithm of
        the sum of exponentials (fp32 [tokens, query heads]).  scale: depth ** -0.5 unless given, 2^-26 to 32.  max_new: the most rows of one request, if known (1
        for a decoding step): a matter of speed, and of how results are rounded, as the number of rows of a call is (fx_kv_attention in
        include/fxhip.h).  With out and lse, rows of no request stay as they are there; out does not overlap q."""
        if scale is None:
            scale = self.k.size(3) ** -0.5
        args = (q, self.k, self.v, self.k_scale, self.v_scale, block_table, lens, starts, scale, window, max_new)
        if (out is None) != (lse is None):
            raise _lib.FxError(C["FX_E_INVALID"], "out and lse are given together")
        if out is None:
            return torch.ops.functs.kv_attention(*args)
        return torch.ops.functs.kv_attention.out(*args, out=out, lse=lse)
