"""Uncompressed paged KV cache: the operators of a decode step.

Compressed weights leave HBM to the KV cache, and a server's ordinary cache is
an uncompressed paged one. These operators run a step of it without a length or
a table on the host, so a step can be captured in a CUDA graph:

* plan_step         block tables, slots and positions from request lengths
* rope_write        rotary positions (one or several axes) on q and k, k and v
                    written to their slots
* paged_attention   one new token per sequence over its pages, or over a list
                    of them
* page_bounds, select_pages, sparse_attention
                    8-bit bounds of complete pages, the choice of pages by
                    those bounds, attention over the chosen pages
* PagedKVCache      the buffers, and the calls above on them

A page pool is a tensor of logical shape [num_blocks, page_size, heads, dim],
bf16 or fp16, its last axis contiguous and the others of any strides that are
multiples of 8 elements: `torch.empty(blocks, heads, page, dim).transpose(1, 2)`
keeps each head's rows of a page together. Every call runs on the current
stream of its tensors' device and synchronises nothing. `err` (optional, int32[1])
collects error bits: 2 = an index was out of range (skipped; a position: taken as
0), 4 = a request was refused by plan_step.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os
from typing import NamedTuple, Optional, Sequence

import torch

from ._lib import ZipServError
from .build_lib import BINDING

_native = None


def _load():
    """The binding (csrc/binding/paged_bind.cpp): argument checks, outputs, launches."""
    global _native
    if _native is None:
        if not os.path.exists(BINDING):
            raise ZipServError(f"{BINDING} is not built (python -m zipserv_asplos26_b200.build_lib)")
        loader = importlib.machinery.ExtensionFileLoader("_paged_native", BINDING)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_paged_native", loader))
        loader.exec_module(module)
        _native = module
    return _native


# ------------------------------------------------------------------- plan
class StepPlan(NamedTuple):
    """What plan_step returns; tokens past cu_tokens[-1] have slot -1, token_seq -1 and position 0."""
    seq_lens: torch.Tensor      # int32 [R]
    free_count: torch.Tensor    # int32 [1]
    cu_tokens: torch.Tensor     # int32 [R + 1], prefix sums of the admitted tokens
    slots: torch.Tensor         # int64 [max_tokens], block * page_size + row
    token_seq: torch.Tensor     # int32 [max_tokens]
    positions: torch.Tensor     # int32 [max_tokens]
    refused: torch.Tensor       # bool [R]


def plan_step(block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
              free_count: torch.Tensor, page_size: int, max_tokens: int, out: Optional[StepPlan] = None,
              err: Optional[torch.Tensor] = None) -> StepPlan:
    """Block tables, slots and positions of one step, on the GPU.

    Request r has seq_lens[r] tokens and gets new_lens[r] more (negative: it has
    ended and its pages return to the free list). A request is admitted, in
    order, when the tokens asked for up to it fit max_tokens, its pages fit the
    table's width and the pages needed up to it are free; otherwise it keeps its
    state and is marked refused.
    block_table and free_blocks (a stack, its first free_count[0] entries) are
    updated in place; the new lengths and count are returned."""
    return (_native or _load()).plan_step(block_table, seq_lens, new_lens, free_blocks, free_count, page_size,
                                          max_tokens, out, err, StepPlan)


# ----------------------------------------------------------- rotary + write
def rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
               slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               sections: Optional[Sequence[int]] = None, interleaved: bool = False,
               q_out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turn q [N, Hq, D] and k [N, Hkv, D] by their positions and write k and v
    to their slots of the cache; returns the turned q.

    cos_sin is fp32 [rows, rot]: rot / 2 cosines, then rot / 2 sines per
    position; the first rot channels of a head turn, in pairs (j, j + rot / 2),
    or (2j, 2j + 1) when interleaved. positions is int32 [N], or [A, N] with one
    row per axis and `sections` (sum rot / 2) saying how many pairs follow each
    axis in turn. Slots (int64, distinct) of -1 are skipped. q, k and v may be
    slices of one projection. q_out (contiguous) may be q itself where q is
    contiguous, and else lies apart from q, k and v."""
    return (_native or _load()).rope_write(q, k, v, positions, cos_sin, slots, k_pages, v_pages, sections,
                                           interleaved, q_out, err)


# -------------------------------------------------------------- attention
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, softmax_scale: Optional[float] = None,
                    pages: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    max_seqlen: Optional[int] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, Hq, D] (or [B, 1, Hq, D]),
    over the first seq_lens[b] tokens of its pages; D is 64 or 128.

    With pages (int32 [B, Hkv, top], distinct logical pages) and counts (int32
    [B, Hkv]) only the listed pages' tokens count. A sequence with nothing to
    attend gets zeros. lse (optional, fp32 [B, Hq]) receives the log of the sum
    of exponentials of the scaled scores. max_seqlen is a bound on seq_lens that
    the host may have (else the table's width is one); only the choice of the
    kernel, and with it the order of sums, depends on it: short sequences want a
    close one. Lengths count up to the table's width."""
    o = (_native or _load()).paged_attention(q, k_pages, v_pages, block_table, seq_lens, softmax_scale, pages, counts,
                                             out, lse, max_seqlen, err)
    return o if q.dim() == 3 and out is None else o.view(q.shape)


# ------------------------------------------------------------------ sparse
def page_bounds(k_pages: torch.Tensor, block_table: torch.Tensor, lens_before: torch.Tensor, seq_lens: torch.Tensor,
                page_codes: torch.Tensor, page_scales: torch.Tensor, max_new: int,
                max_total: Optional[int] = None, err: Optional[torch.Tensor] = None) -> None:
    """Bounds of the pages that sequences completed between lens_before and
    seq_lens, written to page_codes int8 [num_blocks, Hkv, 2, D] (upper, lower)
    and page_scales fp32 [num_blocks, Hkv]. At most max_new tokens are new in a
    sequence, and at most max_total in all sequences where it is given."""
    (_native or _load()).page_bounds(k_pages, block_table, lens_before, seq_lens, page_codes, page_scales, max_new,
                                     max_total, err)


def select_pages(q: torch.Tensor, page_codes: torch.Tensor, page_scales: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, page_size: int, top_pages: int, sink_pages: int = 1, local_pages: int = 1,
                 err: Optional[torch.Tensor] = None):
    """Up to top_pages pages per (sequence, KV head): the first sink_pages, the
    last local_pages (the newest, possibly incomplete, among them) and the best
    of the others by a score: the largest q . k that the page's bounds allow, of q
    rounded to 8 bits (so keys near the clamp of the codes may pass it). Returns pages
    (int32 [B, Hkv, top_pages], ascending, -1 past the count) and counts."""
    return (_native or _load()).select_pages(q, page_codes, page_scales, block_table, seq_lens, page_size, top_pages,
                                             sink_pages, local_pages, err)


def sparse_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_codes: torch.Tensor,
                     page_scales: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, top_pages: int,
                     sink_pages: int = 1, local_pages: int = 1, softmax_scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None):
    """select_pages, then paged_attention over the chosen pages. Returns (out, pages, counts)."""
    o, pages, counts = (_native or _load()).sparse_attention(q, k_pages, v_pages, page_codes, page_scales, block_table,
                                                             seq_lens, top_pages, sink_pages, local_pages,
                                                             softmax_scale, out, err)
    return (o if q.dim() == 3 and out is None else o.view(q.shape)), pages, counts


# ------------------------------------------------------------------- cache
class TokenRows(NamedTuple):
    """What each token of a plan attends: the pages of its row, up to itself."""
    block_table: torch.Tensor   # int32 [tokens, max_blocks_per_seq]
    seq_lens: torch.Tensor      # int32 [tokens], 0 past the plan's last token


class PagedKVCache:
    """Buffers of an uncompressed paged cache of num_layers layers for up to
    max_batch sequences of up to max_blocks_per_seq pages, and a step's calls on
    them (a plan and its rows a step, the others a layer):

        plan = cache.step(new_lens, max_tokens)            # tokens of each row; -1: ended
        rows = cache.token_rows(plan)                      # what each token attends
        q = cache.write(q, k, v, cos_sin, plan, layer)     # rotary, then into the pages
        o = cache.attention(q, layer, rows=rows)           # output of each token
        o = cache.sparse_attention(q, 64, layer, rows=rows)[0]   # over 64 pages per KV head

    A plan holds the admitted tokens one after another, so its i-th token belongs
    to row plan.token_seq[i], not to row i: without `rows` the attention calls
    take one query per row instead, in order of rows.

    All state (tables, lengths, the free list) is on the GPU in fixed buffers, so
    a step can be captured in a CUDA graph and replayed. layout "heads" keeps
    each head's rows of a page together, "tokens" each token's heads. bounds
    keeps the pages' 8-bit bounds for sparse_attention."""

    def __init__(self, num_blocks: int, max_batch: int, max_blocks_per_seq: int, num_kv_heads: int,
                 head_dim: int = 128, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, layout: str = "heads",
                 bounds: bool = True, num_layers: int = 1, device="cuda"):
        if min(num_blocks, max_batch, max_blocks_per_seq, num_kv_heads, num_layers) <= 0:
            raise ValueError("sizes must be positive")
        if layout not in ("heads", "tokens"):
            raise ValueError(f"unknown layout {layout!r}")
        if dtype not in (torch.bfloat16, torch.float16) or head_dim not in (64, 128):
            raise ValueError("pages hold bf16 or fp16 heads of dim 64 or 128")
        if not 16 <= page_size <= 256 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two from 16 to 256")
        self.Hkv, self.D, self.page_size, self.max_batch = num_kv_heads, head_dim, page_size, max_batch

        def pool():
            if layout == "heads":
                return torch.zeros(num_blocks, num_kv_heads, page_size, head_dim, dtype=dtype,
                                   device=device).transpose(1, 2)
            return torch.zeros(num_blocks, page_size, num_kv_heads, head_dim, dtype=dtype, device=device)

        self.k = [pool() for _ in range(num_layers)]
        self.v = [pool() for _ in range(num_layers)]
        self.device = self.k[0].device
        i32 = dict(dtype=torch.int32, device=self.device)
        self.block_table = torch.full((max_batch, max_blocks_per_seq), -1, **i32)
        self.seqlens = torch.zeros(max_batch, **i32)
        self.lens_before = torch.zeros(max_batch, **i32)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_blocks, **i32)
        self._count_before = torch.zeros(1, **i32)
        self.err = torch.zeros(1, **i32)
        self.codes = self.scales = None
        if bounds:
            self.codes = [torch.zeros(num_blocks, num_kv_heads, 2, head_dim, dtype=torch.int8, device=self.device)
                          for _ in range(num_layers)]
            self.scales = [torch.zeros(num_blocks, num_kv_heads, dtype=torch.float32, device=self.device)
                           for _ in range(num_layers)]

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> StepPlan:
        """Admit new_lens (int32 [max_batch]; negative: the row has ended) tokens
        to the rows; max_tokens bounds their sum."""
        self.lens_before.copy_(self.seqlens)
        self._count_before.copy_(self.free_count)
        e, dev, R = torch.empty, self.device, self.max_batch
        out = StepPlan(self.seqlens, self.free_count, e(R + 1, dtype=torch.int32, device=dev),
                       e(max_tokens, dtype=torch.int64, device=dev), e(max_tokens, dtype=torch.int32, device=dev),
                       e(max_tokens, dtype=torch.int32, device=dev), e(R, dtype=torch.bool, device=dev))
        return plan_step(self.block_table, self.lens_before, new_lens, self.free_blocks, self._count_before,
                         self.page_size, max_tokens, out, self.err)

    def write(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos_sin: torch.Tensor, plan: StepPlan,
              layer: int = 0, positions: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None,
              interleaved: bool = False) -> torch.Tensor:
        """rope_write of the step's tokens (positions default to the plan's), then
        the bounds of the pages that it completed."""
        q = rope_write(q, k, v, plan.positions if positions is None else positions, cos_sin, plan.slots,
                       self.k[layer], self.v[layer], sections, interleaved, None, self.err)
        if self.codes is not None:
            n = plan.slots.numel()
            page_bounds(self.k[layer], self.block_table, self.lens_before, self.seqlens, self.codes[layer],
                        self.scales[layer], n, n, self.err)
        return q

    def token_rows(self, plan: StepPlan) -> TokenRows:
        """The rows that the tokens of the last step's plan attend (causal: a token
        sees its row up to itself). For decode steps and short pieces of prompts:
        a row of the table is copied for each token, and attention reads a
        sequence's pages once for each of its tokens."""
        table = self.block_table.index_select(0, plan.token_seq.clamp(min=0))
        return TokenRows(table, (plan.positions + 1).masked_fill_(plan.token_seq < 0, 0))

    def _rows(self, q, rows):
        return rows if rows is not None else (self.block_table[:q.shape[0]], self.seqlens[:q.shape[0]])

    def attention(self, q: torch.Tensor, layer: int = 0, softmax_scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                  max_seqlen: Optional[int] = None, rows: Optional[TokenRows] = None) -> torch.Tensor:
        """Attention of q [N, Hq, D], the plan's tokens with rows=token_rows(plan);
        without rows q is one query per row, of rows 0 .. N-1 (max_seqlen: see
        paged_attention)."""
        table, lens = self._rows(q, rows)
        return paged_attention(q, self.k[layer], self.v[layer], table, lens, softmax_scale, None, None, out, lse,
                               max_seqlen, self.err)

    def sparse_attention(self, q: torch.Tensor, top_pages: int, layer: int = 0, sink_pages: int = 1,
                         local_pages: int = 1, softmax_scale: Optional[float] = None,
                         rows: Optional[TokenRows] = None):
        """Attention of q over top_pages chosen pages per KV head (q and rows as for
        attention): (out, pages, counts)."""
        if self.codes is None:
            raise RuntimeError("the cache was made without bounds")
        table, lens = self._rows(q, rows)
        return sparse_attention(q, self.k[layer], self.v[layer], self.codes[layer], self.scales[layer], table, lens,
                                top_pages, sink_pages, local_pages, softmax_scale, None, self.err)

    def check_errors(self) -> int:
        """Error bits recorded by the kernels (synchronises)."""
        return int(self.err.item())
