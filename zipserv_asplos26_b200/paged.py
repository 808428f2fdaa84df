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
collects error bits: 2 = an index was out of range and skipped, 4 = a request
was refused by plan_step.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import struct
from typing import NamedTuple, Optional, Sequence

import torch

from ._lib import check, lib

# The argument structs of the C ABI (include/zipserv_b200.h), packed whole: one
# pointer a call is several times cheaper through ctypes than twenty arguments.
_POOL = "Qqqqiiiii4x"
_PLAN = struct.Struct("<QQq12Q6i")
_ROPE = struct.Struct("<QQQQ6qQQqQQQ" + _POOL * 2 + "3i4i3i")
_ATTN = struct.Struct("<QQQqQQQQQQQQ" + _POOL * 2 + "4ifi")
_BOUNDS = struct.Struct("<QQqQQQQQ" + _POOL + "4i")
_SELECT = struct.Struct("<QQQQQqQQQQ12i")
_SIGS = {
    "zs_plan_step": ([C.c_char_p], C.c_int),
    "zs_rope_write": ([C.c_char_p], C.c_int),
    "zs_paged_attention_workspace_bytes": ([C.c_int] * 4, C.c_size_t),
    "zs_paged_attention": ([C.c_char_p], C.c_int),
    "zs_page_bounds": ([C.c_char_p], C.c_int),
    "zs_select_pages": ([C.c_char_p], C.c_int),
}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_I32, _I64 = torch.int32, torch.int64
_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes, f.restype = _SIGS[name]
        _fns[name] = f
    return f


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_nothing = contextlib.nullcontext()


def _on(index):
    """Context in which CUDA device `index` is current (nothing to do when it is already)."""
    return _nothing if index == torch.cuda.current_device() else torch.cuda.device(index)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _cuda(t, name):
    """Device index of a CUDA tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _vector(t, n, dtype, name, index):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or t.numel() != n \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n} elements on cuda:{index}")
    return t.data_ptr()


def _table(t, rows, index):
    """(pointer, row stride, width) of a block table."""
    if isinstance(t, torch.Tensor) and t.dtype is _I32 and t.dim() == 2 and t.get_device() == index:
        n, width = t.shape
        stride, inner = t.stride()
        if n == rows and width > 0 and (inner == 1 or width == 1) and (stride >= width or rows <= 1):
            return t.data_ptr(), (stride if rows > 1 else width), width
    raise ValueError(f"block_table must be int32 [{rows}, width] on cuda:{index} with contiguous rows")


def _page_size(page):
    if not 16 <= page <= 256 or page & (page - 1):
        raise ValueError("page_size must be a power of two from 16 to 256")


def _pool(t, name):
    """The fields of a ZsPagePool."""
    _cuda(t, name)
    dtype = _DTYPES.get(t.dtype)
    if dtype is None or t.dim() != 4:
        raise ValueError(f"{name} must be a bf16 or fp16 tensor [num_blocks, page_size, heads, dim]")
    nb, page, heads, dim = t.shape
    sb, st, sh, sd = t.stride()
    _page_size(page)
    if nb <= 0 or heads <= 0 or dim <= 0:
        raise ValueError(f"{name} must not be empty")
    ptr = t.data_ptr()
    if sd != 1 or (sb | st | sh) % 8 or ptr % 16:
        raise ValueError(f"{name}: rows must be contiguous and 16-byte aligned")
    return ptr, sb, st, sh, nb, page, heads, dim, dtype


def _pools(k_pages, v_pages):
    k, v = _pool(k_pages, "k_pages"), _pool(v_pages, "v_pages")
    if k[4:] != v[4:] or k_pages.get_device() != v_pages.get_device():
        raise ValueError("k_pages and v_pages must agree in shape, type and device")
    return k, v


def _err(err, index):
    return 0 if err is None else _vector(err, 1, _I32, "err", index)


def _query(q, hkv, dim, dtype, index):
    """q as contiguous [B, Hq, D]; a [B, 1, Hq, D] query is one token per sequence."""
    if not isinstance(q, torch.Tensor) or q.get_device() != index or q.dtype is not dtype:
        raise ValueError(f"q must be a {dtype} tensor on cuda:{index}")
    if q.dim() == 4 and q.shape[1] == 1:
        q = q.squeeze(1)
    if q.dim() != 3 or q.shape[2] != dim or q.shape[1] <= 0 or q.shape[1] % hkv:
        raise ValueError(f"q must be [B, Hq, {dim}] or [B, 1, Hq, {dim}] with Hq a multiple of {hkv}")
    if not q.is_contiguous():
        q = q.contiguous()
    return q if q.data_ptr() % 16 == 0 else q.clone()


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
    order, when its tokens fit max_tokens, its pages fit the table's width and
    enough pages are free; otherwise it keeps its state and is marked refused.
    block_table and free_blocks (a stack, its first free_count[0] entries) are
    updated in place; the new lengths and count are returned."""
    index = _cuda(seq_lens, "seq_lens")
    R = seq_lens.numel()
    _need(1 <= R <= 8192, "plan_step takes 1 to 8192 requests")
    table, stride, width = _table(block_table, R, index)
    _need(R * width < 2 ** 31, "block_table is too large")
    _page_size(page_size)
    _need(0 <= max_tokens <= 2 ** 30, "max_tokens must be from 0 to 2**30")
    lens = _vector(seq_lens, R, _I32, "seq_lens", index)
    fresh = _vector(new_lens, R, _I32, "new_lens", index)
    cap = free_blocks.numel()
    _need(cap > 0, "free_blocks must not be empty")
    free = _vector(free_blocks, cap, _I32, "free_blocks", index)
    count = _vector(free_count, 1, _I32, "free_count", index)
    err = _err(err, index)
    with _on(index):
        if out is None:
            e, dev = torch.empty, seq_lens.device
            out = StepPlan(e(R, dtype=_I32, device=dev), e(1, dtype=_I32, device=dev),
                           e(R + 1, dtype=_I32, device=dev), e(max_tokens, dtype=_I64, device=dev),
                           e(max_tokens, dtype=_I32, device=dev), e(max_tokens, dtype=_I32, device=dev),
                           e(R, dtype=torch.bool, device=dev))
        else:
            for t, n, d, name in zip(out, (R, 1, R + 1, max_tokens, max_tokens, max_tokens, R),
                                     (_I32, _I32, _I32, _I64, _I32, _I32, torch.bool), StepPlan._fields):
                _vector(t, n, d, f"out.{name}", index)
            _need(out.seq_lens.data_ptr() != lens and out.free_count.data_ptr() != count,
                  "out.seq_lens and out.free_count must be other buffers than the inputs")
        check(_fn("zs_plan_step")(_PLAN.pack(
            _raw_stream(index), table, stride, lens, fresh, free, count, out.seq_lens.data_ptr(),
            out.free_count.data_ptr(), out.cu_tokens.data_ptr(), out.slots.data_ptr(), out.token_seq.data_ptr(),
            out.positions.data_ptr(), out.refused.data_ptr(), err, R, width, cap, page_size, max_tokens, 0)),
            "zs_plan_step")
    return out


# ----------------------------------------------------------- rotary + write
def _rows(t, n, dim, dtype, name, index):
    """[n, heads, dim] with contiguous, 16-byte aligned rows (copied when they are not):
    (tensor, heads, pointer, token stride, head stride)."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dtype is not dtype or t.dim() != 3 \
            or t.shape[0] != n or t.shape[2] != dim or t.shape[1] <= 0:
        raise ValueError(f"{name} must be a {dtype} tensor [{n}, heads, {dim}] on cuda:{index}")
    st, sh, sd = t.stride()
    ptr = t.data_ptr()
    if sd != 1 or (st | sh) % 8 or ptr % 16:
        t = t.contiguous()
        t = t.clone() if t.data_ptr() % 16 else t
        st, sh, sd = t.stride()
        ptr = t.data_ptr()
    return t, t.shape[1], ptr, st, sh


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
    slices of one projection."""
    kp, vp = _pools(k_pages, v_pages)
    index, dtype, hkv, dim = k_pages.get_device(), k_pages.dtype, kp[6], kp[7]
    _need(isinstance(q, torch.Tensor) and q.dim() == 3, "q must be [N, Hq, D]")
    N = q.shape[0]
    # names keep the copies of unaligned inputs alive over the call
    q, hq, qp, q_tok, q_head = _rows(q, N, dim, dtype, "q", index)
    k, kh, kptr, k_tok, k_head = _rows(k, N, dim, dtype, "k", index)
    v, vh, vptr, v_tok, v_head = _rows(v, N, dim, dtype, "v", index)
    _need(kh == hkv and vh == hkv, "k and v must have the cache's heads")
    _need(cos_sin.dtype is torch.float32 and cos_sin.dim() == 2 and cos_sin.get_device() == index
          and cos_sin.is_contiguous() and cos_sin.shape[0] > 0 and cos_sin.data_ptr() % 16 == 0,
          "cos_sin must be a contiguous, 16-byte aligned float32 [rows, rot] tensor on q's device")
    table_rows, rot = cos_sin.shape
    _need(dim % 16 == 0 and dim <= 512, "head dim must be a multiple of 16 up to 512")
    _need(0 < rot <= dim and rot % 16 == 0, "rot must be a multiple of 16, at most the head dim")
    axes = positions.shape[0] if positions.dim() == 2 else 1
    _need(positions.dtype is _I32 and positions.get_device() == index and positions.dim() in (1, 2)
          and positions.shape[-1] == N and (N <= 1 or positions.stride(-1) == 1) and 1 <= axes <= 4,
          "positions must be int32 [N] or [axes, N] with contiguous rows and 1 to 4 axes")
    if sections is None and axes == 1:
        sections = (rot // 2,)
    _need(sections is not None and len(sections) == axes and min(sections) >= 0 and sum(sections) == rot // 2,
          "sections must give each axis its share of the rot / 2 pairs")
    slot = _vector(slots, N, _I64, "slots", index)
    err = _err(err, index)
    with _on(index):
        if q_out is None:
            q_out = torch.empty((N, hq, dim), dtype=dtype, device=q.device)
        else:
            _need(q_out.shape == (N, hq, dim) and q_out.dtype is dtype and q_out.get_device() == index
                  and q_out.is_contiguous() and q_out.data_ptr() % 16 == 0,
                  "q_out must be contiguous, aligned and of q's shape and type")
        check(_fn("zs_rope_write")(_ROPE.pack(
            _raw_stream(index), qp, kptr, vptr, q_tok, q_head, k_tok, k_head, v_tok, v_head, q_out.data_ptr(),
            positions.data_ptr(), positions.stride(0) if axes > 1 else 0, cos_sin.data_ptr(), slot, err, *kp, *vp,
            N, hq, axes, *sections, *(0,) * (4 - axes), table_rows, rot, int(bool(interleaved)))), "zs_rope_write")
    return q_out


# -------------------------------------------------------------- attention
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, softmax_scale: Optional[float] = None,
                    pages: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, q [B, Hq, D] (or [B, 1, Hq, D]),
    over the first seq_lens[b] tokens of its pages; D is 64 or 128.

    With pages (int32 [B, Hkv, top], distinct logical pages) and counts (int32
    [B, Hkv]) only the listed pages' tokens count. A sequence with nothing to
    attend gets zeros. lse (optional, fp32 [B, Hq]) receives the log of the sum
    of exponentials of the scaled scores."""
    kp, vp = _pools(k_pages, v_pages)
    index, page, hkv, dim = k_pages.get_device(), kp[5], kp[6], kp[7]
    _need(dim == 64 or dim == 128, "head dim must be 64 or 128")
    q3 = _query(q, hkv, dim, k_pages.dtype, index)
    B, hq = q3.shape[0], q3.shape[1]
    table, stride, width = _table(block_table, B, index)
    _need(width * page < 2 ** 31, "block_table covers more than 2**31 - 1 tokens")
    lens = _vector(seq_lens, B, _I32, "seq_lens", index)
    _need((pages is None) == (counts is None), "pages and counts go together")
    top = pages_p = counts_p = 0
    if pages is not None:
        _need(pages.dim() == 3 and pages.shape[2] > 0 and pages.shape[2] * page < 2 ** 31,
              "pages must be int32 [B, Hkv, top]")
        top = pages.shape[2]
        pages_p = _vector(pages, B * hkv * top, _I32, "pages", index)
        counts_p = _vector(counts, B * hkv, _I32, "counts", index)
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(dim)
    _need(math.isfinite(scale), "softmax_scale must be finite")
    lse_p = 0 if lse is None else _vector(lse, B * hq, torch.float32, "lse", index)
    err = _err(err, index)
    with _on(index):
        if out is None:
            out = torch.empty_like(q3)
        else:
            _need(out.numel() == q3.numel() and out.dtype is q3.dtype and out.get_device() == index
                  and out.is_contiguous() and out.data_ptr() % 16 == 0,
                  "out must be contiguous, aligned and of q's shape and type")
        nbytes = _fn("zs_paged_attention_workspace_bytes")(B, hq, hkv, dim)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q3.device)
        check(_fn("zs_paged_attention")(_ATTN.pack(
            _raw_stream(index), q3.data_ptr(), table, stride, lens, pages_p, counts_p, ws.data_ptr(), nbytes,
            out.data_ptr(), lse_p, err, *kp, *vp, B, hq, width, top, scale, 0)), "zs_paged_attention")
    return out if q.dim() == 3 else out.view(q.shape)


# ------------------------------------------------------------------ sparse
def _bounds_buffers(codes, scales, nb, hkv, dim, index):
    cp = _vector(codes, nb * hkv * 2 * dim, torch.int8, "page_codes", index)
    sp = _vector(scales, nb * hkv, torch.float32, "page_scales", index)
    if codes.shape != (nb, hkv, 2, dim) or cp % 16:
        raise ValueError(f"page_codes must be int8 [{nb}, {hkv}, 2, {dim}], 16-byte aligned")
    return cp, sp


def page_bounds(k_pages: torch.Tensor, block_table: torch.Tensor, lens_before: torch.Tensor, seq_lens: torch.Tensor,
                page_codes: torch.Tensor, page_scales: torch.Tensor, max_new: int,
                err: Optional[torch.Tensor] = None) -> None:
    """Bounds of the pages that sequences completed between lens_before and
    seq_lens (at most max_new tokens each), written to page_codes int8
    [num_blocks, Hkv, 2, D] (upper, lower) and page_scales fp32 [num_blocks, Hkv]."""
    kp = _pool(k_pages, "k_pages")
    index, nb, hkv, dim = k_pages.get_device(), kp[4], kp[6], kp[7]
    _need(dim in (64, 128, 256), "head dim must be 64, 128 or 256")
    B = seq_lens.numel()
    table, stride, width = _table(block_table, B, index)
    before = _vector(lens_before, B, _I32, "lens_before", index)
    lens = _vector(seq_lens, B, _I32, "seq_lens", index)
    cp, sp = _bounds_buffers(page_codes, page_scales, nb, hkv, dim, index)
    _need(0 <= max_new < 2 ** 31, "max_new must not be negative")
    err = _err(err, index)
    with _on(index):
        check(_fn("zs_page_bounds")(_BOUNDS.pack(_raw_stream(index), table, stride, before, lens, cp, sp, err, *kp, B,
                                                 width, max_new, 0)), "zs_page_bounds")


def select_pages(q: torch.Tensor, page_codes: torch.Tensor, page_scales: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, page_size: int, top_pages: int, sink_pages: int = 1, local_pages: int = 1,
                 err: Optional[torch.Tensor] = None):
    """Up to top_pages pages per (sequence, KV head): the first sink_pages, the
    last local_pages (the newest, possibly incomplete, among them) and the best
    of the others by the bound of q . k over the page's keys. Returns pages
    (int32 [B, Hkv, top_pages], ascending, -1 past the count) and counts."""
    index = _cuda(page_codes, "page_codes")
    _need(page_codes.dim() == 4 and page_codes.shape[2] == 2, "page_codes must be int8 [num_blocks, Hkv, 2, D]")
    nb, hkv, _, dim = page_codes.shape
    _need(nb > 0 and hkv > 0 and dim in (64, 128, 256), "head dim must be 64, 128 or 256")
    dtype = _DTYPES.get(q.dtype)
    _need(dtype is not None, "q must be bf16 or fp16")
    q3 = _query(q, hkv, dim, q.dtype, index)
    B, hq = q3.shape[0], q3.shape[1]
    _need(hq // hkv <= 128, "at most 128 query heads may share a KV head")
    cp, sp = _bounds_buffers(page_codes, page_scales, nb, hkv, dim, index)
    table, stride, width = _table(block_table, B, index)
    _need(width <= 32768, "at most 32768 pages per sequence")
    lens = _vector(seq_lens, B, _I32, "seq_lens", index)
    _page_size(page_size)
    _need(sink_pages >= 0 and local_pages >= 1 and sink_pages + local_pages <= top_pages < 2 ** 31,
          "top_pages must cover sink_pages (>= 0) and local_pages (>= 1)")
    err = _err(err, index)
    with _on(index):
        pages = torch.empty((B, hkv, top_pages), dtype=_I32, device=q3.device)
        counts = torch.empty((B, hkv), dtype=_I32, device=q3.device)
        check(_fn("zs_select_pages")(_SELECT.pack(
            _raw_stream(index), q3.data_ptr(), cp, sp, table, stride, lens, pages.data_ptr(), counts.data_ptr(), err,
            dtype, B, hq, hkv, dim, nb, width, page_size, top_pages, sink_pages, local_pages, 0)), "zs_select_pages")
    return pages, counts


def sparse_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_codes: torch.Tensor,
                     page_scales: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, top_pages: int,
                     sink_pages: int = 1, local_pages: int = 1, softmax_scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None):
    """select_pages, then paged_attention over the chosen pages. Returns (out, pages, counts)."""
    _need(k_pages.dim() == 4 and page_codes.dim() == 4 and page_codes.shape[0] == k_pages.shape[0]
          and page_codes.shape[1] == k_pages.shape[2] and page_codes.shape[3] == k_pages.shape[3],
          "page_codes must describe the pages of k_pages")
    pages, counts = select_pages(q, page_codes, page_scales, block_table, seq_lens, k_pages.shape[1], top_pages,
                                 sink_pages, local_pages, err)
    out = paged_attention(q, k_pages, v_pages, block_table, seq_lens, softmax_scale, pages, counts, out, None, err)
    return out, pages, counts


# ------------------------------------------------------------------- cache
class PagedKVCache:
    """Buffers of an uncompressed paged cache for up to max_batch sequences of up
    to max_blocks_per_seq pages, and a step's calls on them:

        plan = cache.step(new_lens, max_tokens)      # tokens of each row; -1: ended
        q = cache.write(q, k, v, cos_sin, plan)      # rotary, then into the pages
        o = cache.attention(q_last)                  # one new token per row
        o = cache.sparse_attention(q_last, 64)       # over 64 pages per KV head

    All state (tables, lengths, the free list) is on the GPU in fixed buffers, so
    a step can be captured in a CUDA graph and replayed. layout "heads" keeps
    each head's rows of a page together, "tokens" each token's heads."""

    def __init__(self, num_blocks: int, max_batch: int, max_blocks_per_seq: int, num_kv_heads: int,
                 head_dim: int = 128, page_size: int = 64, dtype: torch.dtype = torch.bfloat16, layout: str = "heads",
                 bounds: bool = True, device="cuda"):
        _need(num_blocks > 0 and max_batch > 0 and max_blocks_per_seq > 0 and num_kv_heads > 0,
              "sizes must be positive")
        _need(layout in ("heads", "tokens"), f"unknown layout {layout!r}")
        _need(dtype in _DTYPES and head_dim in (64, 128), "pages hold bf16 or fp16 heads of dim 64 or 128")
        _page_size(page_size)
        self.device = torch.device(device)
        self.Hkv, self.D, self.page_size, self.max_batch = num_kv_heads, head_dim, page_size, max_batch

        def pool():
            if layout == "heads":
                return torch.zeros(num_blocks, num_kv_heads, page_size, head_dim, dtype=dtype,
                                   device=self.device).transpose(1, 2)
            return torch.zeros(num_blocks, page_size, num_kv_heads, head_dim, dtype=dtype, device=self.device)

        i32 = dict(dtype=_I32, device=self.device)
        self.k, self.v = pool(), pool()
        self.device = self.k.device
        self.block_table = torch.full((max_batch, max_blocks_per_seq), -1, **i32)
        self.seqlens = torch.zeros(max_batch, **i32)
        self.lens_before = torch.zeros(max_batch, **i32)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_blocks, **i32)
        self._count_before = torch.zeros(1, **i32)
        self.err = torch.zeros(1, **i32)
        self.codes = self.scales = None
        if bounds:
            self.codes = torch.zeros(num_blocks, num_kv_heads, 2, head_dim, dtype=torch.int8, device=self.device)
            self.scales = torch.zeros(num_blocks, num_kv_heads, dtype=torch.float32, device=self.device)

    def step(self, new_lens: torch.Tensor, max_tokens: int) -> StepPlan:
        """Admit new_lens (int32 [max_batch]; negative: the row has ended) tokens
        to the rows; max_tokens bounds their sum."""
        self.lens_before.copy_(self.seqlens)
        self._count_before.copy_(self.free_count)
        e, dev, R = torch.empty, self.device, self.max_batch
        out = StepPlan(self.seqlens, self.free_count, e(R + 1, dtype=_I32, device=dev),
                       e(max_tokens, dtype=_I64, device=dev), e(max_tokens, dtype=_I32, device=dev),
                       e(max_tokens, dtype=_I32, device=dev), e(R, dtype=torch.bool, device=dev))
        return plan_step(self.block_table, self.lens_before, new_lens, self.free_blocks, self._count_before,
                         self.page_size, max_tokens, out, self.err)

    def write(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos_sin: torch.Tensor, plan: StepPlan,
              positions: Optional[torch.Tensor] = None, sections: Optional[Sequence[int]] = None,
              interleaved: bool = False) -> torch.Tensor:
        """rope_write of the step's tokens (positions default to the plan's), then
        the bounds of the pages that it completed."""
        q = rope_write(q, k, v, plan.positions if positions is None else positions, cos_sin, plan.slots, self.k,
                       self.v, sections, interleaved, None, self.err)
        if self.codes is not None:
            page_bounds(self.k, self.block_table, self.lens_before, self.seqlens, self.codes, self.scales,
                        plan.slots.numel(), self.err)
        return q

    def attention(self, q: torch.Tensor, softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                  lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [B, Hq, D] over rows 0 .. B-1."""
        B = q.shape[0]
        return paged_attention(q, self.k, self.v, self.block_table[:B], self.seqlens[:B], softmax_scale, None, None,
                               out, lse, self.err)

    def sparse_attention(self, q: torch.Tensor, top_pages: int, sink_pages: int = 1, local_pages: int = 1,
                         softmax_scale: Optional[float] = None):
        """Attention of q [B, Hq, D] over top_pages chosen pages of rows 0 .. B-1: (out, pages, counts)."""
        if self.codes is None:
            raise RuntimeError("the cache was made without bounds")
        B = q.shape[0]
        return sparse_attention(q, self.k, self.v, self.codes, self.scales, self.block_table[:B], self.seqlens[:B],
                                top_pages, sink_pages, local_pages, softmax_scale, None, self.err)

    def check_errors(self) -> int:
        """Error bits recorded by the kernels (synchronises)."""
        return int(self.err.item())
