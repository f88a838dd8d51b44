"""A step's place in the paged KV cache, worked out on the GPU (q36_page_plan): from the requests' cached and
new token counts, the row starts, key counts, positions and cache slots that attn_fused's entries take
(attn_proj, attn_front, attn_chunk, attn_decode), with the block tables extended from a list of free pages.
The reference reads these from its serving engine (R = qwen36_nodes_kb34: R/qwen36_layer/attn_fused.py:70-75).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from .._lib import check, check_tensors, pack_plan, ptr

# bits of PagePlan.used[1]: what did not fit
TOKENS, PAGES, TABLE, PAGE_TABLE = 1, 2, 4, 8


@dataclass
class PagePlan:
    """What plan_pages writes for B requests with up to T new tokens."""
    qsl: torch.Tensor        # int32 [B + 1]: first row of each request among the new tokens
    seqlens: torch.Tensor    # int32 [B]: keys of each request, the new tokens included
    positions: torch.Tensor  # int32 [T]: the new tokens' positions (0 behind the last request)
    out_loc: torch.Tensor    # int64 [T]: their cache slots (-1: none)
    used: torch.Tensor       # int32 [2]: pages taken from the free list; 0, or what did not fit (the bits above)

    @staticmethod
    def alloc(B: int, T: int, device) -> "PagePlan":
        i32 = dict(dtype=torch.int32, device=device)
        return PagePlan(torch.empty(B + 1, **i32), torch.empty(B, **i32), torch.empty(T, **i32),
                        torch.empty(T, dtype=torch.int64, device=device), torch.empty(2, **i32))


def _refuse(name: str, shape, dtype="int32"):
    raise ValueError(f"plan_pages: {name} must be a contiguous {dtype} tensor {list(shape)}")


def plan_pages(cached, new, table, free, T: int, page_size: int = 1, req=None, page_table=None, whole: bool = True,
               plan: PagePlan | None = None, stream=None) -> PagePlan:
    """Places the new tokens of B requests: cached, new int32 [B] (keys in the cache, tokens to come); table int32
    [rows, width], the pages of request row req[b] (int32 [B], distinct rows; None: row b), extended in place by
    free (int32), taken from the front in the order of the requests; T: rows of the step (new.sum(), or more for a
    padded batch).  page_table int32 [B, stride] (optional) receives the slot of each request's keys, as attn_decode
    reads them: all keys (whole) or the new tokens' alone; the rest of it is left as it was.  A page number outside
    the cache is the caller's to avoid; what does not fit is told in plan.used[1] and gets no slot."""
    i32 = torch.int32
    if cached.dim() != 1:
        raise ValueError("plan_pages: cached must be [B]")
    B = cached.shape[0]
    if table.dim() != 2 or free.dim() != 1:
        raise ValueError("plan_pages: table must be [rows, width] and free [pages]")
    for name, t in (("cached", cached), ("new", new), ("req", req)):
        if t is not None and (t.dtype is not i32 or t.shape != (B,) or not t.is_contiguous()):
            _refuse(name, (B,))
    rows, width = table.shape
    if table.dtype is not i32 or not table.is_contiguous():
        _refuse("table", (rows, width))
    if free.dtype is not i32 or not free.is_contiguous():
        _refuse("free", free.shape)
    pt_width = 0
    if page_table is not None:
        pt_width = page_table.shape[-1]
        if page_table.dtype is not i32 or page_table.shape != (B, pt_width) or not page_table.is_contiguous():
            _refuse("page_table", (B, pt_width))
    if plan is None:
        plan = PagePlan.alloc(B, T, cached.device)
    else:
        for name, t, n in (("plan.qsl", plan.qsl, B + 1), ("plan.seqlens", plan.seqlens, B),
                           ("plan.positions", plan.positions, T), ("plan.used", plan.used, 2)):
            if t.dtype is not i32 or t.shape != (n,) or not t.is_contiguous():
                _refuse(name, (n,))
        if plan.out_loc.dtype is not torch.int64 or plan.out_loc.shape != (T,) or not plan.out_loc.is_contiguous():
            _refuse("plan.out_loc", (T,), "int64")
    check_tensors("plan_pages", "cached new table free req page_table plan.qsl plan.seqlens plan.positions plan.out_loc plan.used",
                  cached, new, table, free, req, page_table, plan.qsl, plan.seqlens, plan.positions, plan.out_loc, plan.used)
    a = pack_plan(B, T, page_size, rows, width, free.shape[0], pt_width, 1 if whole else 0, cached.data_ptr(), new.data_ptr(),
                  ptr(req), table.data_ptr(), free.data_ptr(), plan.qsl.data_ptr(), plan.seqlens.data_ptr(),
                  plan.positions.data_ptr(), plan.out_loc.data_ptr(), plan.used.data_ptr(), ptr(page_table))
    check(_lib.packed().q36_page_plan(a, _lib.stream_handle(stream)), "q36_page_plan")
    return plan
