"""Attention of one new token a stream to some of its cache's blocks: for every
page the least and the greatest of its keys bound any score in it, a query
picks the blocks with the highest bounds, and attention reads those only.

A step: ``rotary_paged_append``, ``update_page_bounds`` for the pages that got
new tokens, ``select_blocks``, ``paged_sparse_attention``.  ``bounds`` bf16
[num_pages, nheads_kv, 2, head_dim] (page_bounds) belongs to one layer's keys.
C ABI: ``sn_update_page_bounds``, ``sn_select_blocks``,
``sn_paged_sparse_attention``.
"""
from __future__ import annotations

import torch

from .. import _lib
from . import paged_kv as PK
from ._common import call, current_handle, fast, on_stream, require_cuda, same_device

_BF16 = torch.bfloat16


def page_bounds(k_pages: torch.Tensor) -> torch.Tensor:
    """Room for the bounds of the pages of k_pages [..., num_pages, nheads_kv, page_size, head_dim]."""
    *lead, n, h, _, hd = k_pages.shape
    return torch.zeros(*lead, n, h, 2, hd, device=k_pages.device, dtype=_BF16)


def _check_bounds(bounds, hkv=None, hd=None, pages=None):
    require_cuda("bounds", bounds, _BF16, 4)
    if not bounds.is_contiguous() or bounds.shape[2] != 2 or min(bounds.shape) < 1 or any(
            want is not None and have != want for have, want in zip((bounds.shape[0], bounds.shape[1], bounds.shape[3]), (pages, hkv, hd))):
        raise ValueError(f"bounds must be contiguous [{pages or 'num_pages'}, {hkv or 'nheads_kv'}, 2, {hd or 'head_dim'}]: got {tuple(bounds.shape)}")


def _check_table(page_table, seq_lens):
    PK._index("page_table", page_table, 2)
    PK._index("seq_lens", seq_lens)
    if page_table.shape[0] != seq_lens.shape[0] or seq_lens.shape[0] > 1 and seq_lens.stride(0) != 1:
        raise ValueError(f"seq_lens must hold {page_table.shape[0]} contiguous lengths")


def _on(stream, launch):
    if stream is None:
        return launch(current_handle(torch.cuda.current_device()))
    with on_stream(stream) as st:
        return launch(st)


def update_page_bounds(k_pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                       cu_seqlens: torch.Tensor | None = None, stream=None) -> None:
    """bounds[page, head] = elementwise least and greatest of the keys that the
    page holds, for every page with some of the newest positions of a stream:
    the last cu_seqlens[b+1] - cu_seqlens[b] of the seq_lens[b] (None: one a
    stream).  k_pages [num_pages, nheads_kv, page_size, head_dim] by its
    strides."""
    if stream is None:
        r = fast().bounds(k_pages, bounds, page_table, seq_lens, cu_seqlens)
        if r is not None:
            return None if r is True else _lib.check("sn_update_page_bounds", r)
    PK._pool("k_pages", k_pages)
    n, hkv, page, hd = k_pages.shape
    _check_bounds(bounds, hkv, hd, n)
    _check_table(page_table, seq_lens)
    batch, width = page_table.shape
    if cu_seqlens is not None:
        require_cuda("cu_seqlens", cu_seqlens, torch.int32, 1)
        if cu_seqlens.shape[0] != batch + 1 or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must hold {batch + 1} contiguous offsets")
    same_device(k_pages=k_pages, bounds=bounds, page_table=page_table, seq_lens=seq_lens, cu_seqlens=cu_seqlens)
    st = [s if e > 1 else max(s, hd) for e, s in zip(k_pages.shape, k_pages.stride())]
    _on(stream, lambda s: call("sn_update_page_bounds", k_pages.data_ptr(), st[0], st[1], st[2], n, page, page_table.data_ptr(),
                               page_table.stride(0) if batch > 1 else width, width, seq_lens.data_ptr(),
                               cu_seqlens.data_ptr() if cu_seqlens is not None else None, batch, hkv, hd,
                               bounds.data_ptr(), s))


def select_blocks(q: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, page_size: int, count: int,
                  first: int = 1, last: int = 1, stream=None) -> torch.Tensor:
    """The blocks of page_size positions that each stream's new token attends
    to, int32 [batch, nheads_kv, count], ascending, -1 behind: its first `first`
    and last `last` blocks, and of the others those with the highest score, the
    lowest among equal ones (all of them where there are no more than `count`).
    A block's score is the greatest over the key/value head's query heads of
    sum_d max(q_d least_d, q_d greatest_d), no less than any q . k in it; one
    with a bound that is not finite is above all, and with a query that is not
    finite all of the head's blocks are alike.
    q [batch, nheads, head_dim] by batch and head strides."""
    if stream is None:
        r = fast().select(q, bounds, page_table, seq_lens, page_size, count, first, last)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_select_blocks", r)
    require_cuda("q", q, _BF16, 3)
    _check_bounds(bounds)
    _check_table(page_table, seq_lens)
    batch, nheads, hd = q.shape
    pages, hkv = bounds.shape[:2]
    if batch != page_table.shape[0] or hd != bounds.shape[3] or nheads < 1 or nheads % hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match {page_table.shape[0]} streams of {hkv} heads of {bounds.shape[3]}")
    if q.stride(2) != 1 and hd > 1:
        raise ValueError("q must be dense along its last dimension")
    page_size, count, first, last = int(page_size), int(count), int(first), int(last)
    if page_size < 1 or count < 1 or first < 0 or last < 0 or first + last > count:
        raise ValueError(f"page_size and count must be positive, and count cover first and last: got {page_size}, {count}, {first}, {last}")
    same_device(q=q, bounds=bounds, page_table=page_table, seq_lens=seq_lens)
    width = page_table.shape[1]

    def launch(st):
        blocks = torch.empty((batch, hkv, count), device=q.device, dtype=torch.int32)
        need = _lib.lib().sn_select_blocks_workspace_size(batch, hkv, width)
        ws = torch.empty(need, device=q.device, dtype=torch.uint8)
        call("sn_select_blocks", q.data_ptr(), q.stride(0), q.stride(1), bounds.data_ptr(), pages, page_size, page_table.data_ptr(),
             page_table.stride(0) if batch > 1 else width, width, seq_lens.data_ptr(), batch, nheads, hkv, hd, count, first, last,
             blocks.data_ptr(), ws.data_ptr(), need, st)
        return blocks

    return _on(stream, launch)


def paged_sparse_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           seq_lens: torch.Tensor, blocks: torch.Tensor, scale: float | None = None,
                           workspace: torch.Tensor | None = None, return_lse: bool = False, stream=None):
    """paged_decode_attention over the positions of listed blocks only: blocks
    int32 [batch, nheads_kv, count] (contiguous; select_blocks), of which the
    first min(count, ceil(seq_lens[b] / page_size)) are read.  Entries below 0 or
    past the stream's end are left out; a block listed twice counts twice.
    `workspace`: decode_workspace."""
    if stream is None:
        r = fast().sparse(q, k_pages, v_pages, page_table, seq_lens, blocks, scale, workspace, return_lse)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_paged_sparse_attention", r)
    if not (isinstance(page_table, torch.Tensor) and page_table.dim() == 2 and isinstance(k_pages, torch.Tensor) and k_pages.dim() == 4):
        PK._pages(k_pages, v_pages, page_table, seq_lens)
    require_cuda("blocks", blocks, torch.int32, 3)
    if blocks.shape[:2] != (page_table.shape[0], k_pages.shape[1]) or blocks.shape[2] < 1 or not blocks.is_contiguous():
        raise ValueError(f"blocks must be contiguous [{page_table.shape[0]}, {k_pages.shape[1]}, count]: got {tuple(blocks.shape)}")
    return PK.attend("sn_paged_sparse_attention", q, k_pages, v_pages, page_table, seq_lens, scale, workspace, return_lse, stream,
                     PK._workspace_size, (blocks.data_ptr(), blocks.shape[2]), {"blocks": blocks})
