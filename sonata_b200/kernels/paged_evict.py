"""Streams of bounded length in the paged KV cache: attention that adds up what
weight each cached position has had, and the eviction of the positions that
have had the least.

``mass`` fp32 [batch, nheads_kv, >= max_pages * page_size] holds the weights of
one layer's positions, in the order of their places in the cache; it starts
as zeros and the two operators keep it in step with the pages.
PagedKVCache.evict does what an eviction means for the pages; after one, new
tokens need ``rotary_paged_append(..., positions=)``.  C ABI:
``sn_paged_decode_attention_mass``, ``sn_evict_positions``.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from . import paged_kv as PK
from ._common import call, current_handle, fast, on_stream, require_cuda, same_device

EVICT_MOST = 1 << 19  # max_pages * page_size that evict_positions takes


@functools.lru_cache(maxsize=256)
def _mass_size(batch: int, nheads: int, nheads_kv: int, head_dim: int, max_positions: int) -> int:
    return _lib.lib().sn_paged_mass_workspace_size(batch, nheads, nheads_kv, head_dim, max_positions)


def mass_workspace(batch: int, nheads: int, nheads_kv: int, head_dim: int, max_positions: int, device="cuda") -> torch.Tensor:
    """The workspace of paged_decode_attention_mass for up to `batch` streams
    whose page tables reach max_positions (max_pages * page_size): zeroed once,
    kept for every step on one stream of calls.  Four bytes a query head and
    position that the tables reach, whatever the streams' lengths."""
    n = _mass_size(batch, nheads, nheads_kv, head_dim, max_positions)
    if n == 0:
        raise ValueError("every size must be positive, and nheads a multiple of nheads_kv")
    return torch.zeros(n, device=device, dtype=torch.uint8)


def _check_mass(mass, shape, room: int):
    require_cuda("mass", mass, torch.float32, len(shape) + 1)
    if tuple(mass.shape[:-1]) != tuple(shape) or mass.shape[-1] < room or mass.stride(-1) != 1 or min(mass.stride()) < 0 or any(
            st < room for st, e in zip(mass.stride()[:-1], mass.shape) if e > 1):
        raise ValueError(f"mass must be {[*shape, room]} or longer, dense along its last dimension, without overlaps: got "
                         f"{tuple(mass.shape)}, strides {mass.stride()}")


def paged_decode_attention_mass(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                                seq_lens: torch.Tensor, mass: torch.Tensor, scale: float | None = None,
                                workspace: torch.Tensor | None = None, return_lse: bool = False, stream=None):
    """paged_decode_attention, and mass[b, hk, t] += the weight that position t
    has in the query heads of key/value head hk, added up over them.  mass fp32
    [batch, nheads_kv, at least max_pages * page_size] (batch and head strides
    taken from the tensor); places past a stream's end are not touched.
    `workspace`: mass_workspace."""
    if stream is None:
        r = fast().mass(q, k_pages, v_pages, page_table, seq_lens, mass, scale, workspace, return_lse)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_paged_decode_attention_mass", r)
    if not (isinstance(page_table, torch.Tensor) and page_table.dim() == 2 and isinstance(k_pages, torch.Tensor) and k_pages.dim() == 4):
        PK._pages(k_pages, v_pages, page_table, seq_lens)
    (batch, width), (_, hkv, page, _) = page_table.shape, k_pages.shape
    _check_mass(mass, (batch, hkv), width * page)
    return PK.attend("sn_paged_decode_attention_mass", q, k_pages, v_pages, page_table, seq_lens, scale, workspace, return_lse,
                     stream, lambda b, h, hd: _mass_size(b, h, hkv, hd, width * page),
                     (mass.data_ptr(), mass.stride(0), mass.stride(1)), {"mass": mass})


def evict_positions(pool: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, mass: torch.Tensor, keep: int,
                    recent: int = 0, sinks: int = 0, return_source: bool = False, stream=None):
    """Cuts every stream with more than `keep` positions down to `keep`, in every
    layer and key/value head by itself: the first `sinks` and the last `recent`
    stay, and of the others those of the highest mass (the lowest positions
    among equal ones).  pool bf16 [n_layers, 2, num_pages, nheads_kv, page_size,
    head_dim] (contiguous: PagedKVCache.pool), mass fp32 [n_layers, batch,
    nheads_kv, at least max_pages * page_size] (strides taken from the tensor).

    What is kept ends in the places 0 .. keep - 1: it stays where it is below
    keep - recent, later ones fill the places between in order, and the recent
    ones follow in order; mass goes with it and is zero behind.  Streams with no
    more than `keep` positions are left alone.  seq_lens is not changed: the
    caller sets it to min(n, keep) (PagedKVCache.evict does).  A page that two
    streams share must not be cut in either; max_pages * page_size is EVICT_MOST
    at most.  With return_source: int32 [n_layers, batch, nheads_kv, keep], where
    each place's position was (-1 past the end of a stream that was left alone)."""
    if stream is None:
        r = fast().evict(pool, page_table, seq_lens, mass, keep, recent, sinks, return_source)
        if r is not None:
            return _lib.check("sn_evict_positions", r) if type(r) is int else None if r is True else r
    require_cuda("pool", pool, torch.bfloat16, 6)
    if not pool.is_contiguous() or min(pool.shape) < 1 or pool.shape[1] != 2:
        raise ValueError("pool must be a contiguous, non-empty [n_layers, 2, num_pages, nheads_kv, page_size, head_dim] tensor")
    PK._index("page_table", page_table, 2)
    PK._index("seq_lens", seq_lens)
    batch, width = page_table.shape
    layers, _, pages, hkv, page, hd = pool.shape
    if seq_lens.shape[0] != batch or seq_lens.stride(0) != 1 and batch > 1:
        raise ValueError(f"seq_lens must hold {batch} contiguous lengths")
    _check_mass(mass, (layers, batch, hkv), width * page)
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError(f"keep must be positive and cover recent and sinks, which must not be negative: got {keep}, {recent}, {sinks}")
    same_device(pool=pool, page_table=page_table, seq_lens=seq_lens, mass=mass)

    def launch(st):
        source = torch.empty((layers, batch, hkv, keep), device=pool.device, dtype=torch.int32) if return_source else None
        need = _lib.lib().sn_evict_workspace_size(layers, batch, hkv, width * page, keep)
        ws = torch.empty(need, device=pool.device, dtype=torch.uint8)
        call("sn_evict_positions", pool.data_ptr(), layers, pages, page, hkv, hd, page_table.data_ptr(),
             page_table.stride(0) if batch > 1 else width, width, seq_lens.data_ptr(), mass.data_ptr(), mass.stride(0), mass.stride(1),
             mass.stride(2), batch, keep, recent, sinks, source.data_ptr() if return_source else None,
             ws.data_ptr(), need, st)
        return source

    if stream is None:
        return launch(current_handle(torch.cuda.current_device()))
    with on_stream(stream) as st:
        return launch(st)
