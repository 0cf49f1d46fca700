"""A paged KV cache on B200: rotary positions with the append, attention of one
new token a stream, page copies, and the host's book-keeping of the pages.

The pools are bf16 [num_pages, nheads_kv, page_size, head_dim]; a stream's
positions lie in the pages its row of ``page_table`` (int32 [batch,
max_pages], device) names, and ``seq_lens`` (int32 [batch], device) says how
many there are.  Nothing here reads them back to the host, so a captured step
serves growing streams.  C ABI: ``sn_rotary_paged_append``,
``sn_paged_decode_attention``, ``sn_copy_pages``.
"""
from __future__ import annotations

import heapq
import math

import torch

from .. import _lib
from ._common import call, on_stream, require_cuda, same_device

_BF16 = torch.bfloat16


def rotary_table(max_pos: int, rot_dim: int, base: float = 10000.0, factor: float = 1.0, original_max_pos: int | None = None,
                 slow_turns: float = 1.0, fast_turns: float = 32.0, device="cuda"):
    """cos, sin fp32 [max_pos, rot_dim / 2] of the angles pos * base^(-2j / rot_dim), computed in 64 bits.

    For contexts longer than the original ones: with `factor` alone every
    position is divided by it; with `original_max_pos` too, each frequency is
    divided by a factor of its own: those that turn more than `fast_turns`
    times over the original context are kept, those that turn less than
    `slow_turns` times are divided by `factor`, and between the two the
    frequencies are blended linearly in the number of turns."""
    if rot_dim < 2 or rot_dim % 2 or max_pos < 1:
        raise ValueError(f"rot_dim must be even and positive, max_pos positive: got {rot_dim}, {max_pos}")
    if factor < 1.0 or not slow_turns < fast_turns:
        raise ValueError("factor must be at least 1 and slow_turns below fast_turns")
    f64 = torch.float64
    freq = base ** (-torch.arange(0, rot_dim, 2, dtype=f64) / rot_dim)
    if original_max_pos is None:
        freq = freq / factor
    else:
        turns = original_max_pos * freq / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
    ang = torch.arange(max_pos, dtype=f64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


def _pool(name: str, t: torch.Tensor):
    require_cuda(name, t, _BF16, 4)
    if t.stride(3) != 1 or min(t.shape) < 1:
        raise ValueError(f"{name} must be [num_pages, nheads_kv, page_size, head_dim] with a dense last dimension")
    # an axis of extent 1 is never stepped along: its stride may be anything
    return [st if n > 1 else max(st, t.shape[3]) for n, st in zip(t.shape[:3], t.stride()[:3])]


def _index(name: str, t: torch.Tensor, dim: int = 1):
    require_cuda(name, t, torch.int32, dim)
    if t.numel() == 0 or t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be a non-empty int32 tensor with a dense last dimension")


def _pages(k_pages, v_pages, page_table, seq_lens):
    """Checked pools and tables: the arguments both kernels take in the same order."""
    ks, vs = _pool("k_pages", k_pages), _pool("v_pages", v_pages)
    if k_pages.shape != v_pages.shape:
        raise ValueError(f"k_pages and v_pages differ in shape: {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    _index("page_table", page_table, 2)
    _index("seq_lens", seq_lens)
    if page_table.shape[0] != seq_lens.shape[0]:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {seq_lens.shape[0]} streams")
    stride = page_table.stride(0) if page_table.shape[0] > 1 else page_table.shape[1]
    return (k_pages.data_ptr(), *ks, v_pages.data_ptr(), *vs, k_pages.shape[0], k_pages.shape[2], page_table.data_ptr(),
            stride, page_table.shape[1], seq_lens.data_ptr())


def rotary_paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                        seq_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nheads: int,
                        cu_seqlens: torch.Tensor | None = None, interleaved: bool = False, stream=None) -> torch.Tensor:
    """qkv [tokens, (nheads + 2 nheads_kv) head_dim] of the new tokens (row
    stride taken from the tensor): stream b's are rows cu_seqlens[b] ..
    cu_seqlens[b+1]-1 (None: one token a stream) and end at position
    seq_lens[b] - 1 (seq_lens counts them).  The first 2 * cos.shape[1]
    elements of each q and k head are rotated by the position's row of cos /
    sin fp32 [max_pos, rot / 2]: halves (j, j + rot/2), or neighbours (2j, 2j
    + 1) when interleaved.  k and v go to their pages; returns q [tokens,
    nheads, head_dim]."""
    require_cuda("qkv", qkv, _BF16, 2)
    args = _pages(k_pages, v_pages, page_table, seq_lens)
    tokens, (_, hkv, _, hd), batch = qkv.shape[0], k_pages.shape, seq_lens.shape[0]
    if qkv.shape[1] != (nheads + 2 * hkv) * hd or tokens > 0 and qkv.stride(1) != 1:
        raise ValueError(f"qkv must be [tokens, {(nheads + 2 * hkv) * hd}] with a dense last dimension")
    if cu_seqlens is None:
        if tokens != batch:
            raise ValueError(f"{tokens} tokens for {batch} streams: give cu_seqlens")
    else:
        _index("cu_seqlens", cu_seqlens)
        if cu_seqlens.shape[0] != batch + 1:
            raise ValueError(f"cu_seqlens must hold {batch + 1} offsets")
    for name, t in (("cos", cos), ("sin", sin)):
        require_cuda(name, t, torch.float32, 2)
        if not t.is_contiguous() or t.shape != cos.shape or t.shape[0] < 1 or 2 * t.shape[1] > hd:
            raise ValueError(f"{name} must be contiguous fp32 [max_pos, rot / 2], rot at most {hd}, both alike")
    same_device(qkv=qkv, k_pages=k_pages, v_pages=v_pages, page_table=page_table, seq_lens=seq_lens, cos=cos, sin=sin,
                cu_seqlens=cu_seqlens)
    with on_stream(stream) as st:
        q = torch.empty(tokens, nheads, hd, device=qkv.device, dtype=_BF16)
        if tokens:
            call("sn_rotary_paged_append", qkv.data_ptr(), qkv.stride(0) if tokens > 1 else qkv.shape[1], q.data_ptr(),
                 *args, cu_seqlens.data_ptr() if cu_seqlens is not None else None, cos.data_ptr(), sin.data_ptr(),
                 cos.shape[0], tokens, batch, nheads, hkv, hd, 2 * cos.shape[1], int(bool(interleaved)), st)
    return q


def decode_workspace(batch: int, nheads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """The workspace of paged_decode_attention for up to `batch` streams: zeroed
    once, kept for every step on one stream of calls."""
    n = _lib.lib().sn_paged_decode_workspace_size(batch, nheads, head_dim)
    if n == 0:
        raise ValueError("batch, nheads and head_dim must be positive")
    return torch.zeros(n, device=device, dtype=torch.uint8)


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           seq_lens: torch.Tensor, scale: float | None = None, workspace: torch.Tensor | None = None,
                           return_lse: bool = False, stream=None):
    """One new token a stream: q [batch, nheads, head_dim] (batch and head
    strides taken from the tensor) over positions t < seq_lens[b] of the
    stream's pages; scale defaults to head_dim^-0.5.  Returns [batch, nheads,
    head_dim], zeros for an empty stream, and with return_lse also the log of
    the sum of exponentials fp32 [batch, nheads].  `workspace`
    (decode_workspace) saves an allocation and a fill a call; calls that share
    one must not overlap."""
    require_cuda("q", q, _BF16, 3)
    args = _pages(k_pages, v_pages, page_table, seq_lens)
    batch, nheads, hd = q.shape
    hkv = k_pages.shape[1]
    if batch != seq_lens.shape[0] or hd != k_pages.shape[3] or nheads < 1 or nheads % hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match {seq_lens.shape[0]} streams of {hkv} heads of {k_pages.shape[3]}")
    if q.stride(2) != 1 and hd > 1:
        raise ValueError("q must be dense along its last dimension")
    need = _lib.lib().sn_paged_decode_workspace_size(batch, nheads, hd)
    if workspace is not None:
        require_cuda("workspace", workspace, torch.uint8, 1)
        if workspace.numel() < need or not workspace.is_contiguous() or workspace.data_ptr() % 16:
            raise ValueError(f"workspace must hold {need} contiguous, 16-byte aligned bytes (decode_workspace)")
    same_device(q=q, k_pages=k_pages, v_pages=v_pages, page_table=page_table, seq_lens=seq_lens, workspace=workspace)
    with on_stream(stream) as st:
        out = torch.empty(batch, nheads, hd, device=q.device, dtype=_BF16)
        lse = torch.empty(batch, nheads, device=q.device, dtype=torch.float32) if return_lse else None
        ws = workspace
        if ws is None:  # only the arrival counters at its start have to be zero
            ws = torch.empty(need, device=q.device, dtype=torch.uint8)
            ws[:4 * batch * nheads].zero_()
        call("sn_paged_decode_attention", q.data_ptr(), q.stride(0), q.stride(1), *args, out.data_ptr(),
             lse.data_ptr() if return_lse else None, float(hd ** -0.5 if scale is None else scale), batch, nheads, hkv,
             hd, ws.data_ptr(), ws.numel(), st)
    return (out, lse) if return_lse else out


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """pool [..., num_pages, nheads_kv, page_size, head_dim] (contiguous, any
    type): page dst[i] = page src[i] under every leading index; src, dst int32
    [pairs] on the device.  No page may be both copied from and copied to in
    one call, nor copied to twice."""
    require_cuda("pool", pool)
    if pool.dim() < 4 or not pool.is_contiguous() or pool.numel() == 0:
        raise ValueError("pool must be a contiguous, non-empty [..., num_pages, nheads_kv, page_size, head_dim] tensor")
    for name, t in (("src", src), ("dst", dst)):
        require_cuda(name, t, torch.int32, 1)
        if not t.is_contiguous() or t.shape != src.shape:
            raise ValueError("src and dst must be contiguous int32 tensors of one length")
    same_device(pool=pool, src=src, dst=dst)
    n = pool.shape[-4]
    nbytes = pool.shape[-1] * pool.shape[-2] * pool.shape[-3] * pool.element_size()
    with on_stream(stream) as st:
        call("sn_copy_pages", pool.data_ptr(), n * nbytes, nbytes, nbytes, pool.numel() * pool.element_size() // (n * nbytes),
             n, src.data_ptr(), dst.data_ptr(), src.shape[0], st)
