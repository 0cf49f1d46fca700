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

import functools
import heapq
import math

import torch

from .. import _lib
from ._common import call, current_handle, fast, on_stream, require_cuda, same_device

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


# A decode step's calls are short, so the checks are two-tiered: one expression that holds for every valid call, and the
# functions that say what is wrong with the others.

def _pool(name: str, t: torch.Tensor):
    require_cuda(name, t, _BF16, 4)
    if t.stride(3) != 1 or min(t.shape) < 1:
        raise ValueError(f"{name} must be [num_pages, nheads_kv, page_size, head_dim] with a dense last dimension")


def _index(name: str, t: torch.Tensor, dim: int = 1):
    require_cuda(name, t, torch.int32, dim)
    if t.numel() == 0 or t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must be a non-empty int32 tensor with a dense last dimension")


def _check_pages(k_pages, v_pages, page_table, seq_lens):
    _pool("k_pages", k_pages)
    _pool("v_pages", v_pages)
    if k_pages.shape != v_pages.shape:
        raise ValueError(f"k_pages and v_pages differ in shape: {tuple(k_pages.shape)}, {tuple(v_pages.shape)}")
    _index("page_table", page_table, 2)
    _index("seq_lens", seq_lens)
    if page_table.shape[0] != seq_lens.shape[0]:
        raise ValueError(f"page_table has {page_table.shape[0]} rows for {seq_lens.shape[0]} streams")


def _pages(k_pages, v_pages, page_table, seq_lens):
    """Checked pools and tables: the arguments both kernels take in the same order."""
    if not (isinstance(k_pages, torch.Tensor) and isinstance(v_pages, torch.Tensor) and
            isinstance(page_table, torch.Tensor) and isinstance(seq_lens, torch.Tensor)):
        _check_pages(k_pages, v_pages, page_table, seq_lens)
    ks, kt, vt, ts, tt = k_pages.shape, k_pages.stride(), v_pages.stride(), page_table.shape, page_table.stride()
    if not (len(ks) == 4 and ks == v_pages.shape and kt[3] == 1 == vt[3] and k_pages.dtype is _BF16 is v_pages.dtype and
            k_pages.is_cuda and v_pages.is_cuda and 0 not in ks and len(ts) == 2 and 0 not in ts and tt[1] == 1 and
            seq_lens.shape == ts[:1] and seq_lens.stride() == (1,) and page_table.dtype is torch.int32 is seq_lens.dtype
            and page_table.is_cuda and seq_lens.is_cuda):
        _check_pages(k_pages, v_pages, page_table, seq_lens)
    n, h, page, hd = ks
    if n == 1 or h == 1 or page == 1:  # an axis of extent 1 is never stepped along: its stride may be anything
        kt, vt = ([st if e > 1 else max(st, hd) for e, st in zip(ks, t)] for t in (kt, vt))
    return (k_pages.data_ptr(), kt[0], kt[1], kt[2], v_pages.data_ptr(), vt[0], vt[1], vt[2], n, page, page_table.data_ptr(),
            tt[0] if ts[0] > 1 else ts[1], ts[1], seq_lens.data_ptr())


def rotary_paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                        seq_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nheads: int,
                        cu_seqlens: torch.Tensor | None = None, interleaved: bool = False, stream=None,
                        positions: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [tokens, (nheads + 2 nheads_kv) head_dim] of the new tokens (row
    stride taken from the tensor): stream b's are rows cu_seqlens[b] ..
    cu_seqlens[b+1]-1 (None: one token a stream) and end at position
    seq_lens[b] - 1 (seq_lens counts them).  The first 2 * cos.shape[1]
    elements of each q and k head are rotated by the position's row of cos /
    sin fp32 [max_pos, rot / 2]: halves (j, j + rot/2), or neighbours (2j, 2j
    + 1) when interleaved.  k and v go to their pages; returns q [tokens,
    nheads, head_dim], zeros for a row of no stream or a position out of range.
    `positions` int32 [tokens] names the tokens' rows of cos / sin where their
    places in the cache are not their positions (after evict_positions)."""
    if stream is None:
        args = (qkv, k_pages, v_pages, page_table, seq_lens, cos, sin, nheads, cu_seqlens, interleaved)
        r = fast().append(*args) if positions is None else fast().append(*args, positions)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_rotary_paged_append", r)
    if not (isinstance(qkv, torch.Tensor) and qkv.dtype is _BF16 and qkv.is_cuda and qkv.dim() == 2):
        require_cuda("qkv", qkv, _BF16, 2)
    args = _pages(k_pages, v_pages, page_table, seq_lens)
    (tokens, width), (_, hkv, _, hd), batch = qkv.shape, k_pages.shape, seq_lens.shape[0]
    if width != (nheads + 2 * hkv) * hd or tokens > 0 and qkv.stride(1) != 1:
        raise ValueError(f"qkv must be [tokens, {(nheads + 2 * hkv) * hd}] with a dense last dimension")
    if cu_seqlens is None:
        if tokens != batch:
            raise ValueError(f"{tokens} tokens for {batch} streams: give cu_seqlens")
    elif not (isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda and cu_seqlens.dtype is torch.int32 and
              cu_seqlens.shape == (batch + 1,) and cu_seqlens.is_contiguous()):
        _index("cu_seqlens", cu_seqlens)
        raise ValueError(f"cu_seqlens must hold {batch + 1} contiguous offsets")
    if not (isinstance(cos, torch.Tensor) and isinstance(sin, torch.Tensor) and cos.dtype is torch.float32 is sin.dtype and
            cos.is_cuda and sin.is_cuda and cos.dim() == 2 and cos.shape == sin.shape and cos.is_contiguous() and
            sin.is_contiguous() and cos.shape[0] > 0 and 2 * cos.shape[1] <= hd):
        for name, t in (("cos", cos), ("sin", sin)):
            require_cuda(name, t, torch.float32, 2)
        raise ValueError(f"cos and sin must be contiguous fp32 [max_pos, rot / 2], rot at most {hd}, both alike")
    if positions is not None and not (isinstance(positions, torch.Tensor) and positions.is_cuda and positions.dtype is torch.int32
                                      and positions.shape == (tokens,) and positions.is_contiguous()):
        require_cuda("positions", positions, torch.int32, 1)
        raise ValueError(f"positions must hold {tokens} contiguous numbers")
    max_pos, half = cos.shape
    dev = torch.cuda.current_device()
    if not (dev == qkv.get_device() == k_pages.get_device() == v_pages.get_device() == page_table.get_device() ==
            seq_lens.get_device() == cos.get_device() == sin.get_device() == (cos if cu_seqlens is None else cu_seqlens).get_device()
            == (cos if positions is None else positions).get_device()):
        same_device(qkv=qkv, k_pages=k_pages, v_pages=v_pages, page_table=page_table, seq_lens=seq_lens, cos=cos, sin=sin,
                    cu_seqlens=cu_seqlens, positions=positions)
    at = () if positions is None else (positions.data_ptr(),)

    def launch(st):
        q = qkv.new_empty((tokens, nheads, hd))
        if tokens:
            call("sn_rotary_paged_append_at" if at else "sn_rotary_paged_append", qkv.data_ptr(),
                 qkv.stride(0) if tokens > 1 else width, q.data_ptr(), *args,
                 cu_seqlens.data_ptr() if cu_seqlens is not None else None, *at, cos.data_ptr(), sin.data_ptr(),
                 max_pos, tokens, batch, nheads, hkv, hd, 2 * half, 1 if interleaved else 0, st)
        return q

    if stream is None:
        return launch(current_handle(dev))
    with on_stream(stream) as st:
        return launch(st)


@functools.lru_cache(maxsize=256)
def _workspace_size(batch: int, nheads: int, head_dim: int) -> int:
    return _lib.lib().sn_paged_decode_workspace_size(batch, nheads, head_dim)


def decode_workspace(batch: int, nheads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """The workspace of paged_decode_attention for up to `batch` streams: zeroed
    once, kept for every step on one stream of calls."""
    n = _workspace_size(batch, nheads, head_dim)
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
    if stream is None:
        r = fast().attend(q, k_pages, v_pages, page_table, seq_lens, scale, workspace, return_lse)
        if r is not None:
            return r if type(r) is not int else _lib.check("sn_paged_decode_attention", r)
    return attend("sn_paged_decode_attention", q, k_pages, v_pages, page_table, seq_lens, scale, workspace, return_lse, stream,
                  _workspace_size)


def attend(fn: str, q, k_pages, v_pages, page_table, seq_lens, scale, workspace, return_lse, stream, size, extra=(),
           others=None):
    """The C entry `fn`, a form of the attention of one token a stream: `extra`
    are its arguments after seq_lens, `others` more tensors (by name) that have
    to be on the current device, `size` gives the bytes of its workspace."""
    if not (isinstance(q, torch.Tensor) and q.dtype is _BF16 and q.is_cuda and q.dim() == 3):
        require_cuda("q", q, _BF16, 3)
    args = _pages(k_pages, v_pages, page_table, seq_lens)
    (batch, nheads, hd), (qb, qh, qc) = q.shape, q.stride()
    hkv = k_pages.shape[1]
    if batch != seq_lens.shape[0] or hd != k_pages.shape[3] or nheads < 1 or nheads % hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match {seq_lens.shape[0]} streams of {hkv} heads of {k_pages.shape[3]}")
    if qc != 1 and hd > 1:
        raise ValueError("q must be dense along its last dimension")
    need = size(batch, nheads, hd)
    dev = torch.cuda.current_device()
    if not (dev == q.get_device() == k_pages.get_device() == v_pages.get_device() == page_table.get_device() ==
            seq_lens.get_device()) or others:
        same_device(q=q, k_pages=k_pages, v_pages=v_pages, page_table=page_table, seq_lens=seq_lens, **(others or {}))
    if workspace is not None and not (
            isinstance(workspace, torch.Tensor) and workspace.dtype is torch.uint8 and workspace.get_device() == dev and
            workspace.dim() == 1 and workspace.numel() >= need and workspace.is_contiguous()
            and workspace.data_ptr() % 16 == 0):
        require_cuda("workspace", workspace, torch.uint8, 1)
        same_device(workspace=workspace)
        raise ValueError(f"workspace must hold {need} contiguous, 16-byte aligned bytes (decode_workspace, mass_workspace)")

    def launch(st):
        out = q.new_empty((batch, nheads, hd))
        lse = torch.empty((batch, nheads), device=q.device, dtype=torch.float32) if return_lse else None
        ws = workspace
        if ws is None:  # only the arrival counters at its start have to be zero
            ws = torch.empty(need, device=q.device, dtype=torch.uint8)
            ws[:4 * _lib.SN_PAGED_DECODE_COUNTERS].zero_()
        call(fn, q.data_ptr(), qb, qh, *args, *extra, out.data_ptr(),
             lse.data_ptr() if return_lse else None, hd ** -0.5 if scale is None else float(scale), batch, nheads, hkv,
             hd, ws.data_ptr(), need, st)
        return (out, lse) if return_lse else out

    if stream is None:
        return launch(current_handle(dev))
    with on_stream(stream) as st:
        return launch(st)


def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, stream=None) -> None:
    """pool [..., num_pages, nheads_kv, page_size, head_dim] (contiguous, any
    type): page dst[i] = page src[i] under every leading index; src, dst int32
    [pairs] on the device.  No page may be both copied from and copied to in
    one call, nor copied to twice."""
    if stream is None:
        r = fast().copy(pool, src, dst)
        if r is not None:
            return None if r is True else _lib.check("sn_copy_pages", r)
    if not (isinstance(pool, torch.Tensor) and pool.is_cuda and pool.dim() >= 4 and pool.is_contiguous() and pool.numel()):
        require_cuda("pool", pool)
        raise ValueError("pool must be a contiguous, non-empty [..., num_pages, nheads_kv, page_size, head_dim] tensor")
    if not (isinstance(src, torch.Tensor) and isinstance(dst, torch.Tensor) and src.dtype is torch.int32 is dst.dtype and
            src.dim() == 1 and src.shape == dst.shape and src.is_contiguous() and dst.is_contiguous()):
        for name, t in (("src", src), ("dst", dst)):
            require_cuda(name, t, torch.int32, 1)
        raise ValueError("src and dst must be contiguous int32 tensors of one length")
    dev = torch.cuda.current_device()
    if not dev == pool.get_device() == src.get_device() == dst.get_device():
        for name, t in (("src", src), ("dst", dst)):
            require_cuda(name, t)
        same_device(pool=pool, src=src, dst=dst)
    n, heads, page, hd = pool.shape[-4:]
    size = pool.element_size()
    nbytes = heads * page * hd * size
    args = (pool.data_ptr(), n * nbytes, nbytes, nbytes, pool.numel() * size // (n * nbytes), n, src.data_ptr(), dst.data_ptr(),
            src.shape[0])
    if stream is None:
        call("sn_copy_pages", *args, current_handle(dev))
    else:
        with on_stream(stream) as st:
            call("sn_copy_pages", *args, st)


class OutOfPages(RuntimeError):
    """A PagedKVCache has too few free pages for what was asked; nothing was changed."""


class PagedKVCache:
    """The pages of all layers' keys and values, and the host's book-keeping of
    who owns them: `slots` streams, each a list of pages and a length.

    pool bf16 [n_layers, 2, num_pages, nheads_kv, page_size, head_dim]: a page
    number means the same page in every layer, so one table serves all of them
    and one copy_pages call moves a page everywhere.  `page_table` int32
    [slots, max_pages] and `seq_lens` int32 [slots] are device tensors that
    reserve / fork / free / compact update in place, so a captured decode step
    goes on using them.  Full pages may be shared between forked streams (only
    evict writes to them, in copies of its own); a stream's last, partly filled
    page never is.

    track_mass and track_bounds add what paged_evict and paged_sparse keep
    beside the pages, which then follows them: `mass` fp32 [n_layers, slots,
    nheads_kv, max_pages * page_size], `bounds` bf16 [n_layers, num_pages,
    nheads_kv, 2, head_dim]."""

    def __init__(self, n_layers: int, num_pages: int, nheads_kv: int, head_dim: int, slots: int, max_pages: int,
                 page_size: int = 16, device="cuda"):
        if min(n_layers, num_pages, nheads_kv, head_dim, slots, max_pages, page_size) < 1:
            raise ValueError("every size must be positive")
        self.pool = torch.zeros(n_layers, 2, num_pages, nheads_kv, page_size, head_dim, device=device, dtype=_BF16)
        self.page_size, self.num_pages, self.max_pages = page_size, num_pages, max_pages
        self.page_table = torch.full((slots, max_pages), -1, device=device, dtype=torch.int32)
        self.seq_lens = torch.zeros(slots, device=device, dtype=torch.int32)
        self.pages = [[] for _ in range(slots)]  # of each stream, in order
        self.lens = [0] * slots
        self._users = [0] * num_pages
        self._free = list(range(num_pages))  # a heap: the lowest free page first
        self.mass = self.bounds = None

    def k(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.pool[layer, 1]

    def track_mass(self) -> torch.Tensor:
        """The weights that paged_decode_attention_mass adds up, zeros so far:
        mass[layer] is its argument."""
        if self.mass is None:
            layers, _, _, heads = self.pool.shape[:4]
            self.mass = torch.zeros(layers, len(self.lens), heads, self.max_pages * self.page_size, device=self.pool.device)
        return self.mass

    def track_bounds(self) -> torch.Tensor:
        """The bounds of the keys' pages, those of the positions so far: bounds[layer]
        is the argument of update_page_bounds, to be called for the new tokens, and of
        select_blocks."""
        if self.bounds is None:
            from .paged_sparse import page_bounds
            self.bounds = page_bounds(self.pool[:, 0])
            if any(self.lens):
                self._bound(self.lens)
        return self.bounds

    def _bound(self, counts) -> None:
        """The bounds of the pages of each slot's last counts[s] positions, in all layers."""
        from . import paged_sparse
        cu = torch.tensor([sum(counts[:s]) for s in range(len(counts) + 1)], dtype=torch.int32, device=self.pool.device)
        for layer in range(self.pool.shape[0]):
            paged_sparse.update_page_bounds(self.k(layer), self.bounds[layer], self.page_table, self.seq_lens, cu_seqlens=cu)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._users[p] = 1
        return p

    def _drop(self, page: int) -> None:
        self._users[page] -= 1
        if self._users[page] == 0:
            heapq.heappush(self._free, page)

    def _upload(self, slots) -> None:
        for s in slots:
            row = self.pages[s] + [-1] * (self.max_pages - len(self.pages[s]))
            self.page_table[s].copy_(torch.tensor(row, dtype=torch.int32))
        self.seq_lens.copy_(torch.tensor(self.lens, dtype=torch.int32))

    def reserve(self, counts) -> None:
        """Room for counts[s] more positions of every slot s (0: unchanged);
        seq_lens then counts them.  Nothing is changed if there is not enough."""
        if len(counts) != len(self.lens) or any(c < 0 for c in counts):
            raise ValueError(f"counts must hold {len(self.lens)} numbers, none negative")
        want = [-(-(n + c) // self.page_size) for n, c in zip(self.lens, counts)]
        if max(want) > self.max_pages:
            raise ValueError(f"a stream would need {max(want)} pages of at most {self.max_pages}")
        need = sum(w - len(p) for w, p in zip(want, self.pages))
        if need > len(self._free):
            raise OutOfPages(f"out of pages: {need} needed, {len(self._free)} free")
        grown = [s for s, w in enumerate(want) if w > len(self.pages[s])]
        for s in grown:
            self.pages[s] += [self._take() for _ in range(want[s] - len(self.pages[s]))]
        self.lens = [n + c for n, c in zip(self.lens, counts)]
        self._upload(grown)

    def fork(self, src: int, dst: int) -> None:
        """The stream of slot `src` once more in the empty slot `dst`: full pages
        shared, the partly filled last one copied."""
        if self.pages[dst] or self.lens[dst] or src == dst:
            raise ValueError(f"slot {dst} is not empty")
        full = self.lens[src] // self.page_size
        partial = self.lens[src] % self.page_size > 0
        if partial and not self._free:
            raise OutOfPages("out of pages: 1 needed, 0 free")
        self.pages[dst] = self.pages[src][:full]
        for p in self.pages[dst]:
            self._users[p] += 1
        if partial:
            self.pages[dst].append(self._take())
            self._copy([self.pages[src][full]], [self.pages[dst][full]])
        self.lens[dst] = self.lens[src]
        if self.mass is not None:
            self.mass[:, dst].copy_(self.mass[:, src])
        self._upload([dst])

    def free(self, slot: int) -> None:
        """Empties a slot; its pages that no other stream shares are free again."""
        for p in self.pages[slot]:
            self._drop(p)
        self.pages[slot], self.lens[slot] = [], 0
        if self.mass is not None:
            self.mass[:, slot].zero_()
        self._upload([slot])

    def evict(self, keep: int, recent: int = 0, sinks: int = 0) -> list[int]:
        """Cuts every stream with more than `keep` positions down to `keep`, by the
        weights of track_mass (paged_evict.evict_positions); returns the slots that
        were cut.  Pages that another stream shares are copied first.  Where too few
        are free for all copies, the streams that need the fewest are cut first and
        the pages that they leave serve the others; streams for which that is not
        enough stay as they are (OutOfPages if those are all: nothing was changed)."""
        if self.mass is None:
            raise RuntimeError("eviction goes by the positions' weights: track_mass() before the first token")
        if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
            raise ValueError(f"keep must be positive and cover recent and sinks, which must not be negative: got {keep}, {recent}, {sinks}")
        left = [s for s, n in enumerate(self.lens) if n > keep]
        stay = -(-keep // self.page_size)  # pages of a cut stream, all of which may be written
        cut, need = [], 0
        while left:
            now, own, users = [], [], list(self._users)  # streams that can be cut at once, (slot, place) of their pages that become copies
            shared = lambda s: [i for i, p in enumerate(self.pages[s][:stay]) if users[p] > 1]
            for s in sorted(left, key=lambda s: len(shared(s))):
                mine = shared(s)
                if len(own) + len(mine) > len(self._free):
                    need = need or len(own) + len(mine)
                    continue
                for i in mine:
                    users[self.pages[s][i]] -= 1
                    own.append((s, i))
                now.append(s)
            if not now:
                break
            left = [s for s in left if s not in now]
            self._evict(now, own, left, keep, recent, sinks)
            cut += now
        if left and not cut:
            raise OutOfPages(f"out of pages: {need} needed, {len(self._free)} free")
        return sorted(cut)

    def _evict(self, cut, own, left, keep: int, recent: int, sinks: int) -> None:
        """Cuts the streams `cut`, whose pages `own` (slot, place) become copies; those of `left` are over `keep`, too, and stay."""
        src = [self.pages[s][i] for s, i in own]
        dst = [self._take() for _ in own]
        if own:
            self._copy(src, dst)
            for (s, i), p in zip(own, dst):
                self._drop(self.pages[s][i])
                self.pages[s][i] = p
            self._upload({s for s, _ in own})
        lens = self.seq_lens if not left else torch.tensor([0 if s in left else n for s, n in enumerate(self.lens)], dtype=torch.int32,
                                                           device=self.pool.device)
        from . import paged_evict
        paged_evict.evict_positions(self.pool, self.page_table, lens, self.mass, keep, recent=recent, sinks=sinks)
        stay = -(-keep // self.page_size)
        for s in cut:
            for p in self.pages[s][stay:]:
                self._drop(p)
            del self.pages[s][stay:]
            self.lens[s] = keep
        self._upload(cut)
        if self.bounds is not None:
            self._bound([keep if s in cut else 0 for s in range(len(self.lens))])

    def compact(self) -> int:
        """Moves used pages to the lowest numbers; returns how many moved.  (The
        rest of the pool may then be cut off or handed to something else.)"""
        used = [p for p, n in enumerate(self._users) if n]
        src = [p for p in used if p >= len(used)]
        dst = [p for p in range(len(used)) if self._users[p] == 0]  # as many, and none of them a source
        if not src:
            return 0
        self._copy(src, dst)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self._users[a], self._users[b] = 0, self._users[a]
        self.pages = [[to.get(p, p) for p in pages] for pages in self.pages]
        self._free = list(range(len(used), self.num_pages))
        self._upload(range(len(self.pages)))
        return len(src)

    def _copy(self, src, dst) -> None:
        src, dst = (torch.tensor(v, dtype=torch.int32, device=self.pool.device) for v in (src, dst))
        copy_pages(self.pool, src, dst)
        if self.bounds is not None:
            copy_pages(self.bounds, src, dst)
