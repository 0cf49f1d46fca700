"""Ragged serving of the Zonos-hybrid-shaped model: prompts in, then one token a
stream at its own position, over one paged cache.

``RaggedZonos`` runs the weights of a ``decode_step.SyntheticZonos`` (whose
dense cache holds every stream at one common position) for streams of their
own lengths: ``prompt`` takes any number of new tokens of any of the streams
through the layers (``mamba2_prompt``; ``rotary_paged_append`` and attention
over the stream's own positions), ``step`` one token of every stream that
holds any (the decode-step ops; ``rotary_paged_append`` and
``paged_decode_attention``), both on the same recurrent states and pages.
``fork`` continues a stream twice, ``free`` ends one: its slot is idle until
a prompt or a fork starts another there.

    python -m sonata_b200.kernels.serve      # a small run on cuda:0
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import mamba_step as MS
from . import paged_kv as PK
from .decode_step import SyntheticZonos, ZonosBackboneConfig
from .mamba_prompt import mamba2_prompt


class RaggedZonos:
    def __init__(self, model: SyntheticZonos, num_pages: int, max_len: int, page_size: int = 16):
        """`model`: its batch is the number of streams, its weights are used and its
        own decode state is left alone.  `num_pages` pages of `page_size`
        positions for all streams, `max_len` positions at most for one."""
        cfg = model.cfg
        self.model, self.slots, self.max_len = model, model.batch, max_len
        self.attn = [blk for blk in model.backbone.layers if blk.is_attn]
        self.cache = PK.PagedKVCache(max(1, len(self.attn)), num_pages, cfg.num_heads_kv, cfg.head_dim, self.slots,
                                     -(-max_len // page_size), page_size)
        self.cos, self.sin = PK.rotary_table(max_len, cfg.head_dim)
        self.workspace = PK.decode_workspace(self.slots, cfg.num_heads, cfg.head_dim)
        # (conv_state, ssm_state) of each Mamba2 layer, this object's own
        self.states = [blk.mixer.new_state(self.slots) for blk in model.backbone.layers if not blk.is_attn]

    def _reserve(self, counts) -> None:
        """cache.reserve within max_len, which may end inside a page: there are no rotary angles past it."""
        over = [s for s, c in enumerate(counts) if self.cache.lens[s] + c > self.max_len]
        if over:
            raise ValueError(f"stream {over[0]} would have {self.cache.lens[over[0]] + counts[over[0]]} positions of at most "
                             f"{self.max_len}")
        self.cache.reserve(counts)

    def _layers(self, h: torch.Tensor, mamba, attend) -> torch.Tensor:
        """h [rows, d_model] through the layers and the final norm."""
        cfg, residual = self.model.cfg, None
        at, states = iter(range(len(self.attn))), iter(self.states)
        for blk in self.model.backbone.layers:
            h, residual = MS.layer_norm_fn(h, blk.norm_w, blk.norm_b, residual=residual, eps=cfg.norm_epsilon, prenorm=True)
            if blk.is_attn:
                o = attend(next(at), blk.mixer.in_proj(h))
                h = blk.mixer.out_proj(o)
                h, residual = MS.layer_norm_fn(h, blk.norm2_w, blk.norm2_b, residual=residual, eps=cfg.norm_epsilon, prenorm=True)
                h = blk.mlp(h)
            else:
                h = mamba(blk.mixer, next(states), h)
        bb = self.model.backbone
        return MS.layer_norm_fn(h, bb.norm_f_w, bb.norm_f_b, residual=residual, eps=cfg.norm_epsilon)

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        return self.model.head(h.unsqueeze(0).expand(self.model.cfg.n_codebooks, *h.shape).contiguous())

    @torch.no_grad()
    def prompt(self, hidden: torch.Tensor, lens) -> torch.Tensor:
        """hidden [sum(lens), d_model] bf16: lens[s] new tokens of every stream s,
        packed (0: none).  Returns logits fp32 [n_codebooks, streams, vocab]
        after each stream's last token (0 where it has no new one)."""
        cfg, cache = self.model.cfg, self.cache
        lens = [int(n) for n in lens]
        if len(lens) != self.slots or sum(lens) != hidden.shape[0] or hidden.shape[0] == 0:
            raise ValueError(f"lens must hold {self.slots} lengths that add up to hidden's {hidden.shape[0]} rows, not 0")
        self._reserve(lens)
        offs = [sum(lens[:s]) for s in range(self.slots + 1)]
        cu = torch.tensor(offs, dtype=torch.int32, device=hidden.device)

        def mamba(mx, state, h):
            di, ds, nh = cfg.d_inner, cfg.d_state, cfg.nheads
            y = mamba2_prompt(mx.in_proj(h), state[0], mx.conv_w, mx.conv_b, state[1], mx.A_h, mx.D, mx.dt_bias,
                              di, cfg.ngroups, ds, nh, cu_seqlens=cu, gate=True)
            y = MS.rmsnorm_fn(y.view(-1, di), mx.norm_w, None, eps=cfg.norm_epsilon, group_size=di // cfg.ngroups,
                              norm_before_gate=False)
            return mx.out_proj(y)

        def attend(layer, qkv):
            q = PK.rotary_paged_append(qkv, cache.k(layer), cache.v(layer), cache.page_table, cache.seq_lens, self.cos,
                                       self.sin, cfg.num_heads, cu_seqlens=cu)
            out = torch.empty_like(q)
            for s in range(self.slots):  # causal attention over the stream's own positions
                n, total = lens[s], cache.lens[s]
                if n == 0:
                    continue
                pages = torch.tensor(cache.pages[s], device=q.device)
                k, v = (t[pages].transpose(0, 1).flatten(1, 2)[None, :, :total] for t in (cache.k(layer), cache.v(layer)))
                mask = torch.ones(n, total, device=q.device, dtype=torch.bool).tril(total - n)
                o = F.scaled_dot_product_attention(q[None, offs[s]:offs[s] + n].transpose(1, 2), k, v, attn_mask=mask,
                                                   enable_gqa=True)
                out[offs[s]:offs[s] + n] = o[0].transpose(0, 1)
            return out.flatten(1)

        h = self._layers(hidden, mamba, attend)
        has = [s for s in range(self.slots) if lens[s]]
        last = self._logits(h[torch.tensor([offs[s + 1] - 1 for s in has], device=h.device)])
        logits = last.new_zeros(last.shape[0], self.slots, last.shape[2])
        logits[:, torch.tensor(has, device=h.device)] = last
        return logits

    @torch.no_grad()
    def step(self, hidden: torch.Tensor, active=None) -> torch.Tensor:
        """hidden [streams, d_model] bf16: one new token of every stream that
        `active` (a truth value a stream) names, by default of those that hold
        positions.  The other streams' rows are not read and nothing of them
        changes.  Returns logits fp32 [n_codebooks, streams, vocab] (0 for
        those)."""
        cfg, cache = self.model.cfg, self.cache
        if hidden.shape[0] != self.slots:
            raise ValueError(f"hidden must have {self.slots} rows")
        active = [n > 0 for n in cache.lens] if active is None else [bool(a) for a in active]
        if len(active) != self.slots or not any(active):
            raise ValueError(f"active must hold {self.slots} truth values, and at least one stream must take a token")
        self._reserve([int(a) for a in active])
        table, lens, runs, live = cache.page_table, cache.seq_lens, [(0, self.slots)], None
        if not all(active):  # the active streams' rows, packed; their recurrent states stay where they are, in runs of slots
            live = torch.tensor([s for s in range(self.slots) if active[s]], device=hidden.device)
            hidden, table, lens = hidden[live], table[live], lens[live]
            ends = [s for s in range(self.slots + 1) if (s < self.slots and active[s]) != (s > 0 and active[s - 1])]
            runs = list(zip(ends[::2], ends[1::2]))

        def attend(layer, qkv):
            k, v = cache.k(layer), cache.v(layer)
            q = PK.rotary_paged_append(qkv, k, v, table, lens, self.cos, self.sin, cfg.num_heads)
            return PK.paged_decode_attention(q, k, v, table, lens, workspace=self.workspace).flatten(1)

        def mamba(mx, state, h):
            return mx.step(h, state=[(state[0][a:b], state[1][a:b]) for a, b in runs])

        logits = self._logits(self._layers(hidden, mamba, attend))
        if live is None:
            return logits
        out = logits.new_zeros(logits.shape[0], self.slots, logits.shape[2])
        out[:, live] = logits
        return out

    def fork(self, src: int, dst: int) -> None:
        """Stream `src` once more as the empty stream `dst`: its pages shared, its recurrent states copied."""
        self.cache.fork(src, dst)
        for state in self.states:
            for st in state:
                st[dst].copy_(st[src])

    def free(self, slot: int) -> None:
        """Ends a stream: its pages are free, its recurrent states zero for the next one."""
        self.cache.free(slot)
        for state in self.states:
            for st in state:
                st[slot].zero_()


def main() -> int:
    cfg = ZonosBackboneConfig(n_layer=6, attn_layer_idx=[0, 4])
    m = SyntheticZonos(cfg, batch=3, context=1, max_seqlen=16, seed=0)
    r = RaggedZonos(m, num_pages=200, max_len=1000)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = lambda n: torch.randn(n, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    r.prompt(x(300), [170, 0, 130])
    r.fork(0, 1)
    for _ in range(8):
        logits = r.step(x(3))
    r.free(2)
    moved = r.cache.compact()
    torch.cuda.synchronize()
    print(f"3 streams at {r.cache.lens} positions, {r.cache.free_pages} pages free, {moved} moved, "
          f"logits finite: {bool(torch.isfinite(logits).all())}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
