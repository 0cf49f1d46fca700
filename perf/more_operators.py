"""Operators for long streams in the paged cache: what is measured, in plain torch and on the kernels.

Five operators, each a case dict with "op":

* mass       paged_decode_attention_mass: one new token a stream over its pages, its weights added up a position
* evict      evict_positions: the positions of little weight leave the cache, the others close up
* bounds     update_page_bounds: least and greatest key of the pages that new tokens went to
* select     select_blocks: the blocks a query attends to, by an upper bound of its scores from the pages' bounds
* sparse     paged_sparse_attention: one new token a stream over the listed blocks

The model shapes are this repository's decode step: attention with 16 query and 4 key/value heads of 128, 12 attention
layers.
"""
import math

import torch

own = False

BF16 = torch.bfloat16


def listed():
    return [
        # one stream at a short context: latency
        {"name": "mass_1x257", "op": "mass", "streams": 1, "shortest": 257, "longest": 257, "hq": 16, "hkv": 4, "hd": 128, "page": 16},
        # a serving batch of ragged streams, an empty one among them
        {"name": "mass_64_ragged", "op": "mass", "streams": 64, "shortest": 0, "longest": 5000, "hq": 16, "hkv": 4, "hd": 128, "page": 16},
        # few streams over long contexts, just before they are cut down
        {"name": "mass_3x100001", "op": "mass", "streams": 3, "shortest": 60001, "longest": 100001, "hq": 16, "hkv": 4, "hd": 128, "page": 64},
        # one stream over its budget by a few pages: latency of all layers' eviction between two steps
        {"name": "evict_1x2112", "op": "evict", "layers": 12, "streams": 1, "shortest": 2112, "longest": 2112, "keep": 2048, "recent": 64, "sinks": 4, "hkv": 4, "hd": 128, "page": 16, "source": False},
        # a batch, some of its streams over the budget by different amounts
        {"name": "evict_16_ragged", "op": "evict", "layers": 12, "streams": 16, "shortest": 1000, "longest": 2304, "keep": 2048, "recent": 128, "sinks": 0, "hkv": 4, "hd": 128, "page": 16, "source": True},
        # a long prompt cut down to the budget once it has been read
        {"name": "evict_1x30011", "op": "evict", "layers": 12, "streams": 1, "shortest": 30011, "longest": 30011, "keep": 4096, "recent": 256, "sinks": 16, "hkv": 4, "hd": 128, "page": 64, "source": True},
        # a decode step of 48 streams: each one's last page
        {"name": "bounds_48x1", "op": "bounds", "new": "1", "streams": 48, "longest": 4000, "hkv": 4, "hd": 128, "page": 16},
        # prompts of 7 streams, 12288 tokens in all
        {"name": "bounds_12288", "op": "bounds", "new": "4000,1,129,1500,2048,3333,1277", "streams": 7, "longest": 5000, "hkv": 4, "hd": 128, "page": 32},
        # a serving batch of ragged streams; the short ones attend to all they have
        {"name": "select_48_ragged", "op": "select", "streams": 48, "shortest": 0, "longest": 8000, "hq": 16, "hkv": 4, "hd": 128, "page": 16, "count": 64, "first": 1, "last": 2},
        # few streams over long contexts
        {"name": "select_3x100001", "op": "select", "streams": 3, "shortest": 60001, "longest": 100001, "hq": 16, "hkv": 4, "hd": 128, "page": 16, "count": 128, "first": 1, "last": 4},
        # the same batch over what it selected
        {"name": "sparse_48_ragged", "op": "sparse", "streams": 48, "shortest": 0, "longest": 8000, "hq": 16, "hkv": 4, "hd": 128, "page": 16, "count": 64},
        # and the long streams over theirs
        {"name": "sparse_3x100001", "op": "sparse", "streams": 3, "shortest": 60001, "longest": 100001, "hq": 16, "hkv": 4, "hd": 128, "page": 16, "count": 128},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mass", "evict", "bounds", "select", "sparse"])
    hkv, g = rng.choice([(4, 4), (4, 4), (2, 8), (4, 1), (1, 16), (2, 3)])
    hd, page = rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128])
    if op == "bounds":
        streams = rng.choice([1, 2, 5, 16])
        if rng.random() < 0.4:
            streams, new = _log_int(rng, 1, 256), "1"
        else:
            new = ",".join(str(_log_int(rng, 1, 12288 // streams)) for _ in range(streams))
        return {"op": op, "new": new, "streams": streams, "longest": max(_ints(new)) + _log_int(rng, 1, 4000), "hkv": hkv, "hd": hd, "page": page}
    if op == "evict":
        layers, streams = rng.choice([1, 2, 12]), _log_int(rng, 1, 16)
        longest = _log_int(rng, 100, min(30011, 432000 // (layers * streams)))
        keep = max(1, int(longest * rng.choice([rng.uniform(0.05, 0.95), rng.uniform(0.9, 0.999)])))
        recent, sinks = int(keep * rng.choice([0, rng.uniform(0, 0.3), rng.uniform(0, 0.3), 1])), 0
        if recent < keep and rng.random() < 0.5:
            sinks = rng.randrange(min(keep - recent, 64) + 1)
        return {"op": op, "layers": layers, "streams": streams, "shortest": rng.choice([0, longest // 2, longest]), "longest": longest, "keep": keep,
                "recent": recent, "sinks": sinks, "hkv": hkv, "hd": hd, "page": page, "source": rng.random() < 0.5}
    streams, least = _log_int(rng, 1, 200), 16
    if op == "select":  # enough blocks that there is something to choose
        streams, least = _log_int(rng, 1, 100), 16 * page
    longest = _log_int(rng, least, min(100001, 250000 // streams))
    case = {"op": op, "streams": streams, "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest, "hq": hkv * g, "hkv": hkv, "hd": hd, "page": page}
    if op == "sparse":
        case["count"] = _log_int(rng, 4, max(8, 4096 // page))
    if op == "select":
        case["count"] = _log_int(rng, 6, max(8, min(4096, longest * 3 // 4) // page))
        case["first"], case["last"] = rng.randrange(0, 3), rng.randrange(0, 3)
    return case


def _ints(text):
    return [int(v) for v in text.split(",")]


def _lengths(case, g):
    """Context lengths of the streams: evenly from the longest to the shortest, in no order."""
    n, lo, hi = case["streams"], case["shortest"], case["longest"]
    return torch.linspace(hi, lo, n, device="cuda").round().to(torch.int32)[torch.randperm(n, device="cuda", generator=g)]


def _table(case, g, lens):
    """Pages of each stream in no order, all different, and room for the longest; entries past a stream's pages are -1."""
    page = case["page"]
    most = max(1, -(-case["longest"] // page))
    used = torch.arange(most, device="cuda")[None, :] * page < lens[:, None]
    count = int(used.sum())
    total = count + count // 8 + 3
    table = torch.full((case["streams"], most), -1, device="cuda", dtype=torch.int32)
    table[used] = torch.randperm(total, device="cuda", generator=g)[:count].to(torch.int32)
    return table, total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    u = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    s = dict(case)
    op, hkv, hd, page, n = case["op"], case["hkv"], case["hd"], case["page"], case["streams"]
    if op == "bounds":
        new = _ints(case["new"])
        new = new * n if len(new) == 1 else new
        # what each stream holds already: some nothing, some much
        s["lens"] = torch.tensor([a + int((case["longest"] - a) * (0.618 * i % 1)) for i, a in enumerate(new)], dtype=torch.int32, device="cuda")
        s["table"], pages = _table(case, g, s["lens"])
        s["cu"] = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32, device="cuda")
        s["most_new"] = max(new)
        s["k_pages"] = r(pages, hkv, page, hd).to(BF16)
        s["bounds"] = r(pages, hkv, 2, hd).to(BF16)  # pages of before keep theirs
        return s
    s["lens"] = _lengths(case, g)
    s["table"], pages = _table(case, g, s["lens"])
    room = s["table"].shape[1] * page
    if op == "evict":
        s["pool"] = torch.empty(case["layers"], 2, pages, hkv, page, hd, device="cuda", dtype=BF16)
        for layer in range(case["layers"]):
            s["pool"][layer] = r(2, pages, hkv, page, hd).to(BF16)
        # what attention gathers: a few positions have much, most little, some nothing at all
        m = u(case["layers"], n, hkv, room)
        s["mass"] = torch.where(m < 0.9, 3.0 * m ** 6, 0.0)
        return s
    s["q"] = (1.5 * r(n, case["hq"], hd)).to(BF16)
    if op == "select":
        a, b = r(pages, hkv, hd), r(pages, hkv, hd)
        spread = 0.5 + 1.5 * u(pages, hkv, 1)  # pages of one kind of token and of many
        s["bounds"] = torch.stack([a - spread * b.abs(), a + spread * b.abs()], 2).to(BF16)
        return s
    s["k_pages"] = r(pages, hkv, page, hd).to(BF16)
    s["v_pages"] = r(pages, hkv, page, hd).to(BF16)
    if op == "sparse":
        blocks = (s["lens"] + page - 1).div(page, rounding_mode="floor")
        order = u(n, hkv, s["table"].shape[1])
        at = torch.arange(s["table"].shape[1], device="cuda")
        order = torch.where(at == blocks[:, None, None] - 1, 2.0, torch.where(at < blocks[:, None, None], order, -1.0))
        count = min(case["count"], order.shape[2])
        val, idx = order.topk(count, -1)  # the last block and some of the others
        idx = torch.where(val >= 0, idx, 1 << 30).sort(-1).values
        s["blocks"] = torch.full((n, hkv, case["count"]), -1, device="cuda", dtype=torch.int32)
        s["blocks"][..., :count] = torch.where(idx < 1 << 30, idx, -1).to(torch.int32)
    else:
        s["mass"] = u(n, hkv, room)
    if own:  # the handle that a serving loop keeps for all its steps
        from sonata_b200.kernels import paged_evict, paged_kv
        s["workspace"] = (paged_evict.mass_workspace(n, case["hq"], hkv, hd, room) if op == "mass" else
                          paged_kv.decode_workspace(n, case["hq"], hd))
    return s


def run(s):
    if own:
        from sonata_b200.kernels import paged_evict, paged_sparse
        if s["op"] == "mass":
            o = paged_evict.paged_decode_attention_mass(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["mass"], workspace=s["workspace"])
            return {"o": o, "mass": s["mass"]}
        if s["op"] == "evict":
            source = paged_evict.evict_positions(s["pool"], s["table"], s["lens"], s["mass"], s["keep"], recent=s["recent"], sinks=s["sinks"],
                                                 return_source=s["source"])
            return {"pool": s["pool"], "mass": s["mass"], **({"source": source} if s["source"] else {})}
        if s["op"] == "bounds":
            # a decode step says nothing about the counts: one new token a stream
            paged_sparse.update_page_bounds(s["k_pages"], s["bounds"], s["table"], s["lens"], cu_seqlens=None if s["new"] == "1" else s["cu"])
            return s["bounds"]
        if s["op"] == "select":
            return paged_sparse.select_blocks(s["q"], s["bounds"], s["table"], s["lens"], s["page"], s["count"], first=s["first"], last=s["last"])
        return paged_sparse.paged_sparse_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["blocks"], workspace=s["workspace"])
    return {"mass": _plain_mass, "evict": _plain_evict, "bounds": _plain_bounds, "select": _plain_select, "sparse": _plain_sparse}[s["op"]](s)


# ---- plain forms: torch in 32 bits, rounded once at the end; scores that are compared in 64 ----

def _softmax(score, valid):
    score = score.masked_fill(~valid, -math.inf)
    p = torch.where(valid, torch.exp(score - score.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _plain_mass(s):
    n, hq, hd, hkv = s["streams"], s["hq"], s["hd"], s["hkv"]
    table = s["table"].long().clamp(min=0)
    k = s["k_pages"][table].float().transpose(1, 2).reshape(n, hkv, -1, hd)
    v = s["v_pages"][table].float().transpose(1, 2).reshape(n, hkv, -1, hd)
    q = s["q"].float().view(n, hkv, hq // hkv, hd)
    valid = (torch.arange(k.shape[2], device="cuda") < s["lens"][:, None])[:, None, None]
    p = _softmax((q @ k.transpose(2, 3)) / math.sqrt(hd), valid)
    s["mass"] += p.sum(2)
    return {"o": (p @ v).view(n, hq, hd).to(BF16), "mass": s["mass"]}


def _plain_evict(s):
    keep, recent, sinks, page = s["keep"], s["recent"], s["sinks"], s["page"]
    mass, lens, table = s["mass"], s["lens"].long()[:, None, None], s["table"].long()
    layers, n, hkv, room = mass.shape
    at = torch.arange(room, device="cuda")
    over = lens > keep
    free = (at >= sinks) & (at < lens - recent)  # may go
    order = torch.where(free, mass, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order).contiguous())
    chosen = free & (rank < keep - recent - sinks)
    hole = (at >= sinks) & (at < keep - recent) & ~chosen
    mover = (at >= keep - recent) & chosen
    movers = torch.where(mover, at, room).sort(-1).values
    at = at[:keep] if keep <= room else torch.arange(keep, device="cuda")
    whole = torch.where(at < lens, at, -1)  # of a stream that stays as it is
    fill = torch.zeros(layers, n, hkv, keep, dtype=torch.bool, device="cuda")
    w = min(keep, room)
    fill[..., :w] = hole[..., :w]
    nth = (fill.cumsum(-1) - 1).clamp(min=0, max=room - 1)
    source = torch.where(fill, movers.gather(-1, nth), at)
    source = torch.where(at >= keep - recent, at - keep + lens, source)
    source = torch.where(over, source, whole)
    # rows of the streams that are cut: from their source to their place
    rows = over[:, 0, 0].nonzero()[:, 0]
    if rows.numel():
        src = source[:, rows]
        b = rows[:, None, None]
        h = torch.arange(hkv, device="cuda")[:, None]
        to_page, to_at = table[b, (at // page).expand(1, 1, -1)], at % page
        for layer in range(layers):
            pg, row = table[b, src[layer] // page], src[layer] % page
            s["pool"][layer][:, to_page, h, to_at] = s["pool"][layer][:, pg, h, row]
        moved = mass[:, rows].gather(-1, src)
        tail = torch.arange(room, device="cuda") < lens[rows]
        mass[:, rows] = torch.where(tail, 0.0, mass[:, rows])
        mass[:, rows, :, :keep] = moved
    return {"pool": s["pool"], "mass": mass, **({"source": source.to(torch.int32)} if s["source"] else {})}


def _plain_bounds(s):
    page, n, pages = s["page"], s["streams"], s["k_pages"].shape[0]
    lens, cu = s["lens"].long(), s["cu"].long()
    lo = (lens - (cu[1:] - cu[:-1])).div(page, rounding_mode="floor")
    block = lo[:, None] + torch.arange(s["most_new"] // page + 2, device="cuda")
    valid = block * page < lens[:, None]
    pg = torch.where(valid, s["table"].long().gather(1, block.clamp(max=s["table"].shape[1] - 1)), pages)  # no page: a spare one
    k = s["k_pages"][pg.clamp(max=pages - 1)].float()  # [n, blocks, hkv, page, hd]
    there = (block[..., None] * page + torch.arange(page, device="cuda") < lens[:, None, None])[:, :, None, :, None]
    new = torch.stack([k.masked_fill(~there, math.inf).amin(3), k.masked_fill(~there, -math.inf).amax(3)], 3)
    all_pages = torch.cat([s["bounds"], s["bounds"][:1]])
    all_pages[pg] = new.to(BF16)
    s["bounds"].copy_(all_pages[:pages])
    return s["bounds"]


def _plain_select(s):
    n, hq, hkv, hd, page, count = s["streams"], s["hq"], s["hkv"], s["hd"], s["page"], s["count"]
    lo, hi = s["bounds"][s["table"].long().clamp(min=0)].double().permute(3, 0, 2, 4, 1)  # [n, hkv, hd, blocks] each
    q = s["q"].double().view(n, hkv, hq // hkv, hd)
    score = (q.clamp(min=0) @ hi + q.clamp(max=0) @ lo).amax(2)
    at = torch.arange(score.shape[2], device="cuda")
    blocks = (s["lens"].long() + page - 1).div(page, rounding_mode="floor")[:, None, None]
    score = score.masked_fill((at < s["first"]) | (at >= blocks - s["last"]), math.inf).masked_fill(at >= blocks, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :count]
    best = torch.where(best < blocks, best, 1 << 30).sort(-1).values
    out = torch.full((n, hkv, count), -1, device="cuda", dtype=torch.int32)
    out[..., :best.shape[2]] = torch.where(best < 1 << 30, best, -1)
    return out


def _plain_sparse(s):
    n, hq, hkv, hd, page = s["streams"], s["hq"], s["hkv"], s["hd"], s["page"]
    blocks = s["blocks"].long()
    pg = s["table"].long()[:, None].expand(-1, hkv, -1).gather(2, blocks.clamp(min=0)).clamp(min=0)
    h = torch.arange(hkv, device="cuda")[:, None]
    k = s["k_pages"][pg, h].float().reshape(n, hkv, -1, hd)
    v = s["v_pages"][pg, h].float().reshape(n, hkv, -1, hd)
    where = blocks[..., None] * page + torch.arange(page, device="cuda")
    valid = ((where < s["lens"][:, None, None, None]) & (blocks >= 0)[..., None]).reshape(n, hkv, 1, -1)
    q = s["q"].float().view(n, hkv, hq // hkv, hd)
    return (_softmax((q @ k.transpose(2, 3)) / math.sqrt(hd), valid) @ v).view(n, hq, hd).to(BF16)


# ---- 64 bits, from the definitions, a stream and head at a time ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"mass": _exact_mass, "evict": _exact_evict, "bounds": _exact_bounds, "select": _exact_select, "sparse": _exact_sparse}[case["op"]](s)


def _exact_mass(s):
    hq, hkv, hd = s["hq"], s["hkv"], s["hd"]
    g = hq // hkv
    out, mass = torch.zeros(s["streams"], hq, hd, device="cuda", dtype=torch.float64), s["mass"].double()
    for i, n in enumerate(s["lens"].tolist()):
        pages = s["table"][i, : -(-n // s["page"])].long()
        for h in range(hkv if n else 0):
            k = s["k_pages"][pages, h].reshape(-1, hd)[:n].double()
            v = s["v_pages"][pages, h].reshape(-1, hd)[:n].double()
            p = torch.softmax(s["q"][i, h * g:(h + 1) * g].double() @ k.T / hd ** 0.5, -1)
            out[i, h * g:(h + 1) * g] = p @ v
            mass[i, h, :n] += p.sum(0)
    return {"o": out, "mass": mass}


def _exact_evict(s):
    keep, recent, sinks, page = s["keep"], s["recent"], s["sinks"], s["page"]
    pool, mass = s["pool"].clone(), s["mass"].double()
    layers, n, hkv, _ = mass.shape
    source = torch.full((layers, n, hkv, keep), -1, device="cuda", dtype=torch.int32)
    for i, total in enumerate(s["lens"].tolist()):
        if total <= keep:
            source[:, i, :, :total] = torch.arange(total, device="cuda")
            continue
        where = torch.arange(total, device="cuda")
        pg, at = s["table"][i].long()[where // page], where % page
        for layer in range(layers):
            for h in range(hkv):
                old = mass[layer, i, h, :total].clone()
                best = sinks + torch.sort(old[sinks:total - recent], descending=True, stable=True).indices[:keep - recent - sinks]
                best = best.sort().values
                stay = best[best < keep - recent]
                free = torch.ones(keep - recent, dtype=torch.bool, device="cuda")
                free[:sinks] = False
                free[stay] = False
                src = where[:keep].clone()
                src[:keep - recent][free] = best[best >= keep - recent]
                src[keep - recent:] = where[total - recent:]
                for kv in range(2):
                    rows = s["pool"][layer, kv, pg, h, at]
                    pool[layer, kv, pg[:keep], h, at[:keep]] = rows[src]
                mass[layer, i, h, :keep] = old[src]
                mass[layer, i, h, keep:total] = 0
                source[layer, i, h] = src.to(torch.int32)
    return {"pool": pool, "mass": mass, **({"source": source} if s["source"] else {})}


def _exact_bounds(s):
    out, page = s["bounds"].double(), s["page"]
    cu = s["cu"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        for b in range((n - (cu[i + 1] - cu[i])) // page, -(-n // page)):
            pg = int(s["table"][i, b])
            k = s["k_pages"][pg, :, :min(page, n - b * page)].double()
            out[pg, :, 0], out[pg, :, 1] = k.min(1).values, k.max(1).values
    return out


def _exact_select(s):
    hkv, g, page, count = s["hkv"], s["hq"] // s["hkv"], s["page"], s["count"]
    out = torch.full((s["streams"], hkv, count), -1, device="cuda", dtype=torch.int32)
    for i, n in enumerate(s["lens"].tolist()):
        blocks = -(-n // page)
        for h in range(hkv if n else 0):
            b = s["bounds"][s["table"][i, :blocks].long(), h].double()
            best = torch.full((blocks,), -math.inf, device="cuda", dtype=torch.float64)
            for q in s["q"][i, h * g:(h + 1) * g].double():
                best = torch.maximum(best, torch.maximum(b[:, 0] * q, b[:, 1] * q).sum(1))
            best[:s["first"]] = math.inf
            best[max(0, blocks - s["last"]):] = math.inf
            top = torch.sort(best, descending=True, stable=True).indices[:count].sort().values
            out[i, h, :top.numel()] = top.to(torch.int32)
    return out


def _exact_sparse(s):
    hq, hkv, hd, page = s["hq"], s["hkv"], s["hd"], s["page"]
    g = hq // hkv
    out = torch.zeros(s["streams"], hq, hd, device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["lens"].tolist()):
        for h in range(hkv if n else 0):
            blocks = s["blocks"][i, h][s["blocks"][i, h] >= 0].long()
            there = (blocks[:, None] * page + torch.arange(page, device="cuda") < n).flatten()
            pages = s["table"][i, blocks].long()
            k = s["k_pages"][pages, h].reshape(-1, hd)[there].double()
            v = s["v_pages"][pages, h].reshape(-1, hd)[there].double()
            out[i, h * g:(h + 1) * g] = torch.softmax(s["q"][i, h * g:(h + 1) * g].double() @ k.T / hd ** 0.5, -1) @ v
    return out


def _spread(case):
    """The streams' lengths, as prepare() spreads them."""
    n, lo, hi = case["streams"], case["shortest"], case["longest"]
    return [hi] if n == 1 else [round(hi + (lo - hi) * i / (n - 1)) for i in range(n)]


def work(case):
    hkv, hd, page = case["hkv"], case["hd"], case["page"]
    if case["op"] == "bounds":
        new = _ints(case["new"])
        new = new * case["streams"] if len(new) == 1 else new
        pages = sum(-(-a // page) for a in new)
        # the new keys read, the bounds of their pages written, and read where the first of them was begun before
        return {"bytes": sum(new) * hkv * hd * 2 + (pages + len(new)) * hkv * hd * 4, "flops": sum(new) * hkv * hd * 2}
    lens = _spread(case)
    if case["op"] == "evict":
        keep, recent, sinks = case["keep"], case["recent"], case["sinks"]
        total = 0
        for n in lens:
            if n > keep:
                moved = recent + (n - keep) * (keep - recent - sinks) / max(1, n - recent - sinks)
                total += 4 * (n - sinks - recent) + moved * (8 * hd + 8) + 4 * (n - keep) + (4 * keep if case["source"] else 0)
        return {"bytes": max(1, total * case["layers"] * hkv), "flops": 0}
    hq, n = case["hq"], case["streams"]
    if case["op"] == "mass":
        tokens = sum(lens)
        return {"bytes": tokens * hkv * (4 * hd + 8) + tokens / page * 4 + n * hq * hd * 4, "flops": tokens * hq * (4 * hd + 1)}
    blocks = [-(-a // page) for a in lens]
    if case["op"] == "select":
        scored = sum(b for b in blocks if b > case["count"])  # the others take all they have
        return {"bytes": max(1, scored * (hkv * hd * 4 + 4) + n * (hq * hd * 2 + hkv * case["count"] * 4)), "flops": scored * hq * hd * 4}
    tokens = sum(min(a, case["count"] * page) for a in lens)
    return {"bytes": max(1, tokens * hkv * hd * 4 + n * (hq * hd * 4 + hkv * case["count"] * 4)), "flops": tokens * hq * hd * 4}
