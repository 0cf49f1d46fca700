"""Operators of a ragged, paged serving step of the Mamba2 / attention hybrid: what is measured, in plain torch and on the kernels.

Four operators, each a case dict with "op":

* prompt     mamba2_prompt: causal convolution and selective state space scan of packed ragged prompts
* append     rotary_paged_append: rotary positions of q and k, k and v written to the cache's pages
* attend     paged_decode_attention: one new token a stream over its pages
* copy       copy_pages: pages copied in every layer's pool (forks, compaction)

The model shapes are this repository's decode step: 64 heads of 64, state 128, convolution width 4 (4352 channels),
attention with 16 query and 4 key/value heads of 128, 12 attention layers.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
HEADDIM, DSTATE, DCONV = 64, 128, 4


def listed():
    return [
        # the prompt of one short utterance, taken by one stream: latency of a dozen layers' worth of launches
        {"name": "prompt_1x37", "op": "prompt", "lens": "37", "nheads": 64, "ngroups": 1, "gate": False, "fresh": True},
        # one speech prompt with its conditioning prefix
        {"name": "prompt_1x1021", "op": "prompt", "lens": "1021", "nheads": 64, "ngroups": 1, "gate": False, "fresh": True},
        # prompts of a batch of streams arriving together, some continued from an earlier piece, gated output
        {"name": "prompt_9_ragged", "op": "prompt", "lens": "700,1,129,1500,64,333,2048,5,811", "nheads": 64, "ngroups": 1, "gate": True, "fresh": False},
        # a long document read in one piece
        {"name": "prompt_1x16384", "op": "prompt", "lens": "16384", "nheads": 64, "ngroups": 1, "gate": False, "fresh": True},
        # a decode step of 48 streams: one token each at its own position
        {"name": "append_48x1", "op": "append", "new": "1", "streams": 48, "longest": 4000, "hq": 16, "hkv": 4, "hd": 128, "rot": 128, "inter": False, "page": 16},
        # prompts of 9 streams, 12288 tokens in all, halves layout over the whole head
        {"name": "append_12288", "op": "append", "new": "4000,1,129,1500,2048,3333,1277", "streams": 7, "longest": 4000, "hq": 16, "hkv": 4, "hd": 128, "rot": 128, "inter": False, "page": 32},
        # the same kind of prompts where half of each head is rotated in interleaved pairs, more heads, odd count
        {"name": "append_part_inter", "op": "append", "new": "1111,2222,777", "streams": 3, "longest": 5000, "hq": 32, "hkv": 8, "hd": 128, "rot": 64, "inter": True, "page": 64},
        # one stream at a short context: latency
        {"name": "attend_1x257", "op": "attend", "streams": 1, "shortest": 257, "longest": 257, "hq": 16, "hkv": 4, "hd": 128, "page": 16},
        # a serving batch of ragged streams, an empty one among them
        {"name": "attend_64_ragged", "op": "attend", "streams": 64, "shortest": 0, "longest": 5000, "hq": 16, "hkv": 4, "hd": 128, "page": 16},
        # few streams over long contexts: the length has to be split
        {"name": "attend_3x100001", "op": "attend", "streams": 3, "shortest": 60001, "longest": 100001, "hq": 16, "hkv": 4, "hd": 128, "page": 64},
        # forking one stream: its last, partly filled page
        {"name": "copy_fork", "op": "copy", "pairs": 3, "pages": 64, "layers": 12, "hkv": 4, "page": 16, "hd": 128},
        # compaction of a cache after many streams have ended
        {"name": "copy_compact", "op": "copy", "pairs": 1500, "pages": 4000, "layers": 12, "hkv": 4, "page": 16, "hd": 128},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "append", "attend", "copy"])
    if op == "prompt":
        total, n = _log_int(rng, 16, 16384), rng.choice([1, 1, 2, 3, 8, 17])
        cut = sorted(rng.randrange(total + 1) for _ in range(n - 1))
        lens = [b - a for a, b in zip([0] + cut, cut + [total])]
        return {"op": op, "lens": ",".join(map(str, lens)), "nheads": rng.choice([64, 64, 32, 48]), "ngroups": rng.choice([1, 1, 2]), "gate": rng.random() < 0.5, "fresh": rng.random() < 0.5}
    hkv, g = rng.choice([(4, 4), (4, 4), (8, 4), (2, 8), (8, 1), (1, 16)])
    hd, page = rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128])
    if op == "append":
        streams = rng.choice([1, 2, 5, 16])
        if rng.random() < 0.4:
            streams, new = _log_int(rng, 1, 256), "1"
        else:
            new = ",".join(str(_log_int(rng, 1, 16384 // streams)) for _ in range(streams))
        rot = rng.choice([hd, hd, hd // 2, hd // 4])
        if hkv * (g + 2) > 24:
            hkv, g = 4, 4
        return {"op": op, "new": new, "streams": streams, "longest": max(_ints(new)) + _log_int(rng, 1, 4000), "hq": hkv * g, "hkv": hkv, "hd": hd, "rot": rot, "inter": rng.random() < 0.5, "page": page}
    if op == "attend":
        streams = _log_int(rng, 1, 200)
        longest = _log_int(rng, 16, min(100001, 250000 // streams))
        if hkv > 4:
            hkv = 4
        return {"op": op, "streams": streams, "shortest": rng.choice([0, 1, longest // 2, longest]), "longest": longest, "hq": hkv * g, "hkv": hkv, "hd": hd, "page": page}
    layers, pairs = rng.choice([1, 2, 12]), _log_int(rng, 1, 1500)
    return {"op": op, "pairs": pairs, "pages": 2 * pairs + rng.randrange(1, 500), "layers": layers, "hkv": rng.choice([2, 4]), "page": rng.choice([16, 8, 32]), "hd": 64 if layers == 12 else hd}


def _ints(text):
    return [int(v) for v in text.split(",")]


def _gen(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


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
    g = _gen(case, seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    u = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    s = dict(case)
    if case["op"] == "prompt":
        lens, nh, ng = _ints(case["lens"]), case["nheads"], case["ngroups"]
        di, gds, total = nh * HEADDIM, ng * DSTATE, sum(lens)
        s["zxbcdt"] = r(total, 2 * di + 2 * gds + nh).to(BF16)  # what in_proj gives: [z | x B C | dt]
        cd = di + 2 * gds
        s["conv_w"], s["conv_b"] = (0.5 * r(cd, DCONV)).to(BF16), (0.1 * r(cd)).to(BF16)
        s["A"] = -(u(nh) * 15 + 1)
        s["D"], s["dt_bias"] = (1 + 0.2 * r(nh)).to(BF16), (u(nh) * 2 - 4).to(BF16)
        k = 0.0 if case["fresh"] else 1.0
        s["conv_state"] = (k * r(len(lens), cd, DCONV)).to(BF16)
        s["ssm_state"] = (0.5 * k * r(len(lens), nh, HEADDIM, DSTATE)).to(BF16)
        s["cu"], s["longest"] = _cu(lens), max(lens)
    elif case["op"] == "append":
        new = _ints(case["new"])
        new = new * case["streams"] if len(new) == 1 else new
        # what each stream holds already: some nothing, some much
        s["lens"] = torch.tensor([n + int((case["longest"] - n) * (0.618 * i % 1)) for i, n in enumerate(new)], dtype=torch.int32, device="cuda")
        s["table"], pages = _table(case, g, s["lens"])
        s["k_pages"] = torch.zeros(pages, case["hkv"], case["page"], case["hd"], device="cuda", dtype=BF16)
        s["v_pages"] = torch.zeros_like(s["k_pages"])
        s["qkv"] = r(sum(new), (case["hq"] + 2 * case["hkv"]) * case["hd"]).to(BF16)
        s["cu"] = _cu(new)
        half = case["rot"] // 2
        angle = torch.arange(case["longest"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif case["op"] == "attend":
        s["lens"] = _lengths(case, g)
        s["table"], pages = _table(case, g, s["lens"])
        s["k_pages"] = r(pages, case["hkv"], case["page"], case["hd"]).to(BF16)
        s["v_pages"] = r(pages, case["hkv"], case["page"], case["hd"]).to(BF16)
        s["q"] = (1.5 * r(case["streams"], case["hq"], case["hd"])).to(BF16)
        if own:  # the handle that a serving loop keeps for all its steps
            from sonata_b200.kernels import paged_kv
            s["workspace"] = paged_kv.decode_workspace(case["streams"], case["hq"], case["hd"])
    else:
        s["pool"] = r(case["layers"], 2, case["pages"], case["hkv"], case["page"], case["hd"]).to(BF16)
        order = torch.randperm(case["pages"], device="cuda", generator=g)[: 2 * case["pairs"]].to(torch.int32)
        s["src"], s["dst"] = order[: case["pairs"]].contiguous(), order[case["pairs"]:].contiguous()
    return s


def run(s):
    if own:
        from sonata_b200.kernels import mamba_prompt, paged_kv
        if s["op"] == "prompt":
            y = mamba_prompt.mamba2_prompt(s["zxbcdt"], s["conv_state"], s["conv_w"], s["conv_b"], s["ssm_state"], s["A"], s["D"], s["dt_bias"],
                                           s["nheads"] * HEADDIM, s["ngroups"], DSTATE, s["nheads"], cu_seqlens=s["cu"], gate=s["gate"])
            return {"y": y, "conv_state": s["conv_state"], "ssm_state": s["ssm_state"]}
        if s["op"] == "append":
            q = paged_kv.rotary_paged_append(s["qkv"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cos"], s["sin"], s["hq"],
                                             cu_seqlens=s["cu"], interleaved=s["inter"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["op"] == "attend":
            return paged_kv.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], workspace=s["workspace"])
        paged_kv.copy_pages(s["pool"], s["src"], s["dst"])
        return s["pool"]
    return {"prompt": _plain_prompt, "append": _plain_append, "attend": _plain_attend, "copy": _plain_copy}[s["op"]](s)


# ---- plain forms: torch in 32 bits, rounded once at the end ----

def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _plain_prompt(s):
    nh, ng, chunk = s["nheads"], s["ngroups"], 128
    di, gds = nh * HEADDIM, ng * DSTATE
    cu, lens = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    b, nc = lens.numel(), -(-s["longest"] // chunk)
    t = torch.arange(nc * chunk, device="cuda")
    valid = t[None, :] < lens[:, None]  # the streams side by side, padded to whole chunks
    zx = s["zxbcdt"][(cu[:, None] + t).clamp_(max=s["zxbcdt"].shape[0] - 1)].float() * valid[..., None]
    # convolution over [the last W - 1 inputs before the prompt | the prompt]
    hist = s["conv_state"].float().transpose(1, 2)  # [b, W, channels], newest last
    u = torch.cat([hist, zx[..., di:2 * di + 2 * gds]], 1)
    w = s["conv_w"].float()
    n = nc * chunk
    xbc = _silu(s["conv_b"].float() + u[:, 1:1 + n] * w[:, 0] + u[:, 2:2 + n] * w[:, 1] + u[:, 3:3 + n] * w[:, 2] + u[:, 4:4 + n] * w[:, 3])
    last = lens[:, None] + torch.arange(DCONV, device="cuda")
    s["conv_state"].copy_(u.gather(1, last[..., None].expand(-1, -1, u.shape[2])).transpose(1, 2).to(BF16))
    x = xbc[..., :di].reshape(b, nc, chunk, nh, HEADDIM)
    rep = nh // ng
    B = xbc[..., di:di + gds].reshape(b, nc, chunk, ng, DSTATE)
    C = xbc[..., di + gds:].reshape(b, nc, chunk, ng, DSTATE)
    dt = (_softplus(zx[..., 2 * di + 2 * gds:] + s["dt_bias"].float()) * valid[..., None]).reshape(b, nc, chunk, nh).permute(0, 1, 3, 2)  # [b, c, h, l]
    a = (dt * s["A"][:, None]).cumsum(-1)
    low = torch.ones(chunk, chunk, device="cuda", dtype=torch.bool).tril()
    m = torch.exp((a[..., :, None] - a[..., None, :]).masked_fill_(~low, -math.inf)).mul_(dt[..., None, :])
    G = torch.einsum("bcign,bcjgn->bcgij", C, B)
    m = (m.unflatten(2, (ng, rep)) * G[:, :, :, None]).flatten(2, 3)
    y = torch.einsum("bchij,bcjhp->bcihp", m, x)
    # states: of each chunk alone, then carried over the chunks
    xw = x * (torch.exp(a[..., -1:] - a) * dt).permute(0, 1, 3, 2)[..., None]
    st = torch.einsum("bcjgn,bcjgrp->bcgrpn", B, xw.reshape(b, nc, chunk, ng, rep, HEADDIM)).reshape(b, nc, nh, HEADDIM, DSTATE)
    st = torch.cat([s["ssm_state"].float()[:, None], st], 1)
    tot = torch.cat([torch.zeros(b, nh, 1, device="cuda"), a[..., -1].transpose(1, 2)], -1)  # [b, h, 1 + c]
    k = nc + 1
    below = torch.ones(k, k, device="cuda", dtype=torch.bool).tril(-1)
    seg = tot[..., :, None].expand(-1, -1, -1, k).masked_fill(~below, 0).cumsum(-2)  # sum over (j, i]
    carry = torch.exp(seg.masked_fill(~(below | torch.eye(k, device="cuda", dtype=torch.bool)), -math.inf))
    st = torch.einsum("bhij,bjhpn->bihpn", carry, st)
    off = torch.einsum("bcign,bcgrpn->bcigrp", C, st[:, :-1].reshape(b, nc, ng, rep, HEADDIM, DSTATE)).reshape(b, nc, chunk, nh, HEADDIM)
    y = y + off * torch.exp(a).permute(0, 1, 3, 2)[..., None] + x * s["D"].float()[:, None]
    s["ssm_state"].copy_(st[:, -1].to(BF16))
    y = y.reshape(b, n, nh, HEADDIM)
    if s["gate"]:
        y = y * _silu(zx[..., :di]).reshape(b, n, nh, HEADDIM)
    rows = torch.arange(s["zxbcdt"].shape[0], device="cuda")
    of = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    return {"y": y[of, rows - cu[of]].to(BF16), "conv_state": s["conv_state"], "ssm_state": s["ssm_state"]}


def _where(s):
    """(position, page, place in the page) of each new token."""
    rows = torch.arange(s["qkv"].shape[0], device="cuda")
    cu = s["cu"].long()
    of = torch.searchsorted(cu[1:], rows, right=True)
    pos = s["lens"].long()[of] - cu[of + 1] + rows
    return pos, s["table"][of, pos // s["page"]].long(), pos % s["page"]


def _plain_append(s):
    hq, hkv, hd, rot = s["hq"], s["hkv"], s["hd"], s["rot"]
    pos, page, at = _where(s)
    qkv = s["qkv"].float().view(-1, hq + 2 * hkv, hd)
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    x = qkv[:, :hq + hkv]
    if s["inter"]:
        x1, x2 = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([x1 * c - x2 * n, x2 * c + x1 * n], -1).flatten(-2)
    else:
        x1, x2 = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([x1 * c - x2 * n, x2 * c + x1 * n], -1)
    x = torch.cat([turned, x[..., rot:]], -1).to(BF16)
    s["k_pages"][page, :, at] = x[:, hq:]
    s["v_pages"][page, :, at] = qkv[:, hq + hkv:].to(BF16)
    return {"q": x[:, :hq].contiguous(), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    n, hq, hd, hkv = s["streams"], s["hq"], s["hd"], s["hkv"]
    table = s["table"].long().clamp(min=0)
    k = s["k_pages"][table].float().transpose(1, 2).reshape(n, hkv, -1, hd)
    v = s["v_pages"][table].float().transpose(1, 2).reshape(n, hkv, -1, hd)
    q = s["q"].float().view(n, hkv, hq // hkv, hd)
    score = (q @ k.transpose(2, 3)) / math.sqrt(hd)
    valid = (torch.arange(k.shape[2], device="cuda") < s["lens"][:, None])[:, None, None]
    score = score.masked_fill(~valid, -math.inf)
    p = torch.where(valid, torch.exp(score - score.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1, keepdim=True)
    return ((p @ v) / torch.where(total > 0, total, 1.0)).view(n, hq, hd).to(BF16)


def _plain_copy(s):
    s["pool"][:, :, s["dst"].long()] = s["pool"][:, :, s["src"].long()]
    return s["pool"]


# ---- 64 bits, from the definitions ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "append": _exact_append, "attend": _exact_attend, "copy": _exact_copy}[case["op"]](s)


def _exact_prompt(s):
    """The recurrence itself, token by token, each stream on its own."""
    nh, ng = s["nheads"], s["ngroups"]
    di, gds = nh * HEADDIM, ng * DSTATE
    w, bias, A, D = s["conv_w"].double(), s["conv_b"].double(), s["A"].double(), s["D"].double()
    ys, convs, ssms = [], [], []
    for i, n in enumerate(_ints(s["lens"])):
        at = int(s["cu"][i])
        z, u, dt = s["zxbcdt"][at:at + n].double().split([di, di + 2 * gds, nh], 1)
        u = torch.cat([s["conv_state"][i].double().T, u])
        convs.append(u[n:].T)
        xbc = bias + sum(w[:, k] * u[1 + k:1 + k + n] for k in range(DCONV))
        xbc = xbc * torch.sigmoid(xbc)
        dt = torch.logaddexp(dt + s["dt_bias"].double(), torch.zeros((), device="cuda", dtype=torch.float64))
        decay = torch.exp(dt * A)
        x = xbc[:, :di].reshape(n, nh, HEADDIM)
        B, C = (v.reshape(n, ng, DSTATE).repeat_interleave(nh // ng, 1) for v in (xbc[:, di:di + gds], xbc[:, di + gds:]))
        state, y = s["ssm_state"][i].double(), torch.empty(n, nh, HEADDIM, device="cuda", dtype=torch.float64)
        add = x * dt[..., None]
        for t in range(n):
            state = torch.baddbmm(state * decay[t, :, None, None], add[t, :, :, None], B[t, :, None, :])
            y[t] = torch.bmm(state, C[t, :, :, None])[..., 0]
        y += D[:, None] * x
        if s["gate"]:
            y *= (z * torch.sigmoid(z)).view(n, nh, HEADDIM)
        ys.append(y)
        ssms.append(state)
    return {"y": torch.cat(ys), "conv_state": torch.stack(convs), "ssm_state": torch.stack(ssms)}


def _exact_append(s):
    hq, hkv, hd, rot = s["hq"], s["hkv"], s["hd"], s["rot"]
    k, v = s["k_pages"].double(), s["v_pages"].double()
    q = []
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].long()
    for i in range(s["streams"]):
        n = cu[i + 1] - cu[i]
        pos = torch.arange(lens[i] - n, lens[i], device="cuda")
        rows = s["qkv"][cu[i]:cu[i + 1]].double().view(n, hq + 2 * hkv, hd)
        turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
        head = rows[:, :hq + hkv, :rot].reshape(n, hq + hkv, *((rot // 2, 2) if s["inter"] else (2, rot // 2)))
        dim = -1 if s["inter"] else -2
        c = torch.complex(head.select(dim, 0), head.select(dim, 1)) * turn
        qk = torch.cat([torch.stack([c.real, c.imag], dim).flatten(-2), rows[:, :hq + hkv, rot:]], -1)
        q.append(qk[:, :hq])
        page, at = table[i, pos // s["page"]], pos % s["page"]
        k[page, :, at], v[page, :, at] = qk[:, hq:], rows[:, hq + hkv:]
    return {"q": torch.cat(q), "k_pages": k, "v_pages": v}


def _exact_attend(s):
    hq, hkv, hd = s["hq"], s["hkv"], s["hd"]
    out = torch.zeros(s["streams"], hq, hd, device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["lens"].tolist()):
        pages = s["table"][i, : -(-n // s["page"])].long()
        for h in range(hkv if n else 0):
            k = s["k_pages"][pages, h].reshape(-1, hd)[:n].double()
            v = s["v_pages"][pages, h].reshape(-1, hd)[:n].double()
            q = s["q"][i, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            out[i, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.softmax(q @ k.T / hd ** 0.5, -1) @ v
    return out


def _exact_copy(s):
    pool = s["pool"].double()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        pool[:, :, b] = s["pool"][:, :, a].double()
    return pool


def _expected_tokens(case):
    """Tokens of context over all streams, as prepare() spreads their lengths."""
    n, lo, hi = case["streams"], case["shortest"], case["longest"]
    return hi if n == 1 else n * (lo + hi) / 2


def work(case):
    if case["op"] == "prompt":
        lens, nh, ng = _ints(case["lens"]), case["nheads"], case["ngroups"]
        di, gds, total = nh * HEADDIM, ng * DSTATE, sum(lens)
        row = di + 2 * gds + nh + (di if case["gate"] else 0) + di  # xBC and dt (and z) read, y written
        states = len(lens) * 2 * 2 * ((di + 2 * gds) * DCONV + di * DSTATE)
        # the recurrence: the state's decay and update and the product with C; the convolution
        return {"bytes": 2 * total * row + states + 2 * (di + 2 * gds) * (DCONV + 1), "flops": total * (5 * di * DSTATE + (di + 2 * gds) * (2 * DCONV + 4))}
    if case["op"] == "append":
        new = _ints(case["new"])
        total = sum(new) * (case["streams"] if len(new) == 1 else 1)
        heads = case["hq"] + 2 * case["hkv"]
        return {"bytes": total * (heads * case["hd"] * 4 + case["rot"] * 4) + 4 * total // case["page"], "flops": total * (case["hq"] + case["hkv"]) * case["rot"] * 3}
    if case["op"] == "attend":
        tokens = _expected_tokens(case)
        return {"bytes": tokens * (case["hkv"] * case["hd"] * 4 + 4 / case["page"]) + case["streams"] * case["hq"] * case["hd"] * 4, "flops": tokens * case["hq"] * case["hd"] * 4}
    return {"bytes": 2 * 2 * 2 * case["pairs"] * case["layers"] * case["hkv"] * case["page"] * case["hd"], "flops": 0}
