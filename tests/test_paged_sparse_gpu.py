"""Bounds of pages, the choice of blocks and attention over them, against plain implementations in 64 bits.

Bounds and choices are equal.  Attention: the bound of paged_decode_attention's test, E (|o| + P) + 2 E_s P + 2^-19 P, over the
listed positions."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -8
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def PS(cuda_lib):
    from sonata_b200.kernels import paged_sparse
    return paged_sparse


def table(lens, page, g, width=None, spare=3):
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    total = sum(need) + spare
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    t = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, total


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- bounds ----

def bounds_case(PS, lens, new, page=16, hkv=2, hd=128, strided=False, seed=0, width=None, keys=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tab, total = table(lens, page, g, width)
    k = torch.randn(total, hkv, page, hd, device="cuda", generator=g).to(BF16)
    if strided:
        k = torch.randn(total, page, hkv, 2 * hd, device="cuda", generator=g).to(BF16)[..., hd:].transpose(1, 2)
    if keys:
        keys(k)
    b = torch.randn(total, hkv, 2, hd, device="cuda", generator=g).to(BF16)
    want = b.clone()
    for i, (n, a) in enumerate(zip(lens, new)):
        for blk in range(max(n - a, 0) // page, -(-n // page) if a else 0):
            pg = tab[i, blk].item()
            rows = k[pg, :, :min(page, n - blk * page)].double()
            want[pg, :, 0], want[pg, :, 1] = rows.amin(1), rows.amax(1)
    cu = None if new == [1] * len(lens) and seed % 2 == 0 else ints([sum(new[:i]) for i in range(len(new) + 1)])
    PS.update_page_bounds(k, b, tab, ints(lens), cu_seqlens=cu)
    torch.cuda.synchronize()
    assert torch.equal(b.nan_to_num(-12345.0), want.nan_to_num(-12345.0))


@pytest.mark.parametrize("n", [1, 15, 16, 17, 100, 1000])
@pytest.mark.parametrize("new", [1, 0, 5, 16, 17, 1000])
def test_bounds_lengths(PS, n, new):
    bounds_case(PS, [n], [min(n, new)], seed=n + new)


@pytest.mark.parametrize("seed", [0, 1])
def test_bounds_ragged(PS, seed):
    bounds_case(PS, [5, 0, 300, 16, 33, 32], [1, 0, 300, 16, 1, 2], seed=seed)
    bounds_case(PS, [5, 1, 300, 16, 33, 32] * 20, [1] * 120, seed=seed)
    bounds_case(PS, [1, 1, 1], [1, 1, 1], width=5000, seed=seed)


@pytest.mark.parametrize("hd,page,strided", [(64, 16, False), (8, 3, False), (96, 24, True), (256, 64, False), (72, 5, False), (7, 16, False), (300, 16, True),
                                             (128, 1, True), (128, 256, False)])
def test_bounds_rows(PS, hd, page, strided):
    bounds_case(PS, [90, 200, 41], [50, 200, 1], hd=hd, page=page, strided=strided, seed=hd)


@pytest.mark.parametrize("hd", [64, 20])
def test_bounds_odd_values(PS, hd):
    def keys(k):
        k[:, 0, 1::3, 0], k[:, 0, 2::5, 1], k[:, 1, ::4, 2], k[:, 1, :, 3] = float("nan"), float("inf"), -float("inf"), 1e-39
    bounds_case(PS, [90, 17], [50, 17], hd=hd, keys=keys)


def test_bounds_bad_pages(PS, cuda_lib):
    k = torch.ones(3, 1, 16, 64, device="cuda", dtype=BF16)
    b = torch.zeros(3, 1, 2, 64, device="cuda", dtype=BF16)
    assert cuda_lib.sn_device_status(1, None) == 0
    for tab, n, new in (([[0, 7]], 20, 4), ([[0, -1]], 20, 20), ([[1, 2]], 99, 1), ([[1, 2]], -4, 3)):
        PS.update_page_bounds(k, b, ints(tab), ints([n]), cu_seqlens=ints([0, new]))
        torch.cuda.synchronize()
        assert cuda_lib.sn_device_status(1, None) == -1, (tab, n)


# ---- choice ----

def select_truth(q, bounds, tab, lens, page, count, first, last):
    B, hq, hd = q.shape
    hkv = bounds.shape[1]
    out = torch.full((B, hkv, count), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        nb = -(-n // page)
        if nb == 0:
            continue
        lo, hi = bounds[tab[b, :nb].long()].double().unbind(2)  # [nb, hkv, hd]
        qd = q[b].view(hkv, hq // hkv, hd).double()
        score = torch.maximum(lo[:, :, None] * qd, hi[:, :, None] * qd).sum(-1).amax(-1)  # [nb, hkv]
        score[~(torch.isfinite(lo) & torch.isfinite(hi)).all(-1)] = float("inf")
        for h in range(hkv):
            s = score[:, h].clone()
            s[:first] = s[nb - last if last else nb:] = float("inf")
            forced = set(range(min(first, nb))) | set(range(max(nb - last, 0), nb))
            free = sorted((i for i in range(nb) if i not in forced), key=lambda i, v=score[:, h].tolist(): (-v[i], i))
            got = sorted(forced | set(free[:count - len(forced)])) if nb > count else list(range(nb))
            out[b, h, :len(got)] = ints(got)
    return out


def select_case(PS, lens, count, first=1, last=1, hq=16, hkv=4, hd=128, page=16, seed=0, width=None, make=None, strided=False, unaligned=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tab, total = table(lens, page, g, width)
    a, c = (torch.randn(total, hkv, hd, device="cuda", generator=g) for _ in range(2))
    bounds = torch.stack([torch.minimum(a, c), torch.maximum(a, c)], 2).to(BF16)
    if unaligned:
        flat = torch.empty(bounds.numel() + 1, device="cuda", dtype=BF16)
        flat[1:] = bounds.flatten()
        bounds = flat[1:].view(bounds.shape)
    q = torch.randn(len(lens), hq, hd, device="cuda", generator=g).to(BF16)
    if strided:
        q = torch.randn(len(lens), hq + 3, 2 * hd, device="cuda", generator=g).to(BF16)[:, 1:hq + 1, hd:]
    if make:
        make(q, bounds, tab)
    got = PS.select_blocks(q, bounds, tab, ints(lens), page, count, first=first, last=last)
    torch.cuda.synchronize()
    assert torch.equal(got, select_truth(q, bounds, tab, lens, page, count, first, last))
    return got


@pytest.mark.parametrize("blocks", [1, 2, 3, 8, 31, 33, 64, 100, 513, 2000])
@pytest.mark.parametrize("count", [1, 2, 7, 32, 100])
def test_select_lengths(PS, blocks, count):
    select_case(PS, [16 * blocks - 3], count, min(1, count - 1), 1, seed=blocks + count)


@pytest.mark.parametrize("first,last,count", [(0, 0, 5), (0, 1, 1), (1, 0, 1), (5, 5, 10), (0, 10, 10), (3, 0, 40), (2, 3, 40)])
def test_select_windows(PS, first, last, count):
    select_case(PS, [16 * 11, 16 * 10, 16 * 9 + 1, 640, 1000, 0, 1], count, first, last, seed=count)


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (16, 1), (24, 2), (6, 2), (5, 1), (33, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_select_heads(PS, hq, hkv, hd):
    select_case(PS, [1600, 700], 20, hq=hq, hkv=hkv, hd=hd, seed=hq)


@pytest.mark.parametrize("hd", [1, 2, 7, 8, 20, 40, 72, 96, 160, 256, 300, 512])
def test_select_head_dims(PS, hd):
    select_case(PS, [1600, 700], 20, hd=hd, seed=hd)


def test_select_layouts(PS):
    select_case(PS, [1600, 700], 20, strided=True)
    select_case(PS, [1600, 700], 20, unaligned=True)
    select_case(PS, [1600, 700, 0], 20, width=20000)
    select_case(PS, [100001], 128, 1, 4, hkv=1, hq=4)
    select_case(PS, [4003] * 90, 40, 1, 4)
    select_case(PS, [20000], 3000, 1, 4, hkv=1, hq=1, hd=8, page=4)
    select_case(PS, [40, 3], 4, page=7)


@pytest.mark.parametrize("kind", ["same", "zero", "few", "tiny", "huge", "special"])
def test_select_ties_and_odd_values(PS, kind):
    def make(q, bounds, tab):
        if kind == "same":
            bounds.copy_(bounds[:1].clone().expand_as(bounds))
        if kind == "zero":
            q.zero_()
            q[:, ::2] = -0.0
        if kind == "few":  # three kinds of pages
            bounds.copy_(bounds[:3].clone().repeat(-(-len(bounds) // 3), 1, 1, 1)[:len(bounds)])
        if kind == "tiny":  # subnormal bounds and queries
            bounds.copy_((bounds.float() * 1e-39).to(BF16))
            q.copy_((q.float() * 1e-38).to(BF16))
        if kind == "huge":
            bounds.copy_((bounds.float() * 1e38).clamp(-3e38, 3e38).to(BF16))
            q.copy_((q.float() * 1e38).clamp(-3e38, 3e38).to(BF16))
        if kind == "special":
            bounds[3::9, 0, 0, 5], bounds[4::11, 1, 1, 6], bounds[5::13, 1, 0, 0] = float("nan"), float("inf"), -float("inf")
            q[:, :, 5] = 0
    select_case(PS, [16 * 500, 16 * 70], 40, 1, 2, hq=8, hkv=2, make=make, seed=3)


def test_select_near_ties(PS):
    """Scores that differ in the 30th bit."""
    def make(q, bounds, tab):
        q.zero_()
        q[:, :, 0] = 1
        q[:, :, 1] = 2.0 ** -30
        bounds[..., 0] = 1.0
        lo = torch.arange(len(bounds), device="cuda").flip(0)[:, None, None] % 128
        bounds[..., 1] = lo.to(BF16)
    select_case(PS, [16 * 120], 30, 0, 0, make=make, seed=4)


def test_select_bad_pages(PS, cuda_lib):
    q = torch.ones(1, 2, 64, device="cuda", dtype=BF16)
    b = torch.zeros(8, 1, 2, 64, device="cuda", dtype=BF16)
    assert cuda_lib.sn_device_status(1, None) == 0
    got = PS.select_blocks(q, b, ints([[0, 1, -1, 99, 4, 5]]), ints([96]), 16, 3)
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1 and got.tolist() == [[[0, 1, 5]]]
    PS.select_blocks(q, b, ints([[0, 1, 2]]), ints([10000]), 16, 3)
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1


# ---- attention over the listed blocks ----

def sparse_truth(q, kp, vp, tab, lens, blocks, scale):
    B, hq, hd = q.shape
    hkv, page, G = kp.shape[1], kp.shape[2], q.shape[1] // kp.shape[1]
    o = torch.zeros(B, hq, hd, device="cuda", dtype=torch.float64)
    bound, lse = torch.zeros_like(o), torch.full((B, hq), -float("inf"), device="cuda", dtype=torch.float64)
    for b, n in enumerate(lens):
        for h in range(hkv):
            at = [t for e in blocks[b, h, :-(-n // page)].tolist() if e >= 0 for t in range(e * page, min(e * page + page, n))]
            if not at:
                continue
            t = torch.tensor(at, device="cuda")
            pg = tab[b].long()[t // page]
            k, v = kp[pg, h, t % page].double(), vp[pg, h, t % page].double()
            qd = q[b, h * G:(h + 1) * G].double()
            s, sa = qd @ k.T * scale, (qd.abs() @ k.abs().T).amax(1) * abs(scale)
            p = torch.softmax(s, 1)
            rows = slice(h * G, (h + 1) * G)
            lse[b, rows], o[b, rows] = torch.logsumexp(s, 1), p @ v
            P = p @ v.abs()
            bound[b, rows] = E * (o[b, rows].abs() + P) + (2 * (hd + 4) * 2.0 ** -24 * sa[:, None] + 2.0 ** -19) * P
    return o, bound, lse


def sparse_case(PS, lens, count, hq=16, hkv=4, hd=128, page=16, seed=0, order="up", strided=False, workspace=None, scale=None, blocks=None, width=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    tab, total = table(lens, page, g, width)
    kp, vp, q = r(total, hkv, page, hd), r(total, hkv, page, hd), r(len(lens), hq, hd)
    if strided:
        kp = r(total, page, hkv, 2 * hd)[..., :hd].transpose(1, 2)
        vp = r(total, page, hkv, 2 * hd)[..., hd:].transpose(1, 2)
        q = r(len(lens), hq + 2 * hkv, hd)[:, :hq]
    if blocks is None:
        blocks = torch.full((len(lens), hkv, count), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(lens):
            nb = -(-n // page)
            for h in range(hkv):
                pick = torch.randperm(nb, device="cuda", generator=g)[:count]
                blocks[b, h, :len(pick)] = pick.sort().values if order == "up" else pick
    o, bound, lse = sparse_truth(q, kp, vp, tab, lens, blocks, hd ** -0.5 if scale is None else scale)
    got, glse = PS.paged_sparse_attention(q, kp, vp, tab, ints(lens), blocks, scale=scale, workspace=workspace, return_lse=True)
    torch.cuda.synchronize()
    err = (got.double() - o).abs()
    assert (err <= bound + 1e-30).all(), (err - bound).max().item()
    some = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(glse), some) and ((glse.double() - lse).abs()[some] <= 5e-5).all()
    return got, q, kp, vp, tab


@pytest.mark.parametrize("n", [1, 16, 17, 100, 1000, 5000])
@pytest.mark.parametrize("count", [1, 5, 64, 200])
def test_sparse_lengths(PS, n, count):
    sparse_case(PS, [n], count, seed=n + count)


@pytest.mark.parametrize("lens", [[0], [0, 5, 0, 300, 1, 0], [1] * 40, [3000, 1, 17, 0, 999], list(range(0, 3300, 50)), [100001, 30000]])
def test_sparse_ragged(PS, lens):
    sparse_case(PS, lens, 24, seed=len(lens))
    sparse_case(PS, lens, 130, order="any", seed=len(lens))


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (16, 1), (24, 1), (6, 2), (40, 2), (5, 1)])
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_sparse_heads(PS, hq, hkv, hd):
    sparse_case(PS, [700, 177], 9, hq=hq, hkv=hkv, hd=hd, seed=hq)


@pytest.mark.parametrize("hd,page", [(8, 16), (256, 16), (128, 1), (128, 24), (64, 48), (128, 128), (128, 100), (64, 256)])
def test_sparse_pages(PS, hd, page):
    sparse_case(PS, [1500, 1, 77], 5, hd=hd, page=page, order="any", seed=hd + page)


def test_sparse_layouts(PS):
    from sonata_b200.kernels import paged_kv as PK
    ws = PK.decode_workspace(3, 16, 128)
    for _ in range(2):
        sparse_case(PS, [1500, 1, 77], 30, strided=True, workspace=ws)
    sparse_case(PS, [1500, 1, 77], 30, hd=96, strided=True)
    sparse_case(PS, [1500], 30, scale=-0.3)
    sparse_case(PS, [1500, 3], 30, width=3000)


@pytest.mark.parametrize("hd", [128, 80])
def test_sparse_odd_lists(PS, hd):
    """Gaps, blocks past the end, the same block twice, lists with nothing in them."""
    n = -7
    rows = [[[3, n, 1, 0, n, 2], [9, 9, 9, 1 << 30, 4, 0], [n, n, n, n, n, n], [5, 5, 1, 50, 0, 7]],
            [[0, 1, n, n, n, n], [1, 0, 5, 5, 5, 5], [n, 0, 3, 3, 3, 3], [2, 2, 2, 2, 2, 2]]]
    got, *_ = sparse_case(PS, [150, 18], 6, hd=hd, blocks=ints(rows))
    assert not got[0, 8:12].any() and not got[1, 12:].any()


def test_sparse_all_blocks_is_attention(PS):
    from sonata_b200.kernels import paged_kv as PK
    lens = [700, 33, 0, 1000]
    blocks = torch.arange(63, device="cuda", dtype=torch.int32).expand(4, 4, 63).contiguous()
    got, q, kp, vp, tab = sparse_case(PS, lens, 63, blocks=blocks)
    _, bound, _ = sparse_truth(q, kp, vp, tab, lens, blocks, 128 ** -0.5)
    # both are within the bound of the same sums, whatever pieces they are cut into: within twice the bound of one another
    d = (got.double() - PK.paged_decode_attention(q, kp, vp, tab, ints(lens)).double()).abs()
    assert (d <= 2 * bound).all()


@pytest.mark.parametrize("lens,hkv,count", [
    ([16] * 45 + [20000, 300, 20000], 2, 1000),  # over 32 streams, with somewhat larger shares
    ([3000] + [9] * 142 + [2500], 4, 150),            # more pieces than CTAs
    ([40] * 300 + [6400, 0, 6400], 4, 400),      # more (stream, head)s than partial results have places for
])
def test_sparse_cuts(PS, lens, hkv, count):
    from sonata_b200 import _lib
    from sonata_b200.kernels import paged_kv as PK
    ws = PK.decode_workspace(len(lens), 2 * hkv, 64)
    runs = [sparse_case(PS, lens, count, hq=2 * hkv, hkv=hkv, hd=64, workspace=ws, seed=count)[0] for _ in range(2)]
    assert torch.equal(*runs)
    counters = ws[:4 * _lib.SN_PAGED_DECODE_COUNTERS].view(torch.int32)
    assert not counters.any()  # ready for the next call


def test_sparse_bad_pages(PS, cuda_lib):
    g = torch.Generator(device="cuda").manual_seed(0)
    kp, vp = (torch.randn(4, 1, 16, 64, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(1, 2, 64, device="cuda", generator=g).to(BF16)
    assert cuda_lib.sn_device_status(1, None) == 0
    got = PS.paged_sparse_attention(q, kp, vp, ints([[0, 9, 2, 3]]), ints([60]), ints([[[0, 1, 3]]]))
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1
    assert torch.equal(got, PS.paged_sparse_attention(q, kp, vp, ints([[0, 1, 2, 3]]), ints([60]), ints([[[0, -1, 3]]])))


# ---- together ----

def test_a_run_of_steps(PS, cuda_lib):
    """Append, bounds, choice, attention over 40 steps of ragged streams, in one captured graph from the second step on: bounds
    equal those of all keys, choices equal the plain ones, outputs within the attention's bound."""
    from sonata_b200.kernels import paged_kv as PK
    g = torch.Generator(device="cuda").manual_seed(5)
    lens = [300, 15, 16, 999]
    cache = PK.PagedKVCache(1, 120, 2, 64, 4, 70)
    cos, sin = PK.rotary_table(1100, 64)
    bounds, ws = PS.page_bounds(cache.k(0)), PK.decode_workspace(4, 8, 64)
    cache.reserve(lens)
    cu = ints([0, 300, 315, 331, 1330])
    PK.rotary_paged_append(torch.randn(1330, 12 * 64, device="cuda", generator=g).to(BF16), cache.k(0), cache.v(0), cache.page_table,
                           cache.seq_lens, cos, sin, 8, cu_seqlens=cu)
    PS.update_page_bounds(cache.k(0), bounds, cache.page_table, cache.seq_lens, cu_seqlens=cu)
    qkv = torch.empty(4, 12 * 64, device="cuda", dtype=BF16)

    def step():
        q = PK.rotary_paged_append(qkv, cache.k(0), cache.v(0), cache.page_table, cache.seq_lens, cos, sin, 8)
        PS.update_page_bounds(cache.k(0), bounds, cache.page_table, cache.seq_lens)
        blocks = PS.select_blocks(q, bounds, cache.page_table, cache.seq_lens, 16, 12, first=1, last=2)
        return q, blocks, PS.paged_sparse_attention(q, cache.k(0), cache.v(0), cache.page_table, cache.seq_lens, blocks, workspace=ws)

    graph = None
    for i in range(40):
        cache.reserve([1] * 4)
        qkv.copy_(torch.randn(4, 12 * 64, device="cuda", generator=g))
        if i == 0:
            q, blocks, o = step()
        elif graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                q, blocks, o = step()
        if graph:
            graph.replay()
        torch.cuda.synchronize()
        if i % 13 == 0 or i == 39:
            for s, n in enumerate(cache.lens):
                for blk, pg in enumerate(cache.pages[s]):
                    k = cache.k(0)[pg, :, :min(16, n - 16 * blk)]
                    assert torch.equal(bounds[pg], torch.stack([k.amin(1), k.amax(1)], 1))
            assert torch.equal(blocks, select_truth(q, bounds, cache.page_table, cache.lens, 16, 12, 1, 2))
            want, bound, _ = sparse_truth(q, cache.k(0), cache.v(0), cache.page_table, cache.lens, blocks, 64 ** -0.5)
            assert ((o.double() - want).abs() <= bound + 1e-30).all()
    assert cuda_lib.sn_device_status(1, None) == 0


def test_refusals(PS):
    k = torch.zeros(4, 2, 16, 64, device="cuda", dtype=BF16)
    b, tab, lens, cu = PS.page_bounds(k), ints([[0, 1]]), ints([20]), ints([0, 3])
    assert b.shape == (4, 2, 2, 64)
    ok = dict(k_pages=k, bounds=b, page_table=tab, seq_lens=lens, cu_seqlens=cu)
    PS.update_page_bounds(**ok)
    for bad in (dict(k_pages=k.float()), dict(bounds=b[:3]), dict(bounds=b.float()), dict(bounds=b[..., :32]), dict(bounds=b[:, :1]),
                dict(page_table=tab.long()), dict(seq_lens=ints([1, 2])), dict(cu_seqlens=ints([0])), dict(cu_seqlens=cu.long()),
                dict(k_pages=k.cpu()), dict(k_pages=k.transpose(2, 3)), dict(bounds=b.transpose(1, 2)), dict(cu_seqlens=cu.cpu())):
        with pytest.raises((TypeError, ValueError)):
            PS.update_page_bounds(**{**ok, **bad})
    q = torch.zeros(1, 4, 64, device="cuda", dtype=BF16)
    ok = dict(q=q, bounds=b, page_table=tab, seq_lens=lens, page_size=16, count=4)
    PS.select_blocks(**ok)
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(bounds=b[..., 0]), dict(page_size=0), dict(count=0),
                dict(count=1), dict(first=-1), dict(last=-1), dict(first=2, last=3), dict(seq_lens=lens.long()), dict(q=q.expand(2, 4, 64)),
                dict(q=q.cpu())):
        with pytest.raises((TypeError, ValueError)):
            PS.select_blocks(**{**ok, **bad})
    blocks = torch.zeros(1, 2, 3, device="cuda", dtype=torch.int32)
    ok = dict(q=q, k_pages=k, v_pages=k, page_table=tab, seq_lens=lens, blocks=blocks)
    PS.paged_sparse_attention(**ok)
    for bad in (dict(blocks=blocks.long()), dict(blocks=blocks[:, :1]), dict(blocks=blocks[..., :0]), dict(blocks=blocks[..., ::2]), dict(blocks=None),
                dict(blocks=blocks.cpu()), dict(q=q[:, :3]), dict(k_pages=None), dict(page_table=None),
                dict(workspace=torch.zeros(64, device="cuda", dtype=torch.uint8))):
        with pytest.raises((TypeError, ValueError)):
            PS.paged_sparse_attention(**{**ok, **bad})


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["subnormal bounds", "subnormal queries", "cancelling", "border"])
def test_select_where_32_bits_are_not_enough(PS, hd, kind):
    """Bounds or queries below 2^-126 that the sums still depend on, sums whose large terms cancel, and a border at which many
    blocks differ in bits that only 64 hold (more of them than are ranked by comparing all)."""
    def make(q, bounds, tab):
        if kind == "subnormal bounds":
            bounds.copy_((bounds.float() * 1e-39).to(BF16))
            q.copy_((q.float() * 1e37).to(BF16))
        if kind == "subnormal queries":
            bounds.copy_((bounds.float() * 1e37).to(BF16))
            q.copy_((q.float() * 1e-39).to(BF16))
        if kind == "cancelling":
            q[..., 0], q[..., 1] = 1.0, 1.0
            bounds[..., 0] = 2.0 ** 40
            bounds[..., 1] = -2.0 ** 40
        if kind == "border":
            q.fill_(1.0)
            bounds.fill_(1.0)
            n = torch.arange(len(bounds), device="cuda")
            bounds[..., 5] = (2.0 ** -20 * (1 + n % 64))[:, None, None].to(BF16)
            bounds[..., 6] = (2.0 ** -40 * (1 + n * 37 % 101))[:, None, None].to(BF16)
    select_case(PS, [16 * 900, 16 * 130], 90, 1, 2, hq=8, hkv=2, hd=hd, make=make, seed=11)
    select_case(PS, [16 * 6000], 400, 1, 2, hq=4, hkv=1, hd=hd, make=make, seed=12)


@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("odd", [1, 7, 30, 60, 300])
def test_select_with_blocks_that_have_no_score(PS, hd, odd):
    """Blocks with an infinity or a NaN in their bounds, and blocks whose sums overflow 32 bits (on either side), among others:
    fewer and more of them than are wanted."""
    def make(q, bounds, tab):
        g = torch.Generator(device="cuda").manual_seed(odd)
        at = torch.randperm(len(bounds), device="cuda", generator=g)[:odd]
        for i, pg in enumerate(at.tolist()):
            if i % 3 == 0:
                bounds[pg, 0, i % 2, i % hd] = [float("inf"), float("nan"), -float("inf")][i // 3 % 3]
            else:  # finite, but not in 32 bits
                bounds[pg, i % 2, :, :] = (bounds[pg, i % 2].float().sign() * 3e38).to(BF16)
    select_case(PS, [16 * 400, 16 * 90], 40, 1, 2, hq=8, hkv=2, hd=hd, make=make, seed=odd)


@pytest.mark.parametrize("hd", [64, 128, 96, 40])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("hq,nb", [(2, 40), (8, 40), (10, 40), (8, 500), (24, 500)])
def test_select_with_a_query_that_is_not_finite(PS, hd, value, hq, nb):
    """All blocks of its key/value head rank alike, whatever number of them is compared: the lowest ones are listed."""
    def make(q, bounds, tab):
        q[0, hq // 2 - 1, hd // 2] = value
        bounds[::5, 0, :, hd // 2] = 0.0

    g = torch.Generator(device="cuda").manual_seed(hd)
    tab, total = table([16 * nb, 16 * nb - 3], 16, g)
    a, c = (torch.randn(total, 2, hd, device="cuda", generator=g) for _ in range(2))
    bounds = torch.stack([torch.minimum(a, c), torch.maximum(a, c)], 2).to(BF16)
    q = torch.randn(2, hq, hd, device="cuda", generator=g).to(BF16)
    make(q, bounds, tab)
    lens = [16 * nb, 16 * nb - 3]
    got = PS.select_blocks(q, bounds, tab, ints(lens), 16, 12, first=1, last=2)
    want = select_truth(q, bounds, tab, lens, 16, 12, 1, 2)
    want[0, 0] = ints([*range(10), nb - 2, nb - 1])
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("hd", [64, 128, 96, 40])
@pytest.mark.parametrize("nb,count,group", [(50, 20, 2), (300, 100, 2), (1500, 700, 2), (300, 100, 1), (50, 20, 7), (300, 100, 7), (300, 100, 16)])
def test_select_where_64_bits_round(PS, hd, nb, count, group):
    """Sums whose terms span more than 53 bits: each block has the same terms at other places, so that only the rounding of the
    sums tells them apart, and it is that of one order whatever number of blocks is compared: elements d mod 32, then those sums
    in pairs of neighbours."""
    g = torch.Generator(device="cuda").manual_seed(nb + hd)
    terms = torch.randn(hd, device="cuda", generator=g) * 2.0 ** torch.randint(0, 70, (hd,), device="cuda", generator=g)
    place = torch.rand(nb, 2, hd, device="cuda", generator=g).argsort(-1)
    bounds = terms.to(BF16)[place][:, :, None].expand(-1, -1, 2, -1).contiguous()
    q = torch.tensor([1.0, -2.0, 0.5, -1.0], device="cuda").repeat(group)[:2 * group].to(BF16).view(1, -1, 1).expand(1, -1, hd).contiguous()
    x = bounds[:, :, 0].double()[:, :, None] * q.view(2, group, hd).double()  # [nb, hkv, group, hd]
    x = torch.nn.functional.pad(x, (0, -hd % 32)).unflatten(-1, (-1, 32))
    s = torch.zeros_like(x[..., 0, :])
    for i in range(x.shape[-2]):
        s = s + x[..., i, :]
    for _ in range(5):
        s = s[..., ::2] + s[..., 1::2]
    score = s[..., 0].amax(-1)
    assert score[:, 0].unique().numel() > 2  # the order does matter
    tab = torch.arange(nb, device="cuda", dtype=torch.int32)[None]
    got = PS.select_blocks(q, bounds, tab, ints([16 * nb]), 16, count, first=0, last=0)
    for h in range(2):
        v = score[:, h].tolist()
        assert got[0, h].tolist() == sorted(sorted(range(nb), key=lambda i: (-v[i], i))[:count])


def test_sparse_page_of_nearly_2_31_positions(PS):
    """A page so long that its size and a length do not add up in 32 bits: the same bits as with a short one."""
    page, n = 2**31 - 256, 1000
    g = torch.Generator(device="cuda").manual_seed(1)
    q, rows = (torch.randn(s, device="cuda", generator=g).to(BF16) for s in ((1, 2, 1), (1, 1, n, 1)))
    k = torch.empty(1, 1, page, 1, device="cuda", dtype=BF16)
    k[:, :, :n] = rows
    tab, lens, blocks = ints([[0]]), ints([n]), ints([[[0]]])
    got = PS.paged_sparse_attention(q, k, k, tab, lens, blocks, return_lse=True)
    want = PS.paged_sparse_attention(q, rows, rows, tab, lens, blocks, return_lse=True)
    torch.cuda.synchronize()
    assert want[0].ne(0).any() and all(torch.equal(a, b) for a, b in zip(got, want))
