"""Attention that adds up weights, and eviction by them, against plain implementations.

Mass, in 64 bits: a score is off by E_s = (head_dim + 4) 2^-24 of its absolute terms, so a weight by 2 E_s of itself, by
2^-19 for exponentials, sums and joins (as the attention's), by 4 * 2^-24 |lse| for the two changes of base of lse; the
additions to the mass round (group + 1) times at 2^-24.  Eviction moves values and adds nothing: all bits are equal.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -8
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def PE(cuda_lib):
    from sonata_b200.kernels import paged_evict
    return paged_evict


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


def mass_truth(q, kp, vp, tab, lens, mass, scale):
    """(o, its bound, mass, its bound) in 64 bits."""
    B, hq, hd = q.shape
    hkv = kp.shape[1]
    G = hq // hkv
    o = torch.zeros(B, hq, hd, device="cuda", dtype=torch.float64)
    ob, want = torch.zeros_like(o), mass.double()
    mb = 2.0 ** -24 * (G + 1) * want.abs()
    for b, n in enumerate(lens):
        if n == 0:
            mb[b] = 0
            continue
        mb[b, :, n:] = 0
        pg = tab[b, : -(-n // kp.shape[2])].long()
        k, v = (t[pg].transpose(1, 2).reshape(-1, hkv, hd)[:n].double().repeat_interleave(G, 1) for t in (kp, vp))
        qd = q[b].double()
        s = torch.einsum("hd,nhd->hn", qd, k) * scale
        sa = torch.einsum("hd,nhd->hn", qd.abs(), k.abs()).amax(1) * abs(scale)
        p, lse = torch.softmax(s, 1), torch.logsumexp(s, 1)
        rel = 2 * (hd + 4) * 2.0 ** -24 * sa + 2.0 ** -19
        o[b] = torch.einsum("hn,nhd->hd", p, v)
        P = torch.einsum("hn,nhd->hd", p, v.abs())
        ob[b] = E * (o[b].abs() + P) + rel[:, None] * P
        want[b, :, :n] += p.view(hkv, G, n).sum(1)
        mb[b, :, :n] += (p * (rel + 4 * 2.0 ** -24 * lse.abs() + (G + 1) * 2.0 ** -24)[:, None]).view(hkv, G, n).sum(1)
    return o, ob, want, mb


def mass_case(PE, lens, hq=16, hkv=4, hd=128, page=16, seed=0, scale=None, strided=False, qscale=1.5, workspace=None, calls=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    tab, total = table(lens, page, g)
    kp, vp = r(total, hkv, page, hd), r(total, hkv, page, hd)
    q = (qscale * r(len(lens), hq, hd).float()).to(BF16)
    room = tab.shape[1] * page
    mass = torch.rand(len(lens), hkv, room, device="cuda", generator=g)
    if strided:
        kp = r(total, page, hkv, 2 * hd)[..., :hd].transpose(1, 2)
        vp = r(total, page, hkv, 2 * hd)[..., hd:].transpose(1, 2)
        q = r(len(lens), hq + 2 * hkv, hd)[:, :hq]
        mass = torch.rand(hkv, len(lens), room + 37, device="cuda", generator=g).transpose(0, 1)
    sc = hd ** -0.5 if scale is None else scale
    want = mass
    for _ in range(calls):
        o, ob, want, mb = mass_truth(q, kp, vp, tab, lens, mass, sc)
        before = mass.clone()
        got, lse = PE.paged_decode_attention_mass(q, kp, vp, tab, ints(lens), mass, scale=scale, workspace=workspace, return_lse=True)
        torch.cuda.synchronize()
        assert ((got.double() - o).abs() <= ob + 1e-30).all()
        err = (mass.double() - want).abs()
        assert (err <= mb + 1e-30).all(), (err - mb).max().item()
        for b, n in enumerate(lens):
            assert torch.equal(mass[b, :, n:], before[b, :, n:])
    from sonata_b200.kernels import paged_kv
    plain, plain_lse = paged_kv.paged_decode_attention(q, kp, vp, tab, ints(lens), scale=scale, return_lse=True)
    assert torch.equal(plain, got) and torch.equal(plain_lse, lse)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 255, 256, 257, 1000, 4097])
def test_mass_lengths(PE, n):
    mass_case(PE, [n], seed=n)


@pytest.mark.parametrize("lens", [[0], [0, 5, 0, 300, 1, 0], [1] * 40, [3000, 1, 17, 0, 999], list(range(0, 330, 5)), [20011, 9000]])
def test_mass_ragged(PE, lens):
    mass_case(PE, lens, seed=len(lens))


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1), (16, 1), (24, 1), (6, 2), (40, 2), (5, 1), (33, 1)])
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_mass_heads(PE, hq, hkv, hd):
    mass_case(PE, [300, 77], hq=hq, hkv=hkv, hd=hd, seed=hq)


@pytest.mark.parametrize("hd,page", [(8, 16), (256, 16), (128, 1), (128, 24), (64, 48), (128, 128), (128, 100)])
def test_mass_rows(PE, hd, page):
    mass_case(PE, [500, 1, 77], hd=hd, page=page, seed=hd + page)


@pytest.mark.parametrize("hd,page", [(128, 16), (96, 16)])
def test_mass_strides(PE, hd, page):
    mass_case(PE, [500, 1, 77], hd=hd, page=page, strided=True, seed=5)


def test_mass_scales_and_workspace(PE):
    ws = PE.mass_workspace(3, 16, 4, 128, 512)
    mass_case(PE, [500, 1, 77], workspace=ws, calls=2)
    mass_case(PE, [200, 33], workspace=ws, scale=-0.5, qscale=0.5)
    mass_case(PE, [200], scale=0.0, qscale=0.5)


@pytest.mark.parametrize("hd", [128, 80])
def test_mass_masked_places_and_empty_rows(PE, hd):
    """NaN behind a stream's end counts for nothing; a query head whose scores are all -inf gives zeros and adds nothing."""
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [21, 40]
    tab, total = table(lens, 16, g)
    kp, vp = (torch.randn(total, 2, 16, hd, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(2, 4, hd, device="cuda", generator=g).to(BF16)
    kp[tab[0, 1].item(), :, 5:] = vp[tab[0, 1].item(), :, 5:] = float("nan")
    q[1, 0] = 0
    q[1, 0, 3] = 1
    kp[tab[1, :3].long(), 0, :, 3] = -float("inf")
    q[1, 1, 3] = 1
    mass = torch.zeros(2, 2, 48, device="cuda")
    o = PE.paged_decode_attention_mass(q, kp, vp, tab, ints(lens), mass)
    torch.cuda.synchronize()
    assert torch.isfinite(o).all() and torch.isfinite(mass).all()
    assert not o[1, :2].any() and not mass[1, 0].any()
    assert ((mass.double().sum(-1) - torch.tensor([[2, 2], [0, 2]], device="cuda")).abs() <= 2.0 ** -18).all()


def test_mass_bad_pages(PE, cuda_lib):
    """Pages out of range are left out and reported; lengths past the table are cut to it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    kp, vp = (torch.randn(6, 2, 16, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(1, 4, 128, device="cuda", generator=g).to(BF16)
    assert cuda_lib.sn_device_status(1, None) == 0
    for tab, n in (([[0, 9, 2]], 40), ([[0, 1, 2]], 1000)):
        mass = torch.zeros(1, 2, 48, device="cuda")
        PE.paged_decode_attention_mass(q, kp, vp, ints(tab), ints([n]), mass)
        torch.cuda.synchronize()
        assert cuda_lib.sn_device_status(1, None) == -1
        assert ((mass.sum(-1) - 2).abs() <= 2.0 ** -18).all()
        if n == 40:
            assert not mass[:, :, 16:32].any()


# ---- eviction ----

def evict_truth(pool, tab, lens, mass, keep, recent, sinks):
    pool, mass = pool.clone(), mass.clone()
    layers, _, _, hkv, page, _ = pool.shape
    source = torch.full((layers, len(lens), hkv, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        if n <= keep:
            source[:, b, :, :n] = torch.arange(n)
            continue
        pos = torch.arange(n)
        pg, at = tab[b].cpu().long()[pos // page].cuda(), (pos % page).cuda()
        for layer in range(layers):
            for h in range(hkv):
                old = mass[layer, b, h, :n].cpu()
                free = list(range(sinks, n - recent))
                value = [float("inf") if v != v else v for v in old.tolist()]
                nan = [v != v for v in old.tolist()]
                kept = sorted(free, key=lambda i: (not nan[i], -value[i], i))[:keep - recent - sinks]
                stay = set(i for i in kept if i < keep - recent)
                move = sorted(i for i in kept if i >= keep - recent)
                src = [i if i < sinks or i in stay else move.pop(0) for i in range(keep - recent)] + list(range(n - recent, n))
                assert not move
                s = torch.tensor(src, dtype=torch.long)
                for kv in range(2):
                    rows = pool[layer, kv, pg, h, at]
                    pool[layer, kv, pg[:keep], h, at[:keep]] = rows[s.cuda()]
                mass[layer, b, h, :keep] = old[s].cuda()
                mass[layer, b, h, keep:n] = 0
                source[layer, b, h] = s.int()
    return pool, mass, source.cuda()


def same(a, b):
    return torch.equal(a.nan_to_num(-12345.0), b.nan_to_num(-12345.0))


def evict_case(PE, lens, keep, recent=0, sinks=0, layers=1, hkv=2, hd=64, page=16, seed=0, mass=None, width=None, unaligned=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tab, total = table(lens, page, g, width=width)
    shape = (layers, 2, total, hkv, page, hd)
    n = torch.Size(shape).numel()
    pool = torch.randn(n + 1, device="cuda", generator=g).to(BF16)[1 if unaligned else 0:][:n].view(shape)
    room = tab.shape[1] * page
    if mass is None:  # some ties, zeros among them
        mass = torch.rand(layers, len(lens), hkv, room, device="cuda", generator=g)
        mass = torch.where(mass < 0.3, 0.0, (mass * 50).round() / 50)
    else:
        mass = mass(layers, len(lens), hkv, room, g)
    want = evict_truth(pool, tab, lens, mass, keep, recent, sinks)
    other, other_mass = pool.clone(), mass.clone()
    source = PE.evict_positions(pool, tab, ints(lens), mass, keep, recent=recent, sinks=sinks, return_source=True)
    torch.cuda.synchronize()
    assert torch.equal(source, want[2])
    assert torch.equal(pool, want[0])
    assert same(mass, want[1])
    assert PE.evict_positions(other, tab, ints(lens), other_mass, keep, recent=recent, sinks=sinks) is None
    assert torch.equal(other, want[0]) and same(other_mass, want[1])


@pytest.mark.parametrize("n,keep", [(2, 1), (3, 2), (17, 16), (33, 1), (64, 63), (65, 32), (300, 299), (300, 7), (1000, 500), (2112, 2048)])
@pytest.mark.parametrize("recent,sinks", [(0, 0), (1, 0), (0, 1)])
def test_evict_lengths(PE, n, keep, recent, sinks):
    if recent + sinks <= keep:
        evict_case(PE, [n], keep, recent, sinks, seed=n)


@pytest.mark.parametrize("keep,recent,sinks", [(100, 100, 0), (100, 60, 40), (100, 99, 0), (100, 0, 100), (100, 0, 99), (100, 30, 4), (250, 240, 3)])
def test_evict_windows(PE, keep, recent, sinks):
    """Recent positions that overlap their new places, and that do not; no candidates that stay."""
    evict_case(PE, [101, 130, 400, 251, 252, 100, 0], keep, recent, sinks, layers=2, seed=keep)


def test_evict_many_recent(PE):
    """More recent positions than a cluster holds at once, one step apart."""
    evict_case(PE, [6001, 6017], 6000, 5900, 4, hkv=1, seed=1)


@pytest.mark.parametrize("hd,page,unaligned", [(128, 16, False), (64, 1, False), (8, 3, False), (96, 24, False), (256, 64, False), (1024, 16, False),
                                               (7, 16, False), (300, 16, False), (128, 16, True), (1, 5, False)])
def test_evict_rows(PE, hd, page, unaligned):
    evict_case(PE, [90, 200, 41], 64, 20, 2, hd=hd, page=page, unaligned=unaligned, seed=hd)


@pytest.mark.parametrize("n,keep", [(9001, 4000), (30011, 4096), (30011, 29000)])
def test_evict_over_a_cluster(PE, n, keep):
    evict_case(PE, [n], keep, 100, 5, hkv=1, hd=8, page=64, seed=n)


@pytest.mark.parametrize("n,keep", [(49650, 30000), (49700, 1000), (60001, 50000), (200003, 100000), (70000, 69999)])
def test_evict_where_shared_memory_ends(PE, n, keep):
    """Keys that just fit into shared memory, and ever more that do not."""
    evict_case(PE, [n], keep, 130, 3, hkv=1, hd=2, page=64, seed=n)


@pytest.mark.parametrize("streams", [2, 40])
def test_evict_wide_table(PE, streams):
    """A table with room for far more positions than there are (and than shared memory holds keys of)."""
    evict_case(PE, [500, 100] * (streams // 2), 300, 10, 1, width=4000, hkv=4, hd=8, seed=3)


@pytest.mark.parametrize("seed", range(4))
def test_evict_narrow_and_wide_masses(PE, seed):
    """Masses in the last bits of one exponent, and over all exponents: one bin of the first histogram and all of them."""
    def mass(layers, B, hkv, room, g):
        u = torch.rand(layers, B, hkv, room, device="cuda", generator=g)
        if seed == 0:
            return 1 + (u * 64).round() * 2.0 ** -23
        if seed == 1:
            return 1 + (u * 2.0 ** 16).round() * 2.0 ** -23
        return torch.exp2(u * 250 - 125) * (1 if seed == 2 else -1)
    evict_case(PE, [200, 3000, 9000], 150, 20, 3, mass=mass, hd=8, seed=seed)


def test_evict_many_rows(PE):
    evict_case(PE, [40 + 3 * i for i in range(40)], 64, 16, 1, layers=3, hkv=4, hd=8, seed=4)


@pytest.mark.parametrize("kind", ["zero", "equal", "signs", "special"])
def test_evict_ties_and_odd_values(PE, kind):
    def mass(layers, B, hkv, room, g):
        m = torch.zeros(layers, B, hkv, room, device="cuda")
        if kind == "equal":
            m += 0.7
        if kind == "signs":
            m = torch.randn(layers, B, hkv, room, device="cuda", generator=g)
            m[..., ::3] = -0.0
            m[..., 1::3] = 0.0
        if kind == "special":
            m = torch.randn(layers, B, hkv, room, device="cuda", generator=g)
            m[..., 5::7], m[..., 6::11], m[..., 4::13], m[..., 3::17] = float("nan"), float("inf"), -float("inf"), 1e-42
        return m
    evict_case(PE, [200, 3000], 150, 20, 3, mass=mass, hd=8, seed=6)


@pytest.mark.parametrize("recent,sinks", [(0, 0), (64, 4), (65, 0), (128, 4), (129, 0), (256, 0)])
@pytest.mark.parametrize("layers,hkv", [(1, 1), (5, 8)])
def test_evict_few_and_many_moves(PE, layers, hkv, recent, sinks):
    """Streams over their budget by a few positions and by more than one CTA moves, of few rows and of many."""
    evict_case(PE, [601, 664, 640, 728, 800, 855, 856, 857, 1111, 1113, 1300, 600], 600, recent, sinks, layers=layers, hkv=hkv, hd=128, seed=recent)


def test_evict_strides_and_what_lies_behind(PE):
    """A mass with room behind the table's reach, by strides; places past a stream's end and other streams' pages as they were."""
    g = torch.Generator(device="cuda").manual_seed(7)
    lens = [130, 60, 200]
    tab, total = table(lens, 16, g)
    pool = torch.randn(2, 2, total, 2, 16, 64, device="cuda", generator=g).to(BF16)
    room = tab.shape[1] * 16
    whole = torch.rand(3, 2, 2, room + 9, device="cuda", generator=g)
    mass = whole.permute(1, 0, 2, 3)
    want = evict_truth(pool, tab, lens, mass, 100, 10, 1)
    PE.evict_positions(pool, tab, ints(lens), mass, 100, recent=10, sinks=1)
    torch.cuda.synchronize()
    assert torch.equal(pool, want[0]) and torch.equal(mass, want[1])


def test_evict_bad_pages_and_lengths(PE, cuda_lib):
    g = torch.Generator(device="cuda").manual_seed(8)
    pool = torch.randn(1, 2, 4, 1, 16, 64, device="cuda", generator=g).to(BF16)
    before = pool.clone()
    mass = torch.rand(1, 1, 1, 64, device="cuda", generator=g)
    assert cuda_lib.sn_device_status(1, None) == 0
    PE.evict_positions(pool, ints([[0, 99, -5, 1]]), ints([60]), mass, 32, recent=4)
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1
    assert torch.equal(pool[:, :, 2:], before[:, :, 2:])  # pages that the table does not name
    for n in (-3, 1000):  # nothing, and the whole table
        PE.evict_positions(pool, ints([[0, 1, 2, 3]]), ints([n]), mass, 32, recent=4)
        torch.cuda.synchronize()
        assert cuda_lib.sn_device_status(1, None) == -1


def test_evict_bad_pages_of_many_moves(PE, cuda_lib):
    g = torch.Generator(device="cuda").manual_seed(9)
    tab, total = table([1600], 16, g)
    pool = torch.randn(1, 2, total, 1, 16, 64, device="cuda", generator=g).to(BF16)
    mass = torch.rand(1, 1, 1, 1600, device="cuda", generator=g)
    want = evict_truth(pool, tab, [1600], mass, 512, 64, 0)
    hidden, seen = tab[0, 0].item(), tab[0, 31].item()  # a page that stays, the page of the newest places
    tab[0, 0] = total + 5
    before = pool.clone()
    assert cuda_lib.sn_device_status(1, None) == 0
    PE.evict_positions(pool, tab, ints([1600]), mass, 512, recent=64)
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1
    assert torch.equal(pool[:, :, hidden], before[:, :, hidden])
    assert torch.equal(pool[:, :, seen], want[0][:, :, seen])


def test_evict_twice_keeps_the_newest(PE):
    """Step after step: what was written last is what the last places hold, in order."""
    g = torch.Generator(device="cuda").manual_seed(9)
    tab = ints([[3, 0, 2, 1]])
    pool = torch.zeros(1, 2, 4, 1, 16, 8, device="cuda", dtype=BF16)
    mass = torch.zeros(1, 1, 1, 64, device="cuda")
    n = 0
    for t in range(300):
        pool[0, :, tab[0, n // 16], 0, n % 16] = t % 256
        n += 1
        mass[..., :n] += torch.rand(n, device="cuda", generator=g)
        if n > 50:
            PE.evict_positions(pool, tab, ints([n]), mass, 40, recent=20, sinks=2)
            n = 40
            rows = pool[0, 0, tab[0].long()].flatten(0, 2)[:40, 0].tolist()
            assert rows[20:] == [v % 256 for v in range(t - 19, t + 1)] and rows[:2] == [0, 1]
            assert (len(set(rows)) == 40 or t >= 256) and not mass[..., 40:].any()  # values repeat from 256 on


def test_refusals(PE):
    pool = torch.zeros(1, 2, 4, 2, 16, 64, device="cuda", dtype=BF16)
    tab, lens, mass = ints([[0, 1]]), ints([20]), torch.zeros(1, 1, 2, 32, device="cuda")
    ok = dict(pool=pool, page_table=tab, seq_lens=lens, mass=mass, keep=8)
    PE.evict_positions(**ok)
    for bad in (dict(pool=pool.float()), dict(pool=pool[0]), dict(pool=pool[:, :1]), dict(pool=pool.transpose(3, 4)), dict(pool=pool.cpu()),
                dict(page_table=tab.long()), dict(page_table=tab[0]), dict(seq_lens=ints([20, 20])), dict(mass=mass.double()),
                dict(mass=mass[..., :31]), dict(mass=mass[:, :, :1]), dict(mass=mass[0]), dict(keep=0), dict(keep=8, recent=9),
                dict(keep=8, recent=5, sinks=4), dict(keep=8, recent=-1), dict(keep=8, sinks=-1), dict(mass=mass.expand(1, 1, 2, 32)[..., ::2]),
                dict(mass=mass[:, :, :1].expand(1, 1, 2, 32))):
        with pytest.raises((TypeError, ValueError)):
            PE.evict_positions(**{**ok, **bad})
    q = torch.zeros(1, 4, 64, device="cuda", dtype=BF16)
    ok = dict(q=q, k_pages=pool[0, 0], v_pages=pool[0, 1], page_table=tab, seq_lens=lens, mass=mass[0])
    PE.paged_decode_attention_mass(**ok)
    for bad in (dict(mass=mass), dict(mass=mass[0].half()), dict(mass=mass[0, :, :1]), dict(mass=mass[0, ..., :31]), dict(q=q[:, :3]), dict(k_pages=1),
                dict(page_table=None), dict(workspace=torch.zeros(64, device="cuda", dtype=torch.uint8)),
                dict(workspace=PE.mass_workspace(1, 4, 2, 64, 31)), dict(mass=None), dict(mass=mass[0].cpu())):
        with pytest.raises((TypeError, ValueError)):
            PE.paged_decode_attention_mass(**{**ok, **bad})
    with pytest.raises(ValueError):
        PE.mass_workspace(1, 3, 2, 64, 16)


def test_streams_and_graphs(PE):
    """On another stream, and captured once for growing streams, both with one workspace."""
    g = torch.Generator(device="cuda").manual_seed(10)
    tab, total = table([64, 64], 16, g)
    pool = torch.randn(2, 2, total, 2, 16, 64, device="cuda", generator=g).to(BF16)
    q = torch.randn(2, 8, 64, device="cuda", generator=g).to(BF16)
    mass = torch.zeros(2, 2, 2, 64, device="cuda")
    lens, ws = ints([30, 50]), PE.mass_workspace(2, 8, 2, 64, 64)

    def step(stream=None):
        o = [PE.paged_decode_attention_mass(q, pool[i, 0], pool[i, 1], tab, lens, mass[i], workspace=ws, stream=stream) for i in range(2)]
        return o, PE.evict_positions(pool, tab, lens, mass, 40, recent=8, sinks=1, return_source=True, stream=stream)

    state = pool.clone(), mass.clone()

    def plain(a, b):
        pool.copy_(state[0]), mass.copy_(state[1]), lens.copy_(ints([a, b]))
        o, s = step()
        torch.cuda.synchronize()
        return [t.clone() for t in (*o, s, pool, mass)]

    want = {n: plain(*n) for n in ((30, 50), (64, 41))}
    pool.copy_(state[0]), mass.copy_(state[1]), lens.copy_(ints([30, 50]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    o, s = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((*o, s, pool, mass), want[30, 50]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = step()
    for n in ((30, 50), (64, 41), (30, 50)):
        pool.copy_(state[0]), mass.copy_(state[1]), lens.copy_(ints(n))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*o, s, pool, mass), want[n])), n


@pytest.mark.parametrize("interleaved,hd", [(False, 64), (True, 64), (False, 24)])
def test_append_with_positions(cuda_lib, interleaved, hd):
    """The rotary angle of `positions`, the place of seq_lens: the same bits as an append whose places are the positions."""
    from sonata_b200.kernels import paged_kv as PK
    g = torch.Generator(device="cuda").manual_seed(11)
    cos, sin = PK.rotary_table(200, hd)
    qkv = torch.randn(3, 8 * hd, device="cuda", generator=g).to(BF16)
    far, near = (torch.zeros(2, 16, 2, 16, hd, device="cuda", dtype=BF16) for _ in range(2))
    tab = torch.arange(16, device="cuda", dtype=torch.int32).view(1, 16)
    cu = ints([0, 3])
    q1 = PK.rotary_paged_append(qkv, far[0], far[1], tab, ints([150]), cos, sin, 4, cu_seqlens=cu, interleaved=interleaved)
    q2 = PK.rotary_paged_append(qkv, near[0], near[1], tab, ints([33]), cos, sin, 4, cu_seqlens=cu, interleaved=interleaved,
                                positions=ints([147, 148, 149]))
    torch.cuda.synchronize()
    at = lambda t, n: t[:, tab[0].long()].transpose(2, 3).flatten(1, 2)[:, n - 3:n]
    assert torch.equal(q1, q2) and torch.equal(at(far, 150), at(near, 33)) and near.count_nonzero() == far.count_nonzero()
    assert cuda_lib.sn_device_status(1, None) == 0
    q3 = PK.rotary_paged_append(qkv, near[0], near[1], tab, ints([33]), cos, sin, 4, cu_seqlens=cu, positions=ints([147, 200, -1]))
    torch.cuda.synchronize()
    assert cuda_lib.sn_device_status(1, None) == -1 and q3[0].any() and not q3[1:].any()
    for bad in (ints([1, 2]), torch.zeros(3, device="cuda"), ints([1, 2, 3]).cpu()):
        with pytest.raises((TypeError, ValueError)):
            PK.rotary_paged_append(qkv, near[0], near[1], tab, ints([33]), cos, sin, 4, cu_seqlens=cu, positions=bad)
