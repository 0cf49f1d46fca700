"""The paged KV cache's kernels against plain implementations in 64 bits.

Rotary: fp32 products and sums of bf16 values, rounded once to bf16: |err| <=
2^-8 |y| + 2^-22 (|x1| + |x2|).  Attention: the weights are rounded to bf16
once before the product with v, the output once: |err| <= 2^-8 (|o| + P) +
2 E_s P with P = sum_t p_t |v_t| and E_s the error of a score, (head_dim + 4)
2^-24 of its absolute terms, and 2^-19 for exponentials and joins.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -8  # half a unit in the last place of bf16 (8 significant bits)
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def PK(cuda_lib):
    from sonata_b200.kernels import paged_kv
    return paged_kv


def table(lens, page, seed, width=None, spare=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
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


def attend_truth(q, kp, vp, tab, lens, page, scale):
    """(o, bound, lse) in 64 bits."""
    B, hq, hd = q.shape
    hkv = kp.shape[1]
    o = torch.zeros(B, hq, hd, device="cuda", dtype=torch.float64)
    bound, lse = torch.zeros_like(o), torch.full((B, hq), -float("inf"), device="cuda", dtype=torch.float64)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pg = tab[b, : -(-n // page)].long()
        k = kp[pg].transpose(1, 2).reshape(-1, hkv, hd)[:n].double().repeat_interleave(hq // hkv, 1)
        v = vp[pg].transpose(1, 2).reshape(-1, hkv, hd)[:n].double().repeat_interleave(hq // hkv, 1)
        qd = q[b].double()
        s = torch.einsum("hd,nhd->hn", qd, k) * scale
        sa = torch.einsum("hd,nhd->hn", qd.abs(), k.abs()).amax(1) * abs(scale)
        p = torch.softmax(s, 1)
        lse[b] = torch.logsumexp(s, 1)
        o[b] = torch.einsum("hn,nhd->hd", p, v)
        P = torch.einsum("hn,nhd->hd", p, v.abs())
        bound[b] = E * (o[b].abs() + P) + (2 * (hd + 4) * 2.0 ** -24 * sa[:, None] + 2.0 ** -19) * P
    return o, bound, lse


def attend_case(PK, lens, hq=16, hkv=4, hd=128, page=16, seed=0, scale=None, qscale=1.5, strided=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    tab, total = table(lens, page, seed)
    kp, vp = r(total, hkv, page, hd), r(total, hkv, page, hd)
    q = (qscale * r(len(lens), hq, hd).float()).to(BF16)
    if strided:  # token-major pages inside wider rows, q inside a qkv row
        kp = r(total, page, hkv, 2 * hd)[..., :hd].transpose(1, 2)
        vp = r(total, page, hkv, 2 * hd)[..., hd:].transpose(1, 2)
        q = r(len(lens), hq + 2 * hkv, hd)[:, :hq]
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    sc = hd ** -0.5 if scale is None else scale
    o, bound, lse = attend_truth(q, kp, vp, tab, lens, page, sc)
    got, glse = PK.paged_decode_attention(q, kp, vp, tab, seq, scale=scale, return_lse=True)
    torch.cuda.synchronize()
    err = (got.double() - o).abs()
    assert (err <= bound + 1e-30).all(), (err - bound).max().item()
    some = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(glse), some)
    # the log of the sum: scores' errors (3e-5 for |s| < 100 here) and 2^-19
    assert ((glse.double() - lse).abs()[some] <= 5e-5).all()
    return got


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 257, 1000, 4097])
def test_attend_lengths(PK, n):
    attend_case(PK, [n], seed=n)


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [0, 5, 0, 300, 1, 0], [1] * 40, [3000, 1, 17, 0, 999], list(range(0, 330, 5))])
def test_attend_ragged(PK, lens):
    attend_case(PK, lens, seed=len(lens))


@pytest.mark.parametrize("hq,hkv", [(16, 4), (4, 4), (8, 1), (16, 1), (16, 2), (24, 1), (6, 2), (40, 2), (5, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_heads(PK, hq, hkv, hd):
    attend_case(PK, [300, 77], hq=hq, hkv=hkv, hd=hd, seed=hq)


@pytest.mark.parametrize("hd", [8, 32, 72, 80, 96, 160, 192, 256])
def test_attend_head_dims(PK, hd):
    attend_case(PK, [200, 33], hd=hd, seed=hd)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 48, 64, 128, 256, 1000])
def test_attend_page_sizes(PK, page):
    attend_case(PK, [500, 1, 77], page=page, seed=page)


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 32), (96, 16)])
def test_attend_strides(PK, hd, page):
    attend_case(PK, [500, 1, 77], hd=hd, page=page, strided=True, seed=5)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 0.01])
def test_attend_scales(PK, scale):
    attend_case(PK, [200], scale=scale, qscale=0.5, seed=6)


def test_attend_unaligned_base(PK):
    """A pool and a q that start off 16 bytes."""
    lens, hd = [100, 40], 128
    tab, total = table(lens, 16, 3)
    g = torch.Generator(device="cuda").manual_seed(3)
    raw = [torch.randn(n + 1, device="cuda", generator=g).to(BF16)[1:] for n in (total * 4 * 16 * hd,) * 2 + (2 * 16 * hd,)]
    kp, vp, q = raw[0].view(total, 4, 16, hd), raw[1].view(total, 4, 16, hd), raw[2].view(2, 16, hd)
    o, bound, _ = attend_truth(q, kp, vp, tab, lens, 16, hd ** -0.5)
    got = PK.paged_decode_attention(q, kp, vp, tab, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert ((got.double() - o).abs() <= bound).all()


@pytest.mark.parametrize("lens, hq, hkv, hd", [([20011], 16, 1, 128), ([20011], 1, 1, 64), ([13001, 0, 12345], 8, 1, 128),
                                              ([9999, 10001], 20, 2, 64)])
def test_attend_many_pieces(PK, lens, hq, hkv, hd):
    """Streams cut into more pieces than one CTA joins by itself."""
    attend_case(PK, lens, hq=hq, hkv=hkv, hd=hd, page=32, seed=7)


def test_attend_many_pieces_repeat(PK):
    """Joins in groups leave the workspace ready, and do not depend on who comes last."""
    ws = PK.decode_workspace(3, 16, 128)
    runs = []
    for lens in ([20000, 17, 15000], [300, 200, 100], [20000, 17, 15000], [64, 30000, 1]):
        tab, total = table(lens, 16, 9)
        gen = torch.Generator(device="cuda").manual_seed(10)
        kp, vp = (torch.randn(total, 1, 16, 128, device="cuda", generator=gen).to(BF16) for _ in range(2))
        q = torch.randn(3, 16, 128, device="cuda", generator=gen).to(BF16)
        seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
        runs.append([PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws) for _ in range(3)])
        o, bound, _ = attend_truth(q, kp, vp, tab, lens, 16, 128 ** -0.5)
        for got in runs[-1]:
            assert ((got.double() - o).abs() <= bound + 1e-30).all()
            assert torch.equal(got, runs[-1][0])
    assert torch.equal(runs[0][0], runs[2][0])


def test_attend_workspace_of_growing_calls(PK):
    """One workspace for calls of more and more streams, heads and head sizes, all of them cut over CTAs."""
    ws = PK.decode_workspace(40, 32, 128)
    for B, hq, hkv, hd in ((1, 4, 1, 64), (2, 16, 1, 64), (2, 16, 4, 128), (5, 32, 2, 128), (40, 32, 4, 128), (1, 4, 1, 64)):
        lens = [9000 // B + 61 * b + 1500 * (b == 0) for b in range(B)]
        tab, total = table(lens, 16, B)
        gen = torch.Generator(device="cuda").manual_seed(B)
        kp, vp = (torch.randn(total, hkv, 16, hd, device="cuda", generator=gen).to(BF16) for _ in range(2))
        q = torch.randn(B, hq, hd, device="cuda", generator=gen).to(BF16)
        seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
        o, bound, _ = attend_truth(q, kp, vp, tab, lens, 16, hd ** -0.5)
        for _ in range(2):
            got = PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws)
            assert ((got.double() - o).abs() <= bound + 1e-30).all()


def test_attend_long_split(PK):
    """One long stream, split over many CTAs and joined; the same bits every time, one workspace for all calls."""
    lens = [50001, 20000, 3]
    tab, total = table(lens, 64, 9)
    g = torch.Generator(device="cuda").manual_seed(9)
    kp, vp = (torch.randn(total, 4, 64, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(3, 16, 128, device="cuda", generator=g).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    o, bound, lse = attend_truth(q, kp, vp, tab, lens, 64, 128 ** -0.5)
    ws = PK.decode_workspace(3, 16, 128)
    first = PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws)
    for _ in range(20):
        again = PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws)
        assert torch.equal(first, again)
    assert ((first.double() - o).abs() <= bound).all()
    # the same workspace for other, fewer and shorter streams, then the first again
    s2 = torch.tensor([10, 700], dtype=torch.int32, device="cuda")
    o2, b2, _ = attend_truth(q[:2], kp, vp, tab[:2], [10, 700], 64, 128 ** -0.5)
    got2 = PK.paged_decode_attention(q[:2], kp, vp, tab[:2], s2, workspace=ws)
    assert ((got2.double() - o2).abs() <= b2).all()
    assert torch.equal(first, PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws))


def test_attend_many_streams(PK):
    """More streams than one pass over the lengths holds."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 60, (1500,), generator=g).tolist()
    attend_case(PK, lens, hq=4, hkv=1, hd=64, seed=8)


def test_attend_offsets_past_32_bits(PK):
    """Pages past 2^32 bytes and 2^31 elements into the pool."""
    hkv, page, hd = 4, 128, 128
    total = (1 << 31) // (hkv * page * hd) + 64
    kp = torch.zeros(total, hkv, page, hd, device="cuda", dtype=BF16)
    tab = torch.tensor([[total - 1, 3, total - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in (total - 1, 3, total - 2):
        kp[i] = torch.randn(hkv, page, hd, device="cuda", generator=g).to(BF16)
    q = torch.randn(1, 16, hd, device="cuda", generator=g).to(BF16)
    o, bound, _ = attend_truth(q, kp, kp, tab, [300], page, hd ** -0.5)
    got = PK.paged_decode_attention(q, kp, kp, tab, torch.tensor([300], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert ((got.double() - o).abs() <= bound).all()
    cos, sin = PK.rotary_table(400, hd)
    qkv = torch.randn(1, 24 * hd, device="cuda", generator=g).to(BF16)
    vp = torch.zeros_like(kp)
    PK.rotary_paged_append(qkv, kp, vp, tab, torch.tensor([300], dtype=torch.int32, device="cuda"), cos, sin, 16)
    torch.cuda.synchronize()
    assert torch.equal(vp[total - 2, :, 299 % page], qkv.view(24, hd)[20:])
    PK.copy_pages(kp, torch.tensor([total - 1], dtype=torch.int32, device="cuda"), torch.tensor([total - 5], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(kp[total - 5], kp[total - 1])


def test_attend_garbage_past_the_end(PK):
    """NaN and infinities in the rest of a stream's last page, and in pages that are not its own, change nothing."""
    lens = [37, 5, 0, 161]
    tab, total = table(lens, 32, 2)
    g = torch.Generator(device="cuda").manual_seed(2)
    kp, vp = (torch.randn(total, 4, 32, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(4, 16, 128, device="cuda", generator=g).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = PK.paged_decode_attention(q, kp, vp, tab, seq)
    used = torch.zeros(total, 32, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for t in range(n):
            used[tab[b, t // 32].item(), t % 32] = True
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = kp.clone(), vp.clone()
        k2.permute(0, 2, 1, 3)[~used] = bad
        v2.permute(0, 2, 1, 3)[~used] = bad
        assert torch.equal(clean, PK.paged_decode_attention(q, k2, v2, tab, seq))


def test_attend_extreme_scores(PK):
    """Scores of thousands: the running maximum keeps every exponent at or below 0."""
    lens = [700, 33]
    tab, total = table(lens, 16, 12)
    g = torch.Generator(device="cuda").manual_seed(12)
    kp, vp = (torch.randn(total, 4, 16, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = (200 * torch.randn(2, 16, 128, device="cuda", generator=g)).to(BF16)
    got = PK.paged_decode_attention(q, kp, vp, tab, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    o, bound, _ = attend_truth(q, kp, vp, tab, lens, 16, 128 ** -0.5)
    assert torch.isfinite(got).all() and ((got.double() - o).abs() <= bound).all()


def test_attend_graph_and_streams(PK):
    """A captured call follows lengths and pages that change on the device; a call on another stream gives the same bits."""
    lens = [100, 20]
    tab, total = table([400, 400], 16, 6)
    g = torch.Generator(device="cuda").manual_seed(6)
    kp, vp = (torch.randn(total, 4, 16, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = torch.randn(2, 16, 128, device="cuda", generator=g).to(BF16)
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = PK.decode_workspace(2, 16, 128)
    PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = PK.paged_decode_attention(q, kp, vp, tab, seq, workspace=ws)
    for new in ([400, 0], [1, 333]):
        seq.copy_(torch.tensor(new, dtype=torch.int32))
        gr.replay()
        torch.cuda.synchronize()
        o, bound, _ = attend_truth(q, kp, vp, tab, new, 16, 128 ** -0.5)
        assert ((out.double() - o).abs() <= bound + 1e-30).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other = PK.paged_decode_attention(q, kp, vp, tab, seq, stream=s)
    s.synchronize()
    assert torch.equal(other, out)


def test_out_of_range_is_recorded(PK, cuda_lib):
    """Pages that do not exist and lengths past the table: nothing is read there, the status says so."""
    assert cuda_lib.sn_device_status(1, None) == 0
    kp = torch.zeros(4, 4, 16, 128, device="cuda", dtype=BF16)
    q = torch.ones(1, 16, 128, device="cuda", dtype=BF16)
    seq = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")
    for tab, n in (([[0, 99]], 20), ([[0, -1]], 20), ([[0, 1]], 33), ([[0, 1]], -1)):
        t = torch.tensor(tab, dtype=torch.int32, device="cuda")
        assert torch.isfinite(PK.paged_decode_attention(q, kp, kp, t, seq(n))).all()
        assert cuda_lib.sn_device_status(1, None) == -1
    cos, sin = PK.rotary_table(64, 128)
    qkv = torch.ones(1, 24 * 128, device="cuda", dtype=BF16)
    for tab, n in (([[0, 99]], 20), ([[0, -1]], 20), ([[0, 1]], 33), ([[0, 1]], 0), ([[0, 1, 2, 3, 0]], 65)):
        t = torch.tensor(tab, dtype=torch.int32, device="cuda")
        PK.rotary_paged_append(qkv, kp, kp, t, seq(n), cos, sin, 16)
        assert cuda_lib.sn_device_status(1, None) == -1
    assert not kp.any()
    bad = torch.tensor([7], dtype=torch.int32, device="cuda")
    PK.copy_pages(kp, bad, seq(0))
    assert cuda_lib.sn_device_status(1, None) == -1


# ---- rotary and append ----

def rotary_truth(x, cos, sin, pos, inter):
    """x [T, heads, hd] float64 -> rotated, and |x1| + |x2| for the bound."""
    rot = 2 * cos.shape[1]
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    y, a = x.clone(), torch.zeros_like(x)
    i1 = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
    i2 = i1 + (1 if inter else rot // 2)
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = x1 * c - x2 * s, x2 * c + x1 * s
    a[..., i1] = a[..., i2] = x1.abs() + x2.abs()
    return y, a


def append_case(PK, new, before, hq=16, hkv=4, hd=128, rot=128, inter=False, page=16, seed=0, pad=0, offset=0, one_each=False, strided=False):
    lens = [n + b for n, b in zip(new, before)]
    tab, total = table(lens, page, seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, width = sum(new), (hq + 2 * hkv) * hd
    qkv = torch.randn(T, width + pad + offset, device="cuda", generator=g).to(BF16)[:, offset:offset + width]
    if strided:
        kp = torch.full((total, page, hkv, 2 * hd), 7.0, device="cuda", dtype=BF16)[..., :hd].transpose(1, 2)
        vp = torch.full((total, page, hkv, 2 * hd), 7.0, device="cuda", dtype=BF16)[..., hd:].transpose(1, 2)
    else:
        kp = torch.full((total, hkv, page, hd), 7.0, device="cuda", dtype=BF16)
        vp = kp.clone()
    cos, sin = PK.rotary_table(max(lens) + 3, rot) if rot else (torch.zeros(max(lens) + 3, 0, device="cuda"),) * 2
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = PK.rotary_paged_append(qkv, kp, vp, tab, seq, cos, sin, hq, cu_seqlens=None if one_each else cu, interleaved=inter)
    torch.cuda.synchronize()
    pos = torch.cat([torch.arange(b, b + n) for n, b in zip(new, before)] or [torch.zeros(0)]).long().cuda()
    of = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    x = qkv.double().reshape(T, hq + 2 * hkv, hd)
    y, a = rotary_truth(x[:, :hq + hkv], cos, sin, pos, inter)
    bound = E * y.abs() + 2.0 ** -22 * a
    assert ((q.double() - y[:, :hq]).abs() <= bound[:, :hq]).all()
    if rot < hd:  # what is not rotated is copied
        assert torch.equal(q[..., rot:].double(), x[:, :hq, rot:])
    pg, at = tab[of, pos // page].long(), pos % page
    assert ((kp[pg, :, at].double() - y[:, hq:]).abs() <= bound[:, hq:]).all()
    assert torch.equal(vp[pg, :, at].double(), x[:, hq + hkv:])
    for p in (kp, vp):  # and nothing else is written
        rest = torch.ones(total, page, dtype=torch.bool, device="cuda")
        rest[pg, at] = False
        assert (p.permute(0, 2, 1, 3)[rest] == 7.0).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot,hd", [(128, 128), (64, 128), (32, 128), (64, 64), (16, 64), (6, 64), (2, 8), (0, 64), (40, 80), (48, 96)])
def test_append_rotations(PK, rot, hd, inter):
    append_case(PK, [70, 1, 33], [0, 200, 15], hd=hd, rot=rot, inter=inter, seed=rot + hd)


@pytest.mark.parametrize("new,before", [([1], [0]), ([1], [999]), ([0, 3, 0, 0, 200, 1, 0], [5, 0, 0, 17, 16, 31, 2]),
                                        ([1] * 70, list(range(70))), ([2] * 1100, [7] * 1100), ([2100], [0])])
def test_append_lengths(PK, new, before):
    append_case(PK, new, before, seed=len(new))


def test_append_one_token_each(PK):
    append_case(PK, [1] * 50, list(range(0, 500, 10)), one_each=True, seed=1)


@pytest.mark.parametrize("page", [1, 5, 16, 64, 100])
def test_append_page_sizes(PK, page):
    append_case(PK, [130, 7], [3, 0], page=page, seed=page)


@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (8, 8)])
def test_append_strides(PK, pad, offset):
    append_case(PK, [130, 7], [3, 0], pad=pad, offset=offset, seed=2)
    append_case(PK, [130, 7], [3, 0], pad=pad, offset=offset, seed=2, strided=True, inter=True)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (8, 1), (7, 2)])
def test_append_heads(PK, hq, hkv):
    append_case(PK, [33, 2], [3, 0], hq=hq, hkv=hkv, seed=hq)


def test_append_no_tokens(PK):
    append_case(PK, [0, 0], [3, 9])


def test_append_equals_the_dense_cache(PK):
    """The same bits as rotary_kv_append at one common position."""
    from sonata_b200.kernels import decode_step as DS, mamba_step as MS
    qkv = torch.randn(3, 24 * 128, device="cuda").to(BF16)
    kc, vc = (torch.zeros(3, 4, 64, 128, device="cuda", dtype=BF16) for _ in range(2))
    cos, sin = PK.rotary_table(64, 128)
    q0 = MS.rotary_kv_append(qkv, kc, vc, cos[40].contiguous(), sin[40].contiguous(), 16, 40)
    kp, vp = (torch.zeros(12, 4, 16, 128, device="cuda", dtype=BF16) for _ in range(2))
    tab = torch.arange(12, device="cuda", dtype=torch.int32).view(3, 4)
    q1 = PK.rotary_paged_append(qkv, kp, vp, tab, torch.full((3,), 41, dtype=torch.int32, device="cuda"), cos, sin, 16)
    torch.cuda.synchronize()
    assert torch.equal(q0.view(3, 16, 128), q1)
    dense = kp.view(3, 4, 4, 16, 128).transpose(1, 2).reshape(3, 4, 64, 128)
    assert torch.equal(dense, kc) and torch.equal(vp.view(3, 4, 4, 16, 128).transpose(1, 2).reshape(3, 4, 64, 128), vc)


def test_rotary_tables(PK):
    cos, sin = PK.rotary_table(5000, 64, base=10000.0)
    j = torch.arange(32, dtype=torch.float64)
    ang = torch.arange(5000, dtype=torch.float64)[:, None] * 10000.0 ** (-j / 32)
    assert (cos.cpu().double() - ang.cos()).abs().max() <= 2.0 ** -25 + 1e-12
    c2, _ = PK.rotary_table(5000, 64, factor=4.0)
    assert (c2.cpu().double() - (ang / 4).cos()).abs().max() <= 2.0 ** -25 + 1e-9
    c3, _ = PK.rotary_table(5000, 64, factor=4.0, original_max_pos=1000)
    turns = 1000 * 10000.0 ** (-j / 32) / (2 * np.pi)
    fast, slow = turns > 32, turns < 1
    assert fast.any() and slow.any()
    assert torch.allclose(c3.cpu()[:, fast], cos.cpu()[:, fast], atol=1e-6)
    assert torch.allclose(c3.cpu()[:, slow], c2.cpu()[:, slow], atol=1e-6)


# ---- page copies ----

@pytest.mark.parametrize("shape", [(9, 4, 16, 128), (2, 2, 9, 4, 16, 128), (3, 9, 1, 5, 7), (9, 2, 3, 1), (1, 9, 4, 128, 128)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32, torch.uint8])
def test_copy(PK, shape, dtype):
    pool = (torch.rand(shape, device="cuda") * 200).to(dtype)
    want = pool.clone()
    src, dst = [8, 0, 3], [1, 7, 2]
    want[..., dst, :, :, :] = pool[..., src, :, :, :]
    PK.copy_pages(pool, *(torch.tensor(v, dtype=torch.int32, device="cuda") for v in (src, dst)))
    torch.cuda.synchronize()
    assert torch.equal(pool, want)


def test_copy_unaligned_and_empty(PK):
    raw = torch.randn(9 * 64 + 1, device="cuda").to(BF16)
    pool, want = raw[1:].view(9, 2, 4, 8), raw[1:].clone().view(9, 2, 4, 8)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    PK.copy_pages(pool, i32(), i32())
    assert torch.equal(pool, want)
    PK.copy_pages(pool, i32(5), i32(0))
    want[0] = want[5]
    assert torch.equal(pool, want)


# ---- refusals ----

def test_refusals(PK):
    B, hd = 2, 128
    kp = torch.zeros(8, 4, 16, hd, device="cuda", dtype=BF16)
    q = torch.zeros(B, 16, hd, device="cuda", dtype=BF16)
    tab = torch.zeros(B, 3, device="cuda", dtype=torch.int32)
    seq = torch.ones(B, device="cuda", dtype=torch.int32)
    ok = dict(q=q, k_pages=kp, v_pages=kp, page_table=tab, seq_lens=seq)
    for change, err in ((dict(q=q.float()), TypeError), (dict(q=q.cpu()), ValueError), (dict(q=q[:1]), ValueError),
                        (dict(q=q[:, :6]), ValueError), (dict(q=q[..., :64]), ValueError), (dict(k_pages=kp[:4]), ValueError),
                        (dict(v_pages=kp.transpose(2, 3)), ValueError), (dict(k_pages=kp[0]), ValueError),
                        (dict(page_table=tab.long()), TypeError), (dict(page_table=tab[:1]), ValueError),
                        (dict(seq_lens=seq.float()), TypeError), (dict(page_table=tab[:, :0]), ValueError),
                        (dict(workspace=torch.zeros(1, dtype=torch.uint8, device="cuda")), ValueError)):
        with pytest.raises(err):
            PK.paged_decode_attention(**dict(ok, **change))
    qkv = torch.zeros(B, 24 * hd, device="cuda", dtype=BF16)
    cos, sin = PK.rotary_table(64, hd)
    ok = dict(qkv=qkv, k_pages=kp, v_pages=kp, page_table=tab, seq_lens=seq, cos=cos, sin=sin, nheads=16)
    for change, err in ((dict(qkv=qkv[:, :-1]), ValueError), (dict(qkv=qkv[:1]), ValueError), (dict(nheads=15), ValueError),
                        (dict(cos=cos.double()), TypeError), (dict(cos=cos[:5]), ValueError),
                        (dict(cu_seqlens=seq), ValueError), (dict(cu_seqlens=torch.zeros(3, device="cuda")), TypeError)):
        with pytest.raises(err):
            PK.rotary_paged_append(**dict(ok, **change))
    with pytest.raises(ValueError):
        PK.copy_pages(kp.transpose(1, 2), seq, seq)
    with pytest.raises(ValueError):
        PK.copy_pages(kp, seq, seq[:1])
    with pytest.raises(TypeError):
        PK.copy_pages(kp, seq.long(), seq.long())
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(factor=0.5), dict(max_pos=0)):
        with pytest.raises(ValueError):
            PK.rotary_table(**dict(dict(max_pos=8, rot_dim=4), **bad))
    with pytest.raises(ValueError):
        PK.decode_workspace(0, 16, 128)


@pytest.mark.parametrize("hd,rot,inter", [(128, 128, False), (128, 64, True), (40, 24, False)])
def test_append_refused_tokens_have_zero_q(PK, cuda_lib, hd, rot, inter):
    """Positions past the rotary table or before the stream's start, and rows of no stream: q is zero there and the pages
    are left alone, whatever the memory of the output held before; the other tokens are as they are in a call without them."""
    assert cuda_lib.sn_device_status(1, None) == 0
    g = torch.Generator(device="cuda").manual_seed(21)
    qkv = torch.randn(14, (6 + 2 * 2) * hd, device="cuda", generator=g).to(BF16)
    cos, sin = PK.rotary_table(20, rot)
    tab = torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2)  # two pages of 16 for each of 3 streams
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")

    def run(lens, cu, rows):
        kp, vp = (torch.full((6, 2, 16, hd), 7.0, device="cuda", dtype=BF16) for _ in range(2))
        poison = torch.full((rows.shape[0], 6, hd), float("nan"), device="cuda", dtype=BF16)
        del poison  # the output gets this block
        q = PK.rotary_paged_append(rows, kp, vp, tab, lens, cos, sin, 6, cu_seqlens=cu, interleaved=inter)
        torch.cuda.synchronize()
        return q, kp, vp

    # rows 0, 1 and 12, 13 belong to no stream; stream 0: positions 18 .. 21 of a table of 20; stream 1: -2 .. 1; stream 2: 3, 4
    q, kp, vp = run(ints(22, 2, 5), ints(2, 6, 10, 12), qkv)
    assert cuda_lib.sn_device_status(1, None) == -1
    kept = [2, 3, 8, 9, 10, 11]  # positions 18, 19 of stream 0; 0, 1 of stream 1; 3, 4 of stream 2
    want = run(ints(20, 2, 5), ints(0, 2, 4, 6), qkv[kept])
    assert cuda_lib.sn_device_status(1, None) == 0
    assert torch.equal(q[kept], want[0]) and torch.isfinite(want[0]).all()
    rest = [t for t in range(14) if t not in kept]
    assert not q[rest].any()
    assert torch.equal(kp, want[1]) and torch.equal(vp, want[2])


@pytest.mark.parametrize("lens,hq,hkv,hd", [([257], 16, 4, 128), ([1000, 0, 33], 16, 4, 64), ([700, 90], 32, 2, 128), ([500, 77], 24, 1, 64),
                                            ([20011], 16, 1, 128), ([9000, 4097, 5], 16, 4, 128), ([300, 40], 8, 4, 96)])
def test_attend_weights_keep_their_bits(PK, lens, hq, hkv, hd):
    """The weights are not rounded to bf16 on the way into the product: two operands hold 16 bits of them.  |err| <= 2^-8 |o|
    for the output, 2^-16 P for the weights and the scores' and joins' errors as above; the norm of the error that of the
    output's rounding (1.62e-3 over evenly spread mantissas), held to 1.8e-3."""
    g = torch.Generator(device="cuda").manual_seed(40 + hd)
    tab, total = table(lens, 32, 40)
    kp, vp = (torch.randn(total, hkv, 32, hd, device="cuda", generator=g).to(BF16) for _ in range(2))
    q = (1.5 * torch.randn(len(lens), hq, hd, device="cuda", generator=g)).to(BF16)
    o, loose, _ = attend_truth(q, kp, vp, tab, lens, 32, hd ** -0.5)
    absv, _, _ = attend_truth(q, kp, vp.abs(), tab, lens, 32, hd ** -0.5)  # P
    bound = loose - E * absv + 2.0 ** -16 * absv
    got = PK.paged_decode_attention(q, kp, vp, tab, torch.tensor(lens, dtype=torch.int32, device="cuda")).double()
    torch.cuda.synchronize()
    assert ((got - o).abs() <= bound + 1e-30).all(), ((got - o).abs() - bound).max().item()
    assert ((got - o).norm() / o.norm()).item() <= 1.8e-3
