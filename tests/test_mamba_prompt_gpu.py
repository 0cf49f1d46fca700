"""mamba2_prompt against the recurrence in 64 bits.

Tolerances, from where the kernels round to bf16 (relative 2^-8 each): the
convolved x, B and C, and on the way of a term into y either the masked
score (once) or the weighted x and the state operand (twice): at most five,
and the output itself.  With Yabs = the same recurrence on absolute values,
|err| <= 5 2^-8 Yabs + 2^-8 |y|, and 1e-3 Yabs for the fp32 sums and
exponents (|sum dt A| < 400 in a chunk here).  States: x, B and the weighted
x, and the stored state.  Roundings are independent, so the norm of the
error is far below: 6 roundings, each uniform within half a unit (0.72 2^-8 /
sqrt(3) = 1.6e-3 rms over evenly spread mantissas), 4e-3, held to 5e-3.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -8  # half a unit in the last place of bf16 (8 significant bits)


@pytest.fixture(scope="module")
def MP(cuda_lib):
    from sonata_b200.kernels import mamba_prompt
    return mamba_prompt


def make(lens, nh=4, hd=64, ds=128, ng=1, W=4, seed=0, fresh=False, extra=0, dt_shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    u = lambda *s: torch.rand(*s, device="cuda", generator=g)
    di, gds, B, T = nh * hd, ng * ds, len(lens), sum(lens)
    cd = di + 2 * gds
    bf = torch.bfloat16
    a = dict(zxbcdt=r(T, di + cd + nh + extra).to(bf), conv_state=r(B, cd, W).to(bf), weight=(0.5 * r(cd, W)).to(bf),
             bias=(0.1 * r(cd)).to(bf), ssm_state=(0.5 * r(B, nh, hd, ds)).to(bf), A=-(u(nh) * 15 + 1),
             D=(1 + 0.2 * r(nh)).to(bf), dt_bias=(u(nh) * 2 - 4 + dt_shift).to(bf), d_inner=di, ngroups=ng, d_state=ds,
             nheads=nh)
    if fresh:
        a["conv_state"].zero_()
        a["ssm_state"].zero_()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    a["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    return a


def truth(a, gate=False):
    """(y, Yabs, conv_state, ssm_state, Sabs) in 64 bits, token by token."""
    nh, ng, ds, di = a["nheads"], a["ngroups"], a["d_state"], a["d_inner"]
    hd, W, cd = di // nh, a["weight"].shape[1], di + 2 * ng * ds
    d = lambda t: t.double() if t is not None else None
    w, bias, D, dtb = d(a["weight"]), d(a["bias"]), d(a["D"]), d(a["dt_bias"])
    cu = a["cu_seqlens"].tolist() if a["cu_seqlens"] is not None else [0, a["zxbcdt"].shape[0]]
    T = a["zxbcdt"].shape[0]
    y = torch.zeros(T, nh, hd, device="cuda", dtype=torch.float64)
    ya = torch.zeros_like(y)
    conv, ssm, sabs = d(a["conv_state"]).clone(), d(a["ssm_state"]).clone(), d(a["ssm_state"]).abs()
    for i in range(len(cu) - 1):
        n = cu[i + 1] - cu[i]
        row = a["zxbcdt"][cu[i]:cu[i + 1]].double()
        u = torch.cat([conv[i].T, row[:, di:di + cd]])
        conv[i] = u[n:].T
        x = sum(w[:, k] * u[1 + k:1 + k + n] for k in range(W)) + (bias if bias is not None else 0)
        x = x * torch.sigmoid(x)
        dt = row[:, di + cd:di + cd + nh] + (dtb if dtb is not None else 0)
        dt = torch.logaddexp(dt, torch.zeros_like(dt))
        xs = x[:, :di].reshape(n, nh, hd)
        Bm, Cm = (v.reshape(n, ng, ds).repeat_interleave(nh // ng, 1) for v in (x[:, di:di + ng * ds], x[:, di + ng * ds:]))
        for t in range(n):
            dec = torch.exp(dt[t] * a["A"].double())[:, None, None]
            add = (dt[t][:, None] * xs[t])[:, :, None] * Bm[t][:, None, :]
            ssm[i] = ssm[i] * dec + add
            sabs[i] = sabs[i] * dec + add.abs()
            y[cu[i] + t] = (ssm[i] * Cm[t][:, None, :]).sum(-1)
            ya[cu[i] + t] = (sabs[i] * Cm[t][:, None, :].abs()).sum(-1)
        s = slice(cu[i], cu[i + 1])
        if D is not None:
            y[s] += D[:, None] * xs
            ya[s] += (D[:, None] * xs).abs()
        if gate:
            z = row[:, :di].reshape(n, nh, hd)
            f = z * torch.sigmoid(z)
            y[s] *= f
            ya[s] *= f.abs()
    return y, ya, conv, ssm, sabs


def check(got, ref, bound, what, norm=5e-3):
    err = (got.double() - ref).abs()
    over = (err - bound).max().item() if err.numel() else 0.0
    assert over <= 0, (what, over, err.max().item())
    if ref.numel() and ref.norm() > 0:
        assert (err.norm() / ref.norm()).item() <= norm, (what, (err.norm() / ref.norm()).item())


def run_and_check(MP, a, gate=False, norm=5e-3):
    y0, ya, conv, ssm, sabs = truth(a, gate)
    y = MP.mamba2_prompt(gate=gate, **a)
    torch.cuda.synchronize()
    check(y, y0, (5 * E + 1e-3) * ya + E * y0.abs() + 1e-30, "y", norm)
    check(a["ssm_state"], ssm, (3 * E + 1e-3) * sabs + E * ssm.abs() + 1e-30, "ssm_state", norm)
    assert torch.equal(a["conv_state"].double(), conv)
    return y


@pytest.mark.parametrize("lens", [[1], [2], [3], [5], [16], [127], [128], [129], [256], [300], [1000],
                                  [0, 5, 0, 130, 3, 0], [1, 1, 1, 1], [128, 128], [129, 255, 7]])
@pytest.mark.parametrize("gate", [False, True])
def test_lengths(MP, lens, gate):
    run_and_check(MP, make(lens, seed=sum(lens)), gate)


@pytest.mark.parametrize("nh,hd,ds,ng,W", [(64, 64, 128, 1, 4), (6, 64, 128, 2, 4), (3, 64, 128, 1, 3), (8, 64, 128, 8, 2),
                                           (4, 32, 128, 1, 4), (2, 64, 64, 1, 4), (3, 20, 16, 3, 4), (2, 64, 256, 2, 4),
                                           (2, 128, 128, 1, 8), (5, 64, 100, 5, 1), (2, 64, 128, 1, 5)])
def test_shapes(MP, nh, hd, ds, ng, W):
    run_and_check(MP, make([70, 140, 9], nh=nh, hd=hd, ds=ds, ng=ng, W=W, seed=nh + ds))


@pytest.mark.parametrize("off", ["bias", "D", "dt_bias"])
def test_without_optional(MP, off):
    a = make([150, 31], seed=3)
    a[off] = None
    if off == "dt_bias":  # keep dt in its usual range
        a["zxbcdt"][:, -a["nheads"]:] -= 3
    run_and_check(MP, a)


@pytest.mark.parametrize("extra", [0, 1, 3, 8])
def test_row_strides(MP, extra):
    """Rows wider than the projection, on and off 16-byte strides, and a base off 16 bytes."""
    a = make([150, 31], seed=4, extra=extra + 8)
    a["zxbcdt"] = a["zxbcdt"][:, extra:]
    run_and_check(MP, a, gate=True)


def test_one_prompt_without_offsets(MP):
    a = make([333], seed=5)
    a["cu_seqlens"] = None
    run_and_check(MP, a)


def test_no_tokens(MP):
    a = make([0, 0], seed=6)
    before = a["conv_state"].clone(), a["ssm_state"].clone()
    y = MP.mamba2_prompt(**a)
    torch.cuda.synchronize()
    assert y.shape == (0, 4, 64)
    assert torch.equal(a["conv_state"], before[0]) and torch.equal(a["ssm_state"], before[1])


@pytest.mark.parametrize("T", [4000, 9000])
def test_long_prompts(MP, T):
    """Many chunks, and enough of them that a prompt is cut into segments."""
    run_and_check(MP, make([T], nh=2, seed=7))
    run_and_check(MP, make([T // 3, 1, T // 2], nh=64, seed=8)) if T == 4000 else None


def test_strong_decay(MP):
    """dt A of some hundreds a token: everything but the newest token underflows, nothing turns into NaN."""
    a = make([300, 40], seed=9, dt_shift=24.0)
    y0, ya, conv, ssm, sabs = truth(a)
    y = MP.mamba2_prompt(**a)
    torch.cuda.synchronize()
    assert torch.isfinite(y).all()
    # |sum dt A| reaches 128 * 28 * 16 in a chunk: the exponents' error is 6e4 2^-23 = 7e-3 of the terms left
    check(y, y0, (5 * E + 1e-2) * ya + E * y0.abs() + 1e-30, "y")


def test_pieces_equal_the_whole(MP):
    """A prompt in three pieces: the states carried between them (rounded to bf16 there) give the whole's outputs."""
    a = make([500], nh=8, seed=10, fresh=True)
    y0, ya, conv, ssm, sabs = truth(a)
    got = []
    for s, e in ((0, 130), (130, 131), (131, 500)):
        p = dict(a, zxbcdt=a["zxbcdt"][s:e], cu_seqlens=None)
        got.append(MP.mamba2_prompt(**p))
    torch.cuda.synchronize()
    check(torch.cat(got), y0, (6 * E + 1e-3) * ya + E * y0.abs(), "y")  # one more rounding: the stored state
    assert torch.equal(a["conv_state"].double(), conv)


def test_goes_on_into_decoding(MP):
    """The states a prompt leaves are those of the single-token kernels: one decode step equals the prompt's next token."""
    from sonata_b200.kernels import mamba_step as MS
    nh, di, ds = 8, 512, 128
    a = make([201, 77], nh=nh, seed=11)
    y0, ya, conv, ssm, sabs = truth(a)
    last = torch.tensor([200, 277], device="cuda")
    part = dict(a, zxbcdt=torch.cat([a["zxbcdt"][:200], a["zxbcdt"][201:277]]).contiguous(),
                cu_seqlens=torch.tensor([0, 200, 276], dtype=torch.int32, device="cuda"))
    MP.mamba2_prompt(**part)
    sync = torch.zeros(2, dtype=torch.int32, device="cuda")
    z, y = MS.mamba2_conv_ssu(a["zxbcdt"][last].contiguous(), a["conv_state"], a["weight"], a["bias"], a["ssm_state"], a["A"],
                              a["D"], a["dt_bias"], di, 1, ds, nh, sync)
    torch.cuda.synchronize()
    check(y, y0[last], (6 * E + 1e-3) * ya[last] + E * y0[last].abs(), "y")
    check(a["ssm_state"], ssm, (4 * E + 1e-3) * sabs + E * ssm.abs(), "ssm_state")
    assert torch.equal(a["conv_state"].double(), conv)


def test_prompts_do_not_touch_each_other(MP):
    """NaN and infinities in one prompt leave every other's outputs and states bit for bit as they were."""
    lens = [40, 200, 129, 1]
    a, b = make(lens, seed=12), make(lens, seed=12)
    b["zxbcdt"][40:240] = float("nan")
    b["zxbcdt"][100] = float("inf")
    ya, yb = MP.mamba2_prompt(**a), MP.mamba2_prompt(**b)
    torch.cuda.synchronize()
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[40:240] = False
    assert torch.equal(ya[keep], yb[keep])
    for s in ("conv_state", "ssm_state"):
        assert torch.equal(a[s][[0, 2, 3]], b[s][[0, 2, 3]])
    assert torch.isnan(yb[~keep]).any()


def test_same_call_same_bits_and_other_streams(MP):
    a, b = make([700, 90], nh=64, seed=13), make([700, 90], nh=64, seed=13)
    ya = MP.mamba2_prompt(**a)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    yb = MP.mamba2_prompt(**b, stream=s)
    s.synchronize()
    assert torch.equal(ya, yb) and torch.equal(a["ssm_state"], b["ssm_state"])


def test_in_a_graph_with_new_offsets(MP):
    """The offsets are read on the device: a captured call serves another split of the same tokens."""
    a = make([100, 200], seed=14)
    y = MP.mamba2_prompt(**a)  # first call outside capture
    torch.cuda.synchronize()
    st = [a["conv_state"].clone(), a["ssm_state"].clone()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = MP.mamba2_prompt(**a)
    a["cu_seqlens"].copy_(torch.tensor([0, 290, 300], dtype=torch.int32, device="cuda"))
    a["conv_state"].copy_(st[0])
    a["ssm_state"].copy_(st[1])
    y0, ya, conv, ssm, sabs = truth(a)
    g.replay()
    torch.cuda.synchronize()
    check(y, y0, (5 * E + 1e-3) * ya + E * y0.abs(), "y")
    check(a["ssm_state"], ssm, (3 * E + 1e-3) * sabs + E * ssm.abs(), "ssm_state")


def test_bad_offsets_are_recorded(MP, cuda_lib):
    assert cuda_lib.sn_device_status(1, None) == 0
    a = make([30, 30], seed=15)
    a["cu_seqlens"].copy_(torch.tensor([0, 90, 60], dtype=torch.int32, device="cuda"))
    MP.mamba2_prompt(**a)
    assert cuda_lib.sn_device_status(1, None) == -1
    assert cuda_lib.sn_device_status(0, None) == 0


def test_refusals(MP):
    from sonata_b200._lib import SonataError
    a = make([10, 10], seed=16)
    for change, err in ((dict(zxbcdt=a["zxbcdt"].cpu()), ValueError), (dict(zxbcdt=a["zxbcdt"].float()), TypeError),
                        (dict(zxbcdt=a["zxbcdt"][:, :-1]), ValueError), (dict(zxbcdt=a["zxbcdt"].T.contiguous().T), ValueError),
                        (dict(ssm_state=a["ssm_state"][:1]), ValueError), (dict(conv_state=a["conv_state"][:, :-1]), ValueError),
                        (dict(A=a["A"].double()), TypeError), (dict(D=a["D"][:2]), ValueError), (dict(nheads=3), ValueError),
                        (dict(cu_seqlens=a["cu_seqlens"].long()), TypeError), (dict(cu_seqlens=a["cu_seqlens"][:1]), ValueError),
                        (dict(weight=a["weight"][:, :3]), ValueError)):
        with pytest.raises(err):
            MP.mamba2_prompt(**dict(a, **change))
    with pytest.raises(SonataError):  # convolutions wider than 8
        MP.mamba2_prompt(**make([10], W=9))
    with pytest.raises(SonataError):  # states longer than 256
        MP.mamba2_prompt(**make([10], ds=264))


@pytest.mark.parametrize("hd,extra", [(64, 4), (64, 0), (32, 0)])  # by chunks (rows of 776 elements); token by token
def test_rows_of_no_prompt_are_zero(MP, hd, extra):
    """Tokens before the first and past the last prompt (a padded buffer): zeros, whatever the output's memory held; the
    prompts are as they are without them."""
    for front, back in ((3, 0), (0, 200), (5, 1)):
        a, b = (make([70, 130], hd=hd, extra=extra, seed=17) for _ in range(2))
        a["zxbcdt"] = torch.cat([a["zxbcdt"][:front], a["zxbcdt"], a["zxbcdt"][:back]])
        a["cu_seqlens"] += front
        poison = torch.full((front + 200 + back, 4, hd), float("nan"), device="cuda", dtype=torch.bfloat16)
        del poison  # the output gets this block
        ya, yb = MP.mamba2_prompt(**a), MP.mamba2_prompt(**b)
        torch.cuda.synchronize()
        assert torch.equal(ya[front:front + 200], yb)
        assert not ya[:front].any() and not ya[front + 200:].any()
        for s in ("conv_state", "ssm_state"):
            assert torch.equal(a[s], b[s])


@pytest.mark.parametrize("hd,extra", [(64, 4), (64, 0), (32, 0)])
def test_falling_offsets_do_not_overlap(MP, cuda_lib, hd, extra):
    """An offset below the one before it counts as that one, and is recorded: no token has two prompts."""
    a, b = (make([100, 0, 20], hd=hd, extra=extra, seed=18) for _ in range(2))
    a["cu_seqlens"][2] = 50
    ya, yb = MP.mamba2_prompt(**a), MP.mamba2_prompt(**b)
    assert cuda_lib.sn_device_status(1, None) == -1
    assert torch.equal(ya, yb)
    for s in ("conv_state", "ssm_state"):
        assert torch.equal(a[s], b[s])


# ---- the form by chunks, on the tensor cores: heads of 64, 128 states, widths 2 to 4, rows of whole 16 bytes ----
#
# Its products' operands are rounded to fp16 (2^-11 each): x, B and C, and the masked score, or the weighted x and the state
# operand: at most five in a term of y, three in one of the state.  Exponents: |sum dt A| < 400 in a chunk here, 577 as
# powers of two, with about nine fp32 roundings of the sum (577 * 9 * 2^-24 ln 2 = 2e-4) and dt good to 5e-7 (2e-4): 5e-4.
# Norm: the output's rounding (1.62e-3) and five of 2.0e-4, 1.7e-3 together, held to 2.2e-3.
F = 2.0 ** -11


def tile(lens, nh=4, ng=1, W=4, **k):
    """make() with rows padded to whole 16 bytes."""
    wide = 2 * nh * 64 + 2 * ng * 128 + nh
    a = make(lens, nh=nh, ng=ng, W=W, extra=-wide % 8, **k)
    assert a["zxbcdt"].stride(0) % 8 == 0
    return a


def check_tile(MP, a, gate=False, norm=2.2e-3, **k):
    y0, ya, conv, ssm, sabs = truth(a, gate)
    y = MP.mamba2_prompt(gate=gate, **a, **k)
    torch.cuda.synchronize()
    check(y, y0, (5 * F + 5e-4) * ya + E * y0.abs() + 1e-30, "y", norm)
    check(a["ssm_state"], ssm, (3 * F + 5e-4) * sabs + E * ssm.abs() + 1e-30, "ssm_state", norm)
    assert torch.equal(a["conv_state"].double(), conv)
    return y


@pytest.mark.parametrize("lens", [[1], [2], [3], [5], [7], [8], [31], [32], [33], [64], [127], [128], [129], [130], [256], [300],
                                  [1000], [0, 5, 0, 130, 3, 0], [1, 1, 1, 1], [128, 128], [129, 255, 7], [1] * 70])
@pytest.mark.parametrize("gate", [False, True])
def test_tile_lengths(MP, lens, gate):
    check_tile(MP, tile(lens, seed=sum(lens)), gate)


@pytest.mark.parametrize("nh,ng,W", [(64, 1, 4), (6, 2, 4), (3, 1, 3), (8, 8, 2), (1, 1, 4), (5, 5, 4), (10, 2, 2), (48, 1, 3)])
def test_tile_heads_and_groups(MP, nh, ng, W):
    check_tile(MP, tile([70, 140, 9], nh=nh, ng=ng, W=W, seed=nh), gate=nh % 2 == 0)


@pytest.mark.parametrize("off", ["bias", "D", "dt_bias", "cu_seqlens"])
def test_tile_without_optional(MP, off):
    a = tile([150, 31] if off != "cu_seqlens" else [333], seed=3)
    a[off] = None
    if off == "dt_bias":  # keep dt in its usual range
        a["zxbcdt"][:, 2 * 256 + 256:] -= 3
    check_tile(MP, a)


@pytest.mark.parametrize("nh,ng,lens", [
    (2, 1, [4000]), (2, 1, [9000]),      # many segments
    (6, 2, [3000]), (3, 1, [1500, 900, 77]),  # three heads a group: a head alone in its pair, several prompts cut
    (64, 1, [2048, 1, 2100, 129, 40]),   # two prompts cut once among short ones
    (4, 1, [700] * 9), (1, 1, [5, 2000, 0, 2001, 128, 384])])
def test_tile_segments(MP, nh, ng, lens):
    check_tile(MP, tile(lens, nh=nh, ng=ng, seed=len(lens) + nh))


def test_tile_strong_decay(MP):
    """As test_strong_decay."""
    a = tile([300, 40], seed=9, dt_shift=24.0)
    y0, ya, conv, ssm, sabs = truth(a)
    y = MP.mamba2_prompt(**a)
    torch.cuda.synchronize()
    assert torch.isfinite(y).all()
    check(y, y0, (5 * F + 1e-2) * ya + E * y0.abs() + 1e-30, "y")


def test_tile_pieces_equal_the_whole(MP):
    a = tile([500], nh=8, seed=10, fresh=True)
    y0, ya, conv, ssm, sabs = truth(a)
    got = []
    for s, e in ((0, 130), (130, 131), (131, 500)):
        got.append(MP.mamba2_prompt(**dict(a, zxbcdt=a["zxbcdt"][s:e], cu_seqlens=None)))
    torch.cuda.synchronize()
    check(torch.cat(got), y0, (5 * F + 5e-4 + E) * ya + E * y0.abs(), "y")  # and the stored state, to bf16
    assert torch.equal(a["conv_state"].double(), conv)


def test_tile_prompts_do_not_touch_each_other(MP):
    lens = [40, 200, 129, 1]
    a, b = tile(lens, seed=12), tile(lens, seed=12)
    b["zxbcdt"][40:240] = float("nan")
    b["zxbcdt"][100] = float("inf")
    ya, yb = MP.mamba2_prompt(**a), MP.mamba2_prompt(**b)
    torch.cuda.synchronize()
    keep = torch.ones(sum(lens), dtype=torch.bool, device="cuda")
    keep[40:240] = False
    assert torch.equal(ya[keep], yb[keep])
    for s in ("conv_state", "ssm_state"):
        assert torch.equal(a[s][[0, 2, 3]], b[s][[0, 2, 3]])
    assert torch.isnan(yb[~keep]).any()


def test_tile_in_a_graph_with_new_offsets(MP):
    a = tile([100, 200], seed=14)
    MP.mamba2_prompt(**a)  # first call outside capture
    torch.cuda.synchronize()
    st = [a["conv_state"].clone(), a["ssm_state"].clone()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = MP.mamba2_prompt(**a)
    a["cu_seqlens"].copy_(torch.tensor([0, 290, 300], dtype=torch.int32, device="cuda"))
    a["conv_state"].copy_(st[0])
    a["ssm_state"].copy_(st[1])
    y0, ya, conv, ssm, sabs = truth(a)
    g.replay()
    torch.cuda.synchronize()
    check(y, y0, (5 * F + 5e-4) * ya + E * y0.abs(), "y")
    check(a["ssm_state"], ssm, (3 * F + 5e-4) * sabs + E * ssm.abs(), "ssm_state")


# Values of unequal size: every element within the bound above, which is relative to the absolute values of its own terms.

@pytest.mark.parametrize("down", [16, 22])
@pytest.mark.parametrize("lens", [[300], [2100, 77]])  # the second with states of segments
def test_tile_quiet_head(MP, down, lens):
    """Every other head's x 2^-down of its neighbour's, and a quiet channel in each."""
    a = tile(lens, nh=4, seed=30)
    a["D"] = None
    for h in (1, 3):
        a["weight"][64 * h:64 * h + 64] *= 2.0 ** -down
        a["bias"][64 * h:64 * h + 64] *= 2.0 ** -down
    a["weight"][10:64 * 4:64] *= 2.0 ** -16
    a["bias"][10:64 * 4:64] *= 2.0 ** -16
    check_tile(MP, a)


@pytest.mark.parametrize("down", [4, 8])
def test_tile_quiet_then_loud(MP, down):
    """The first tokens of a chunk with x, B, C and dt 2^-down of the later ones': their outputs are as good."""
    a = tile([128, 333], nh=4, seed=31, fresh=True)
    a["D"] = a["bias"] = None
    di, cd = 256, 512
    for at in (0, 128, 128 + 256):
        a["zxbcdt"][at:at + 60, di:di + cd] *= 2.0 ** -down
        a["zxbcdt"][at:at + 60, di + cd:di + cd + 4] -= down * 0.69
    check_tile(MP, a)


def test_tile_spread_over_tokens(MP):
    """Runs of tokens whose rows are 2^0 to 2^-8 as large as others', and dt from 2^-16 to 2, in no order."""
    a = tile([1000, 200], nh=4, seed=32)
    a["D"] = a["bias"] = None
    g = torch.Generator(device="cuda").manual_seed(33)
    size = 2.0 ** -(8 * torch.rand(150, 1, device="cuda", generator=g)).repeat_interleave(8, 0)
    di, cd = 256, 512
    a["zxbcdt"][:, di:di + cd] *= size
    a["zxbcdt"][:, di + cd:di + cd + 4] = torch.rand(1200, 4, device="cuda", generator=g) * 13 - 8
    a["A"] /= 16  # dt reaches 2 here: sums of dt A as the bound has them
    check_tile(MP, a)


def test_tile_quiet_states(MP):
    """B and C of every fourth state 2^-10 of the others, and an initial state of widely different elements."""
    a = tile([260], nh=4, seed=34)
    a["D"] = None
    for at in (256, 384):
        for t in ("weight", "bias"):
            a[t][at:at + 128:4] *= 2.0 ** -10
    g = torch.Generator(device="cuda").manual_seed(35)
    a["ssm_state"] *= 2.0 ** -(8 * torch.rand(a["ssm_state"].shape, device="cuda", generator=g))
    check_tile(MP, a)
