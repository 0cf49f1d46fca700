"""The short way from tensors to the C ABI takes the plain calls, gives the same bits as the wrappers' own way, and leaves
every other call to them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def ways(cuda_lib):
    from sonata_b200 import build
    from sonata_b200.kernels import _common, mamba_prompt, paged_kv
    build.build_bind()
    assert _common.fast() is not _common._NoFast
    return _common, paged_kv, mamba_prompt


def _both(common, monkeypatch, run):
    """run() by the short way, which has to take it, and without it."""
    taken = []

    class Spy:
        pass
    for name in ("attend", "append", "copy", "prompt"):
        f = getattr(common.fast(), name)
        setattr(Spy, name, staticmethod(lambda *a, f=f: taken.append(f(*a)) or taken[-1]))
    monkeypatch.setattr(common, "_fast", Spy)
    a = run()
    assert taken and all(t is not None for t in taken)
    monkeypatch.setattr(common, "_fast", common._NoFast)
    b = run()
    torch.cuda.synchronize()
    return a, b


def test_same_bits(ways, monkeypatch):
    common, PK, MP = ways
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    kp, vp = r(12, 4, 16, 128), r(12, 4, 16, 128)
    tab = torch.arange(12, device="cuda", dtype=torch.int32).view(2, 6)
    lens = torch.tensor([90, 33], device="cuda", dtype=torch.int32)
    ws = PK.decode_workspace(2, 16, 128)
    q = r(2, 24, 128)[:, 4:20]
    for scale in (None, 0.1):
        a, b = _both(common, monkeypatch, lambda: PK.paged_decode_attention(q, kp, vp, tab, lens, scale=scale, workspace=ws))
        assert torch.equal(a, b)
        monkeypatch.undo()
    cos, sin = PK.rotary_table(100, 64)
    cu = torch.tensor([0, 5, 7], device="cuda", dtype=torch.int32)
    for qkv, c in ((r(7, 24 * 128 + 8)[:, :24 * 128], cu), (r(2, 24 * 128), None)):
        a, b = _both(common, monkeypatch, lambda: PK.rotary_paged_append(qkv, kp, vp, tab, lens, cos, sin, 16, cu_seqlens=c))
        assert torch.equal(a, b)
        monkeypatch.undo()
    one, two = (torch.tensor([v], device="cuda", dtype=torch.int32) for v in (1, 2))
    _both(common, monkeypatch, lambda: PK.copy_pages(kp, one, two))
    assert torch.equal(kp[1], kp[2])
    monkeypatch.undo()
    zx, conv, ssm = r(50, 2 * 256 + 256 + 4), r(2, 512, 4), r(2, 4, 64, 128)
    w, bias, A, D = r(512, 4), r(512), -torch.rand(4, device="cuda", generator=g), r(4)
    cu = torch.tensor([0, 20, 50], device="cuda", dtype=torch.int32)
    run = lambda: MP.mamba2_prompt(zx, conv.clone(), w, bias, ssm.clone(), A, D, None, 256, 1, 128, 4, cu_seqlens=cu, gate=True)
    a, b = _both(common, monkeypatch, run)
    assert torch.equal(a, b)


def test_leaves_the_rest_alone(ways):
    common, PK, MP = ways
    f = common.fast()
    t = torch.zeros(2, 16, 128, device="cuda", dtype=BF16)
    assert f.attend() is None and f.attend(t, 1, 2, 3, 4, None, None, False) is None
    assert f.copy(t, t, t) is None and f.append(*[t] * 10) is None and f.prompt(*[t] * 14) is None
    assert f.prompt(*[None] * 14) is None
