"""The short way from tensors to the C ABI for the operators of long streams: it takes the plain calls, gives the same bits as
the wrappers' own way, and leaves every other call to them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture
def ways(cuda_lib):
    from sonata_b200 import build
    from sonata_b200.kernels import _common, paged_evict, paged_kv, paged_sparse
    build.build_bind()
    assert _common.fast() is not _common._NoFast
    return _common, paged_kv, paged_evict, paged_sparse


def _both(common, monkeypatch, run):
    """run() by the short way, which has to take it, and without it."""
    taken = []

    class Spy:
        pass
    for name in ("append", "mass", "evict", "bounds", "select", "sparse"):
        f = getattr(common.fast(), name)
        setattr(Spy, name, staticmethod(lambda *a, f=f: taken.append(f(*a)) or taken[-1]))
    with monkeypatch.context() as m:
        m.setattr(common, "_fast", Spy)
        a = run()
        assert taken and all(t is not None for t in taken)
        m.setattr(common, "_fast", common._NoFast)
        b = run()
    torch.cuda.synchronize()
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_same_bits(ways, monkeypatch):
    common, PK, PE, PS = ways
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    pool = r(3, 2, 12, 4, 16, 128)
    kp, vp = pool[1, 0], pool[1, 1]
    tab = torch.arange(12, device="cuda", dtype=torch.int32).view(2, 6)
    lens = torch.tensor([90, 33], device="cuda", dtype=torch.int32)
    q = r(2, 24, 128)[:, 4:20]
    mass = torch.rand(3, 2, 4, 100, device="cuda", generator=g)
    ws = PE.mass_workspace(2, 16, 4, 128, 96)

    def attend(scale=None):
        m = mass.clone()
        return PE.paged_decode_attention_mass(q, kp, vp, tab, lens, m[1], scale=scale, workspace=ws), m

    def evict(source):
        p, m = pool.clone(), mass.clone()
        s = PE.evict_positions(p, tab, lens, m, 40, recent=8, sinks=2, return_source=source)
        assert (s is not None) == source
        return (p, m, s) if source else (p, m)

    bounds = PS.page_bounds(kp)

    def update(cu):
        b = bounds.clone()
        PS.update_page_bounds(kp, b, tab, lens, cu_seqlens=cu)
        return b,

    _both(common, monkeypatch, attend)
    _both(common, monkeypatch, lambda: attend(0.1))
    _both(common, monkeypatch, lambda: evict(True))
    _both(common, monkeypatch, lambda: evict(False))
    _both(common, monkeypatch, lambda: update(None))
    cu = torch.tensor([0, 90, 123], device="cuda", dtype=torch.int32)
    _both(common, monkeypatch, lambda: update(cu))
    PS.update_page_bounds(kp, bounds, tab, lens, cu_seqlens=cu)
    _both(common, monkeypatch, lambda: (PS.select_blocks(q, bounds, tab, lens, 16, 3, first=1, last=1),))
    blocks = PS.select_blocks(q, bounds, tab, lens, 16, 3)
    _both(common, monkeypatch, lambda: (PS.paged_sparse_attention(q, kp, vp, tab, lens, blocks, workspace=ws),))


def test_append_with_positions(ways, monkeypatch):
    common, PK, *_ = ways
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    tab = torch.arange(12, device="cuda", dtype=torch.int32).view(2, 6)
    lens, cu = (torch.tensor(v, device="cuda", dtype=torch.int32) for v in ([90, 33], [0, 5, 7]))
    cos, sin = PK.rotary_table(300, 64)
    for qkv, c, at in ((r(7, 24 * 128), cu, range(200, 207)), (r(2, 24 * 128), None, (299, 3))):
        at = torch.tensor(list(at), device="cuda", dtype=torch.int32)

        def run():
            kp, vp = torch.zeros(12, 4, 16, 128, device="cuda", dtype=BF16), torch.zeros(12, 4, 16, 128, device="cuda", dtype=BF16)
            return PK.rotary_paged_append(qkv, kp, vp, tab, lens, cos, sin, 16, cu_seqlens=c, positions=at), kp, vp
        _both(common, monkeypatch, run)
        f = common.fast().append
        plain = (qkv, *(torch.zeros(12, 4, 16, 128, device="cuda", dtype=BF16) for _ in range(2)), tab, lens, cos, sin, 16, c, False)
        assert f(*plain, at.long()) is None and f(*plain, at[:-1]) is None and f(*plain, at, at) is None


def test_leaves_the_rest_alone(ways):
    common, *_ = ways
    f = common.fast()
    t = torch.zeros(2, 16, 128, device="cuda", dtype=BF16)
    for name, n in (("mass", 9), ("evict", 8), ("bounds", 5), ("select", 8), ("sparse", 9)):
        call = getattr(f, name)
        assert call() is None and call(*[None] * n) is None and call(*[t] * n) is None and call(*[1] * n) is None
