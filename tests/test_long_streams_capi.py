"""Host-side argument checks of the entry points for long streams: no device is touched."""
import ctypes

import pytest

from sonata_b200 import _lib

p = ctypes.c_void_p(256)  # never dereferenced: validation fails first
BIG = 1 << 30


@pytest.fixture(scope="module")
def L():
    from sonata_b200 import build
    build.build()
    return _lib.lib()


POOLS = dict(kp=p, kps=8192, khs=2048, kts=128, vp=p, vps=8192, vhs=2048, vts=128, np=8, page=16, tab=p, ts=4, mp=4, lens=p)


def mass(L, **k):
    a = dict(q=p, qb=2048, qh=128, **POOLS, mass=p, mb=256, mh=64, out=p, lse=None, scale=0.1, batch=2, hq=16, hkv=4, hd=128, ws=p, wsb=BIG,
             stream=None)
    a.update(k)
    return L.sn_paged_decode_attention_mass(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(mass=None), -1), (dict(ws=None), -1), (dict(hq=15), -1), (dict(hkv=0), -1), (dict(wsb=0), -1),
    (dict(wsb=4096), -1), (dict(page=0), -1), (dict(ts=3), -1), (dict(batch=0), -1), (dict(kts=64), -1), (dict(mh=63), -1), (dict(mb=63), -1),
    (dict(ws=ctypes.c_void_p(264)), -2), (dict(hd=257, kps=BIG, khs=BIG, kts=BIG, vps=BIG, vhs=BIG, vts=BIG), -3),
    (dict(mp=1 << 28, ts=1 << 28, mb=1 << 40, mh=1 << 33), -3)])
def test_mass(L, change, rc):
    assert mass(L, **change) == rc


def test_mass_workspace(L):
    f = L.sn_paged_mass_workspace_size
    for bad in ((0, 16, 4, 128, 100), (1, 0, 4, 128, 100), (1, 16, 3, 128, 100), (1, 16, 4, 0, 100), (1, 16, 4, 128, 0), (1, 16, 0, 128, 100)):
        assert f(*bad) == 0
    assert L.sn_paged_decode_workspace_size(2, 16, 128) < f(2, 16, 4, 128, 100) < f(2, 16, 4, 128, 1000) < f(3, 16, 4, 128, 1000)
    assert f(3, 33, 1, 128, 1 << 20) >= 3 * 33 * (1 << 20) * 4


def evict(L, **k):
    a = dict(pool=p, layers=2, np=8, page=16, hkv=4, hd=128, tab=p, ts=4, mp=4, lens=p, mass=p, ml=512, mb=256, mh=64, batch=2, keep=32, recent=8,
             sinks=1, source=None, ws=p, wsb=BIG, stream=None)
    a.update(k)
    return L.sn_evict_positions(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(pool=None), -1), (dict(tab=None), -1), (dict(lens=None), -1), (dict(mass=None), -1), (dict(layers=0), -1), (dict(np=0), -1), (dict(page=0), -1),
    (dict(hkv=0), -1), (dict(hd=0), -1), (dict(mp=0), -1), (dict(ts=3), -1), (dict(batch=0), -1), (dict(keep=0), -1), (dict(recent=-1), -1),
    (dict(sinks=-1), -1), (dict(recent=32), -1), (dict(recent=31, sinks=2), -1), (dict(mh=63), -1), (dict(mb=63), -1), (dict(ml=63), -1),
    (dict(ws=None), -1), (dict(wsb=2 * 2 * 4 * (64 * 4 + 8)), -1), (dict(wsb=2 * 2 * 4 * (64 * 4 + 8) + 16, batch=0), -1), (dict(ws=ctypes.c_void_p(264)), -2),
    (dict(mp=32769, ts=32769, ml=BIG, mb=BIG, mh=BIG), -3), (dict(hd=8193), -3), (dict(batch=1 << 28, wsb=1 << 50), -3)])
def test_evict(L, change, rc):
    assert evict(L, **change) == rc


def test_evict_workspace(L):
    f = L.sn_evict_workspace_size
    assert f(0, 1, 1, 1, 1) == f(1, 0, 1, 1, 1) == f(1, 1, 0, 1, 1) == f(1, 1, 1, 0, 1) == f(1, 1, 1, 1, 0) == 0
    assert 0 < f(1, 2, 4, 100, 9) < f(2, 2, 4, 100, 9) < f(2, 2, 4, 100, 50) == f(2, 2, 4, 100, 90) < f(2, 2, 4, 1000, 90)
    assert f(12, 48, 4, 30000, 2048) < 40 << 20  # lists of at most keep pairs
    assert f(12, 300, 8, 1 << 19, 1 << 18) > 1 << 36


def bounds(L, **k):
    a = dict(kp=p, kps=8192, khs=2048, kts=128, np=8, page=16, tab=p, ts=4, mp=4, lens=p, cu=p, batch=2, hkv=4, hd=128, bounds=p, stream=None)
    a.update(k)
    return L.sn_update_page_bounds(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(kp=None), -1), (dict(tab=None), -1), (dict(lens=None), -1), (dict(bounds=None), -1), (dict(kts=127), -1), (dict(khs=127), -1), (dict(page=0), -1),
    (dict(ts=3), -1), (dict(batch=0), -1), (dict(hkv=0), -1), (dict(hd=0), -1), (dict(mp=1 << 28, ts=1 << 28), -3)])
def test_update_page_bounds(L, change, rc):
    assert bounds(L, **change) == rc


def select(L, **k):
    a = dict(q=p, qb=2048, qh=128, bounds=p, np=8, page=16, tab=p, ts=4, mp=4, lens=p, batch=2, hq=16, hkv=4, hd=128, count=3, first=1, last=1, blocks=p,
             ws=p, wsb=BIG, stream=None)
    a.update(k)
    return L.sn_select_blocks(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(q=None), -1), (dict(bounds=None), -1), (dict(tab=None), -1), (dict(lens=None), -1), (dict(blocks=None), -1), (dict(hq=15), -1), (dict(count=0), -1),
    (dict(first=-1), -1), (dict(last=-1), -1), (dict(first=2, last=2), -1), (dict(first=4), -1), (dict(qb=-1), -1), (dict(page=0), -1), (dict(ts=3), -1),
    (dict(ws=None), -1), (dict(wsb=2 * 4 * 4 * 16 - 1), -1), (dict(ws=ctypes.c_void_p(264)), -2), (dict(mp=262145, ts=262145), -3)])
def test_select_blocks(L, change, rc):
    assert select(L, **change) == rc


def test_select_workspace(L):
    f = L.sn_select_blocks_workspace_size
    assert f(0, 4, 10) == f(1, 0, 10) == f(1, 4, 0) == 0
    assert 0 < f(1, 4, 10) < f(2, 4, 10) < f(2, 4, 1000)
    assert f(3000, 8, 200000) > 1 << 36


def sparse(L, **k):
    a = dict(q=p, qb=2048, qh=128, **POOLS, blocks=p, count=3, out=p, lse=None, scale=0.1, batch=2, hq=16, hkv=4, hd=128, ws=p, wsb=BIG, stream=None)
    a.update(k)
    return L.sn_paged_sparse_attention(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(blocks=None), -1), (dict(count=0), -1), (dict(ws=None), -1), (dict(hq=15), -1), (dict(wsb=0), -1),
    (dict(page=0), -1), (dict(ts=3), -1), (dict(count=1 << 28), -3), (dict(hd=257, kps=BIG, khs=BIG, kts=BIG, vps=BIG, vhs=BIG, vts=BIG), -3)])
def test_sparse(L, change, rc):
    assert sparse(L, **change) == rc


def test_append_at(L):
    a = dict(qkv=p, ld=24 * 128, q=p, kp=p, kps=8192, khs=2048, kts=128, vp=p, vps=8192, vhs=2048, vts=128, np=8, page=16, tab=p, ts=4, mp=4, lens=p,
             cu=p, pos=p, cos=p, sin=p, max_pos=64, tokens=5, batch=2, hq=16, hkv=4, hd=128, rot=128, inter=0, stream=None)
    for change, rc in ((dict(pos=None), -1), (dict(qkv=None), -1), (dict(rot=130), -1), (dict(tokens=0), 0), (dict(tokens=0, pos=None), 0)):
        assert L.sn_rotary_paged_append_at(*{**a, **change}.values()) == rc


@pytest.mark.parametrize("reach", [2**31 - 1, 2**31 - 3])
def test_steps_past_2_31(L, reach):
    """Position by position, four at a time, a step from the last of so many would not fit into 32 bits."""
    few = dict(hd=1, hq=1, hkv=1, batch=1, qb=1, qh=1, page=reach, mp=1, ts=1, kps=reach, khs=reach, kts=1, vps=reach, vhs=reach, vts=1, mh=reach,
               mb=reach, wsb=1 << 50)
    assert mass(L, **few) == -3
    a = dict(q=p, qb=2048, qh=128, **POOLS, out=p, lse=None, scale=0.1, batch=2, hq=16, hkv=4, hd=128, ws=p, wsb=BIG, stream=None)
    a.update({k: v for k, v in few.items() if k in a})
    assert L.sn_paged_decode_attention(*a.values()) == -3
