"""Host-side argument checks of the prompt and paged-cache entry points: no device is touched."""
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


def prompt(L, **k):
    a = dict(zx=p, ld=8512, cs=p, cw=p, cb=p, ss=p, A=p, D=p, dtb=p, y=p, cu=p, batch=2, tokens=10, di=4096, ng=1, ds=128, nh=64,
             hd=64, W=4, gate=0, ws=p, wsb=BIG, stream=None)
    a.update(k)
    return L.sn_mamba2_prompt(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(zx=None), -1), (dict(cs=None), -1), (dict(ss=None), -1), (dict(A=None), -1), (dict(y=None), -1), (dict(ws=None), -1),
    (dict(batch=0), -1), (dict(tokens=-1), -1), (dict(cu=None), -1), (dict(ld=8511), -1), (dict(hd=32), -1), (dict(ng=3), -1),
    (dict(W=0), -1), (dict(W=9), -1), (dict(wsb=64), -1), (dict(ds=257, ld=1 << 20), -3), (dict(tokens=0), 0)])
def test_mamba2_prompt(L, change, rc):
    assert prompt(L, **change) == rc


def test_workspace_sizes(L):
    assert L.sn_mamba2_prompt_workspace_size(-1, 1, 4096, 1, 128, 64) == 0
    assert L.sn_mamba2_prompt_workspace_size(100, 0, 4096, 1, 128, 64) == 0
    sizes = [L.sn_mamba2_prompt_workspace_size(t, 3, 4096, 1, 128, 64) for t in (1, 100, 1000, 100000)]
    assert 0 < sizes[0] <= sizes[1] < sizes[2] < sizes[3]
    assert L.sn_paged_decode_workspace_size(0, 16, 128) == 0
    assert 0 < L.sn_paged_decode_workspace_size(1, 16, 128) <= L.sn_paged_decode_workspace_size(100, 16, 128)


def append(L, **k):
    a = dict(qkv=p, ld=24 * 128, q=p, kp=p, kps=8192, khs=2048, kts=128, vp=p, vps=8192, vhs=2048, vts=128, np=8, page=16, tab=p,
             ts=4, mp=4, lens=p, cu=p, cos=p, sin=p, max_pos=64, tokens=5, batch=2, hq=16, hkv=4, hd=128, rot=128, inter=0, stream=None)
    a.update(k)
    return L.sn_rotary_paged_append(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(qkv=None), -1), (dict(q=None), -1), (dict(kp=None), -1), (dict(tab=None), -1), (dict(lens=None), -1), (dict(cos=None), -1),
    (dict(ld=24 * 128 - 1), -1), (dict(hd=127), -1), (dict(rot=130), -1), (dict(rot=3), -1), (dict(page=0), -1), (dict(ts=3), -1),
    (dict(max_pos=0), -1), (dict(cu=None), -1), (dict(kts=64), -1), (dict(np=0), -1), (dict(hkv=0), -1), (dict(tokens=-1), -1),
    (dict(tokens=0), 0)])
def test_rotary_paged_append(L, change, rc):
    assert append(L, **change) == rc


def attend(L, **k):
    a = dict(q=p, qb=2048, qh=128, kp=p, kps=8192, khs=2048, kts=128, vp=p, vps=8192, vhs=2048, vts=128, np=8, page=16, tab=p, ts=4,
             mp=4, lens=p, out=p, lse=None, scale=0.1, batch=2, hq=16, hkv=4, hd=128, ws=p, wsb=BIG, stream=None)
    a.update(k)
    return L.sn_paged_decode_attention(*a.values())


@pytest.mark.parametrize("change,rc", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(hq=15), -1), (dict(hkv=0), -1), (dict(wsb=0), -1),
    (dict(page=0), -1), (dict(ts=3), -1), (dict(batch=0), -1), (dict(kts=64), -1), (dict(qb=-1), -1),
    (dict(hd=257, kps=BIG, khs=BIG, kts=BIG, vps=BIG, vhs=BIG, vts=BIG), -3), (dict(mp=1 << 28, ts=1 << 28), -3)])
def test_paged_decode_attention(L, change, rc):
    assert attend(L, **change) == rc


@pytest.mark.parametrize("args,rc", [
    ((None, 1024, 64, 64, 2, 16, p, p, 3, None), -1), ((p, 1024, 64, 64, 2, 16, None, p, 3, None), -1),
    ((p, 1024, 32, 64, 2, 16, p, p, 3, None), -1), ((p, 32, 64, 64, 2, 16, p, p, 3, None), -1), ((p, 1024, 64, 64, 2, 16, p, p, -1, None), -1),
    ((p, 1024, 64, 64, 70000, 16, p, p, 3, None), -3), ((p, 1024, 64, 64, 2, 16, None, None, 0, None), 0)])
def test_copy_pages(L, args, rc):
    assert L.sn_copy_pages(*args) == rc
