"""What evict_positions launches, on a runtime without a device (fake_cudart.cpp): the plan has put the weights in order when the
moves are launched, so what these need is found out before."""
import ctypes
import subprocess
from pathlib import Path

import pytest

from sonata_b200 import _lib, build

PTR = ctypes.c_void_p(256)  # never dereferenced


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    build.build()
    src, obj = build.CSRC / "paged_evict.cu", build.BUILD / "paged_evict.o"
    if not obj.exists() or obj.stat().st_mtime < src.stat().st_mtime:
        build.BUILD.mkdir(exist_ok=True)
        build._compile(src)
    where = tmp_path_factory.mktemp("fake")
    cuda = Path(build.nvcc()).resolve().parent.parent
    subprocess.run(["g++", "-O1", "-fPIC", "-shared", "-I", str(cuda / "include"), str(Path(__file__).with_name("fake_cudart.cpp")), str(obj), "-o",
                    str(where / "lib.so"), "-Wl,-Bsymbolic"], check=True)

    def load(name, *answers):  # a library of its own: what a device has answered is kept
        path = where / f"{name}.so"
        path.write_bytes((where / "lib.so").read_bytes())
        lib = ctypes.CDLL(str(path))
        lib.fake_set(*answers)
        lib.sn_evict_positions.argtypes, lib.sn_evict_positions.restype = _lib.SIGNATURES["sn_evict_positions"]
        lib.sn_evict_workspace_size.argtypes, lib.sn_evict_workspace_size.restype = _lib.SIGNATURES["sn_evict_workspace_size"]
        return lib

    return load


def evict(lib, layers, hd=128):
    room = 16 * 2000
    return lib.sn_evict_positions(PTR, layers, 9000, 16, 4, hd, PTR, 2000, 2000, PTR, PTR, 4 * room, 4 * room, room, 1, 64, 8, 1, None, PTR,
                                  lib.sn_evict_workspace_size(layers, 1, 4, room, 64), None)


@pytest.mark.parametrize("hd", [128, 64, 96, 7])
@pytest.mark.parametrize("name,answers,want", [("all", (1, 4), 16), ("attribute", (0, 4), 8), ("none fits", (1, 0), 8), ("not answered", (1, -1), 8)])
def test_large_clusters_that_a_device_refuses(fake, hd, name, answers, want):
    lib = fake(f"{name} {hd}", *answers)
    for n in (2, 4):  # the second call goes by what the first has found
        assert evict(lib, 1, hd) == _lib.SN_OK
        assert lib.fake_launches() == n and [lib.fake_cluster(i) for i in range(n)] == [1, want] * (n // 2)


def test_many_rows_take_portable_clusters(fake):
    lib = fake("many", 0, 0)
    assert evict(lib, 12) == _lib.SN_OK
    assert lib.fake_launches() == 2 and lib.fake_cluster(1) == 7
