"""PagedKVCache's book-keeping on the CPU: reserve, fork, free, compact against a model that keeps every stream's
positions in plain lists.  The device copy is replaced by an index copy."""
import random

import pytest
import torch

from sonata_b200.kernels import paged_kv as PK


@pytest.fixture
def cpu_copy(monkeypatch):
    def copy(pool, src, dst, stream=None):
        assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == dst.numel()
        pool[:, :, dst.long()] = pool[:, :, src.long()].clone()
    monkeypatch.setattr(PK, "copy_pages", copy)


def make(pages=40, slots=4, page=4, width=16):
    return PK.PagedKVCache(2, pages, 1, 1, slots, width, page_size=page, device="cpu")


def write(c, slot, values):
    """Appends values to a stream as the kernel would, through its table."""
    n = c.lens[slot]
    counts = [0] * len(c.lens)
    counts[slot] = len(values)
    c.reserve(counts)
    for i, v in enumerate(values):
        page, at = c.page_table[slot, (n + i) // c.page_size].item(), (n + i) % c.page_size
        assert page >= 0
        c.pool[:, :, page, 0, at, 0] = v


def read(c, slot):
    n = c.seq_lens[slot].item()
    return [c.pool[1, 1, c.page_table[slot, i // c.page_size].item(), 0, i % c.page_size, 0].item() for i in range(n)]


def consistent(c):
    users = [0] * c.num_pages
    for s, pages in enumerate(c.pages):
        assert len(pages) == -(-c.lens[s] // c.page_size)
        assert c.page_table[s].tolist() == pages + [-1] * (c.max_pages - len(pages))
        for p in pages:
            users[p] += 1
    assert users == c._users and sorted(c._free) == [p for p, n in enumerate(users) if n == 0]
    assert c.seq_lens.tolist() == c.lens
    for s, pages in enumerate(c.pages):  # the partly filled page is nobody else's
        if c.lens[s] % c.page_size:
            assert users[pages[-1]] == 1


@pytest.mark.parametrize("seed", range(8))
def test_random_histories(cpu_copy, seed):
    rng = random.Random(seed)
    c, want, stamp = make(), [[] for _ in range(4)], 0
    for _ in range(150):
        op, s = rng.choice(["append", "append", "append", "fork", "free", "compact"]), rng.randrange(4)
        if op == "append":
            vals = [float((stamp + i) % 200) for i in range(rng.randrange(0, 9))]
            stamp += len(vals)
            try:
                write(c, s, vals)
                want[s] += vals
            except (RuntimeError, ValueError):
                pass  # full: nothing may have changed
        elif op == "fork":
            d = rng.randrange(4)
            if want[d] or d == s:
                with pytest.raises(ValueError):
                    c.fork(s, d)
            else:
                try:
                    c.fork(s, d)
                    want[d] = list(want[s])
                except RuntimeError:
                    pass
        elif op == "free":
            c.free(s)
            want[s] = []
        else:
            used = c.num_pages - c.free_pages
            c.compact()
            assert all(p < used for pages in c.pages for p in pages)
        consistent(c)
        assert [read(c, i) for i in range(4)] == want


def test_limits(cpu_copy):
    c = make(pages=5, slots=2, page=4, width=4)
    with pytest.raises(ValueError):
        c.reserve([17, 0])  # more than a stream's table holds
    with pytest.raises(ValueError):
        c.reserve([1])
    with pytest.raises(ValueError):
        c.reserve([-1, 0])
    c.reserve([13, 0])
    with pytest.raises(RuntimeError):
        c.reserve([0, 8])
    assert c.lens == [13, 0] and c.free_pages == 1
    c.reserve([0, 4])
    with pytest.raises(RuntimeError):
        make(pages=1, slots=2).reserve([1, 4])
    d = make(pages=1, slots=2)
    d.reserve([3, 0])
    with pytest.raises(RuntimeError):
        d.fork(0, 1)
    consistent(d)
    with pytest.raises(ValueError):
        PK.PagedKVCache(1, 0, 1, 1, 1, 1, device="cpu")
