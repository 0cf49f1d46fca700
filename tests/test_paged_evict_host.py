"""PagedKVCache's eviction on the CPU: pages, lengths, shared pages and what follows the pages, against a model that keeps every
stream's positions in plain lists.  The device operators are replaced by index arithmetic."""
import random

import pytest
import torch

from sonata_b200.kernels import paged_evict as PE
from sonata_b200.kernels import paged_kv as PK
from sonata_b200.kernels import paged_sparse as PS


@pytest.fixture
def cpu(monkeypatch):
    def copy(pool, src, dst, stream=None):
        assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == dst.numel()
        at = (slice(None),) * (pool.dim() - 4)
        pool[(*at, dst.long())] = pool[(*at, src.long())].clone()

    def evict(pool, table, lens, mass, keep, recent=0, sinks=0, return_source=False, stream=None):
        page = pool.shape[4]
        for s, n in enumerate(lens.tolist()):
            if n <= keep:
                continue
            pg, at = table[s, torch.arange(n) // page].long(), torch.arange(n) % page
            for layer in range(pool.shape[0]):
                old = mass[layer, s, 0, :n].tolist()
                best = sorted(range(sinks, n - recent), key=lambda i: (-old[i], i))[:keep - recent - sinks]
                move = sorted(i for i in best if i >= keep - recent)
                src = [i if i < sinks or i in best else move.pop(0) for i in range(keep - recent)] + list(range(n - recent, n))
                for kv in range(2):
                    rows = pool[layer, kv, pg, 0, at]
                    pool[layer, kv, pg[:keep], 0, at[:keep]] = rows[src]
                mass[layer, s, 0, :keep] = torch.tensor(old)[src]
                mass[layer, s, 0, keep:n] = 0

    def bounds(k, b, table, lens, cu_seqlens=None, stream=None):
        for s, n in enumerate(lens.tolist()):
            new = 1 if cu_seqlens is None else int(cu_seqlens[s + 1] - cu_seqlens[s])
            for blk in range((n - new) // k.shape[2], -(-n // k.shape[2]) if new else 0):
                pg = int(table[s, blk])
                rows = k[pg, :, :n - blk * k.shape[2]]
                b[pg] = torch.stack([rows.amin(1), rows.amax(1)], 1)

    monkeypatch.setattr(PK, "copy_pages", copy)
    monkeypatch.setattr(PE, "evict_positions", evict)
    monkeypatch.setattr(PS, "update_page_bounds", bounds)
    return bounds


def make(pages=60, slots=4, page=4, width=16, bounds=False):
    c = PK.PagedKVCache(2, pages, 1, 1, slots, width, page_size=page, device="cpu")
    c.track_mass()
    if bounds:
        c.track_bounds()
    return c


def write(c, slot, values, update=None):
    n = c.lens[slot]
    counts = [0] * len(c.lens)
    counts[slot] = len(values)
    c.reserve(counts)
    for i, v in enumerate(values):
        page, at = c.page_table[slot, (n + i) // c.page_size].item(), (n + i) % c.page_size
        assert page >= 0 and c.mass[:, slot, 0, n + i].eq(0).all()
        c.pool[:, :, page, 0, at, 0] = v
        c.mass[0, slot, 0, n + i], c.mass[1, slot, 0, n + i] = v * 37 % 101, v * 53 % 103
    if update and values:
        for layer in range(2):
            new = [len(values) if s == slot else 0 for s in range(len(c.lens))]
            update(c.k(layer), c.bounds[layer], c.page_table, c.seq_lens, torch.tensor([sum(new[:i]) for i in range(len(new) + 1)]))


def read(c, slot, layer=1):
    n = c.seq_lens[slot].item()
    return [c.pool[layer, 1, c.page_table[slot, i // c.page_size].item(), 0, i % c.page_size, 0].item() for i in range(n)]


def consistent(c):
    users = [0] * c.num_pages
    for s, pages in enumerate(c.pages):
        assert len(pages) == -(-c.lens[s] // c.page_size)
        assert c.page_table[s].tolist() == pages + [-1] * (c.max_pages - len(pages))
        for p in pages:
            users[p] += 1
        assert c.mass[:, s, :, c.lens[s]:].eq(0).all()
    assert users == c._users and sorted(c._free) == [p for p, n in enumerate(users) if n == 0]
    assert c.seq_lens.tolist() == c.lens
    for s, pages in enumerate(c.pages):
        if c.lens[s] % c.page_size:
            assert users[pages[-1]] == 1
        if c.bounds is not None:
            for blk, pg in enumerate(pages):
                k = c.pool[:, 0, pg, 0, :c.lens[s] - blk * c.page_size, 0]
                assert torch.equal(c.bounds[:, pg, 0, :, 0], torch.stack([k.amin(1), k.amax(1)], 1))


@pytest.mark.parametrize("seed", range(8))
def test_random_histories(cpu, seed):
    rng = random.Random(seed)
    c, want, stamp = make(bounds=seed % 2 == 0), [[] for _ in range(4)], 0
    for _ in range(120):
        op, s = rng.choice(["append"] * 4 + ["fork", "free", "compact", "evict"]), rng.randrange(4)
        if op == "append":
            vals = [float((stamp + i) % 200 + 1) for i in range(rng.randrange(0, 9))]
            stamp += len(vals)
            try:
                write(c, s, vals, cpu if c.bounds is not None else None)
                want[s] += vals
            except (RuntimeError, ValueError):
                pass  # full: nothing may have changed
        elif op == "fork":
            d = rng.randrange(4)
            if not want[d] and d != s:
                try:
                    c.fork(s, d)
                    want[d] = list(want[s])
                except RuntimeError:
                    pass
        elif op == "free":
            c.free(s)
            want[s] = []
        elif op == "compact":
            c.compact()
        else:
            keep = rng.randrange(1, 30)
            recent = rng.randrange(keep + 1)
            sinks = rng.randrange(keep - recent + 1)
            try:
                cut = c.evict(keep, recent, sinks)
            except RuntimeError:
                consistent(c)
                continue
            assert cut == [i for i in range(4) if len(want[i]) > keep]
            for i in cut:
                got = read(c, i)
                old = want[i]
                assert len(got) == keep and got[:sinks] == old[:sinks] and got[keep - recent:] == old[len(old) - recent:]
                free = old[sinks:len(old) - recent]
                best = sorted(range(len(free)), key=lambda j: (-(free[j] * 53 % 103), j))[:keep - recent - sinks]
                # places may have been rearranged before, so ties may go either way: weights are compared
                assert sorted(v * 53 % 103 for v in got[sinks:keep - recent]) == sorted(free[j] * 53 % 103 for j in best)
                want[i] = got
        consistent(c)
        assert [read(c, i) for i in range(4)] == want


def test_forked_streams_are_cut_apart(cpu):
    c = make()
    write(c, 0, [float(i + 1) for i in range(30)])
    c.fork(0, 1)
    c.fork(0, 2)
    write(c, 1, [200.0])
    before, free = read(c, 0), c.free_pages
    assert c.evict(30, 4) == [1]
    consistent(c)
    assert read(c, 0) == read(c, 2) == before and c.lens == [30, 30, 30, 0] and read(c, 1)[-4:] == [28.0, 29.0, 30.0, 200.0]
    assert c.free_pages == free - 7  # its seven full pages became its own; the eighth, partly filled, was
    assert c.evict(8, 4) == [0, 1, 2]
    consistent(c)


def test_bounds_of_what_is_there(cpu):
    """track_bounds after the first tokens: their pages' bounds, too."""
    c = make()
    write(c, 0, [float(i * 7 % 31) for i in range(30)])
    write(c, 2, [5.0])
    c.fork(0, 1)
    assert c.track_bounds() is c.track_bounds() is c.bounds
    consistent(c)
    c.evict(9, 3)
    consistent(c)


def test_limits(cpu):
    c = make(pages=9)
    write(c, 0, [1.0] * 29)
    c.fork(0, 1)
    assert c.free_pages == 0
    lens, pages = list(c.lens), [list(p) for p in c.pages]
    with pytest.raises(RuntimeError):
        c.evict(8, 4)  # two pages for the first of them, none free
    assert c.lens == lens and c.pages == pages
    consistent(c)
    for bad in ((0,), (4, 5), (4, -1), (4, 0, -1), (4, 2, 3)):
        with pytest.raises(ValueError):
            c.evict(*bad)
    assert c.evict(29) == []
    with pytest.raises(RuntimeError):
        PK.PagedKVCache(1, 1, 1, 1, 1, 1, device="cpu").evict(1)


def test_budget_passes_errors_on(cpu):
    """A budget's cut waits for free pages, and for nothing else."""
    from sonata_b200.kernels import serve
    r = object.__new__(serve.RaggedZonos)
    r.budget, r.recent, r.sinks, r.cache = 8, 4, 1, make(pages=9)
    write(r.cache, 0, [1.0] * 29)
    r.cache.fork(0, 1)
    r._cut()  # two pages for the first of them, none free
    assert r.cache.lens == [29, 29, 0, 0]
    r.cache.free(1)

    def fail(*args, **kwargs):
        raise RuntimeError("of the device")

    right, PE.evict_positions = PE.evict_positions, fail  # the fixture puts the operator back
    with pytest.raises(RuntimeError, match="of the device"):
        r._cut()
    assert r.cache.lens == [29, 0, 0, 0]
    PE.evict_positions = right
    r._cut()
    assert r.cache.lens == [8, 0, 0, 0]


def test_budget_refusals():
    from sonata_b200.kernels import serve
    for bad in (dict(budget=0, recent=0, sinks=0), dict(budget=8, recent=-1, sinks=1), dict(budget=8, recent=1, sinks=-1),
                dict(budget=8, recent=4, sinks=5), dict(budget=80, attend_blocks=8), dict(budget=80, max_len=PE.EVICT_MOST + 1)):
        with pytest.raises(ValueError):
            serve.RaggedZonos(None, num_pages=9, **{"max_len": 100, **bad})


def kept(old, keep, recent):
    """The values of a stream cut to `keep`, by the weights that write() gives layer 1 (in any order)."""
    free = sorted(old[:len(old) - recent], key=lambda v: -(v * 53 % 103))
    return sorted(free[:keep - recent] + old[len(old) - recent:])


@pytest.mark.parametrize("bounds", [False, True])
def test_a_cut_that_needs_no_pages_goes_first(cpu, bounds):
    """No free page, two streams that share all of theirs and one that shares none: its pages serve the others' copies."""
    c, update = make(pages=15, bounds=bounds), cpu if bounds else None
    write(c, 1, [float(i + 1) for i in range(28)], update)
    c.fork(1, 0)
    write(c, 2, [float(i + 40) for i in range(29)], update)
    assert c.free_pages == 0
    before = [read(c, s) for s in range(3)]
    assert c.evict(8, 4) == [0, 1, 2] and c.lens == [8, 8, 8, 0] and c.free_pages == 15 - 6
    consistent(c)
    for s in range(3):
        assert sorted(read(c, s)) == kept(before[s], 8, 4) and read(c, s)[4:] == before[s][-4:]


def test_streams_without_pages_for_their_copies_are_left(cpu):
    c = make(pages=15)
    write(c, 1, [float(i + 1) for i in range(28)])
    c.fork(1, 0)
    write(c, 2, [float(i + 40) for i in range(29)])
    before, mass = [read(c, s) for s in range(3)], c.mass.clone()
    assert c.evict(24, 4) == [2] and c.lens == [28, 28, 24, 0] and c.free_pages == 2  # six copies for either of the others
    consistent(c)
    assert [read(c, 0), read(c, 1)] == before[:2] and torch.equal(c.mass[:, :2], mass[:, :2])
    assert sorted(read(c, 2)) == kept(before[2], 24, 4)
    with pytest.raises(PK.OutOfPages):  # nothing that can be cut
        c.evict(24, 4)
    consistent(c)
    assert c.lens == [28, 28, 24, 0]
    c.free(2)
    assert c.evict(24, 4) == [0, 1] and c.lens == [24, 24, 0, 0]
    consistent(c)
    for s in range(2):
        assert sorted(read(c, s)) == kept(before[s], 24, 4)


def test_budget_of_a_stream_beside_shared_ones(cpu):
    """RaggedZonos: a stream of pages of its own is cut although others, which share theirs, would need free ones."""
    from sonata_b200.kernels import serve
    r = object.__new__(serve.RaggedZonos)
    r.budget, r.recent, r.sinks, r.cache = 20, 4, 1, make(pages=24)
    write(r.cache, 0, [1.0] * 40)
    r.cache.fork(0, 1)
    write(r.cache, 2, [2.0] * 56)
    assert r.cache.free_pages == 0
    r._cut()
    assert r.cache.lens == [20, 20, 20, 0]
    r.cache.reserve([1, 1, 1, 0])


def test_streams_over_a_budget_are_cut_together(cpu):
    """No stream is cut before one has four pages more than the budget; then all that are over it are, and no other."""
    from sonata_b200.kernels import serve
    r = object.__new__(serve.RaggedZonos)
    r.budget, r.recent, r.sinks, r.cache = 8, 4, 1, make()
    for slot, n in enumerate((9, 23, 8, 3)):
        write(r.cache, slot, [float(i + 1) for i in range(n)])
    r._cut()
    assert r.cache.lens == [9, 23, 8, 3]
    write(r.cache, 1, [24.0])
    r._cut()
    assert r.cache.lens == [8, 8, 8, 3]
    consistent(r.cache)
