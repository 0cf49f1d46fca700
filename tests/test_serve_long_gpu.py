"""Long streams end to end: RaggedZonos with a budget of cached positions, and with steps that attend to some of the blocks.

Where nothing is cut or left out the logits are those without the options, bit for bit; where positions leave, they are those
of a run in which a plain implementation moves them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda_lib):
    from sonata_b200.kernels import decode_step as DS
    cfg = DS.ZonosBackboneConfig(n_layer=4, attn_layer_idx=[1, 3])
    return cfg, DS.SyntheticZonos(cfg, batch=3, context=0, max_seqlen=8, seed=7)


def run(model, steps=70, check=None, partial=True, **options):
    """Prompts of two streams, a third one forked, a second piece of a prompt, steps of all and of some streams, a free."""
    from sonata_b200.kernels import serve
    cfg, m = model
    g = torch.Generator(device="cuda").manual_seed(3)
    x = lambda n: torch.randn(n, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    r = serve.RaggedZonos(m, num_pages=90, max_len=400, **options)
    out = [r.prompt(x(177), [37, 140, 0])]
    r.fork(1, 2)
    out.append(r.prompt(x(23), [20, 0, 3]))
    for t in range(steps):
        if partial and t % 7 == 3:
            out.append(r.step(x(3), active=[True, False, t % 2 == 0]))
        else:
            out.append(r.step(x(3)))
        if check:
            check(r)
    r.cache.compact()
    out.append(r.step(x(3)))
    r.free(1)
    out.append(r.step(x(3)))
    out.append(r.prompt(x(9), [0, 9, 0]))
    out.append(r.step(x(3)))
    torch.cuda.synchronize()
    return r, out


def test_nothing_cut(model, cuda_lib):
    _, want = run(model)
    r, got = run(model, budget=1000)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert r.cache.lens == r.seen
    # every step's weights of a head's four query heads add up to 4, a prompt's last 32 tokens' to 4 each: positions of the
    # stream that was freed and started again
    total = r.cache.mass.sum(-1)[:, 1]
    assert ((total - 4 * (9 + 1)).abs() < 1e-3).all()
    assert cuda_lib.sn_device_status(1, None) == 0


def test_all_blocks(model, cuda_lib):
    _, want = run(model)
    r, got = run(model, attend_blocks=25)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    for layer in range(2):
        for s in range(3):
            for blk, pg in enumerate(r.cache.pages[s]):
                k = r.cache.k(layer)[pg, :, :min(16, r.cache.lens[s] - 16 * blk)]
                assert torch.equal(r.cache.bounds[layer, pg], torch.stack([k.amin(1), k.amax(1)], 1))
    assert cuda_lib.sn_device_status(1, None) == 0


def test_budget(model, cuda_lib, monkeypatch):
    from sonata_b200.kernels import paged_evict as PE
    from test_paged_evict_gpu import evict_truth

    def check(r):
        assert max(r.cache.lens) < 64 + 64 and all(n <= s for n, s in zip(r.cache.lens, r.seen))
        assert sum(map(len, r.cache.pages)) <= 3 * 8

    r, got = run(model, check=check, budget=64, recent=24, sinks=2)
    assert max(r.cache.lens) < max(r.seen) and all(torch.isfinite(t).all() for t in got)
    cuts = []

    def plain(pool, table, lens, mass, keep, recent=0, sinks=0):
        cuts.append(lens.tolist())
        p, m, _ = evict_truth(pool, table, lens.tolist(), mass, keep, recent, sinks)
        pool.copy_(p)
        mass.copy_(m)

    monkeypatch.setattr(PE, "evict_positions", plain)
    r2, want = run(model, budget=64, recent=24, sinks=2)
    assert len(cuts) == 2 and r.cache.lens == r2.cache.lens  # after the first prompt, and when a stream has 128 again
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert cuda_lib.sn_device_status(1, None) == 0


def test_some_blocks(model, cuda_lib, monkeypatch):
    from sonata_b200.kernels import paged_sparse as PS
    from test_paged_sparse_gpu import select_truth
    r, got = run(model, attend_blocks=5)
    assert all(torch.isfinite(t).all() for t in got)
    _, all_blocks = run(model)
    assert not all(torch.equal(a, b) for a, b in zip(got, all_blocks, strict=True))

    def plain(q, bounds, table, lens, page, count, first=1, last=1):
        return select_truth(q, bounds, table, lens.tolist(), page, count, first, last)

    monkeypatch.setattr(PS, "select_blocks", plain)
    _, want = run(model, attend_blocks=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    assert cuda_lib.sn_device_status(1, None) == 0


def test_refusals(model):
    from sonata_b200.kernels import serve
    for bad in (dict(budget=64, attend_blocks=8), dict(budget=64, recent=64, sinks=1), dict(attend_blocks=2)):
        with pytest.raises(ValueError):
            serve.RaggedZonos(model[1], num_pages=9, max_len=100, **bad)
    r = serve.RaggedZonos(model[1], num_pages=20, max_len=100, budget=20, recent=8)
    x = torch.zeros(3, model[0].d_model, device="cuda", dtype=torch.bfloat16)
    r.prompt(x[:1].expand(99, -1).contiguous(), [99, 0, 0])
    assert r.cache.lens == [20, 0, 0] and r.seen == [99, 0, 0]
    r.step(x)
    with pytest.raises(ValueError):  # max_len counts positions, not what is cached
        r.step(x)
    assert r.cache.lens == [21, 0, 0]
