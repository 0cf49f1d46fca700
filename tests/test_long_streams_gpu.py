"""The operators of long streams together and at their limits: pages past 2^31 elements, workspaces that two captured graphs
share, streams other than the current one, calls repeated on what the last one left."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from sonata_b200.kernels import paged_evict, paged_kv, paged_sparse
    return paged_kv, paged_evict, paged_sparse


def test_pages_past_2_31_elements(ops, cuda_lib):
    """Every operator on the last pages of a 9 GB pool and the same values in a small one: the same bits."""
    PK, PE, PS = ops
    g = torch.Generator(device="cuda").manual_seed(0)
    page, hkv, hd, n = 64, 4, 128, 4
    many = 2**31 // (page * hkv * hd) + 100
    near = torch.randn(1, 2, n, hkv, page, hd, device="cuda", generator=g).to(BF16)
    far = torch.empty(1, 2, many, hkv, page, hd, device="cuda", dtype=BF16)
    far[:, :, -n:] = near
    q = torch.randn(1, 16, hd, device="cuda", generator=g).to(BF16)
    qkv = torch.randn(1, 24 * hd, device="cuda", generator=g).to(BF16)
    mass = torch.rand(1, 1, hkv, n * page, device="cuda", generator=g)
    cos, sin = PK.rotary_table(300, hd)
    out = []
    for pool, first in ((near, 0), (far, many - n)):
        tab, lens, m = ints([range(first, first + n)]), ints([250]), mass.clone()
        k, v = pool[0, 0], pool[0, 1]
        r = [PK.rotary_paged_append(qkv, k, v, tab, lens, cos, sin, 16, positions=ints([299]))]
        r.append(PE.paged_decode_attention_mass(q, k, v, tab, lens, m[0]))
        b = PS.page_bounds(k)
        PS.update_page_bounds(k, b, tab, lens, cu_seqlens=ints([0, 250]))
        r.append(PS.select_blocks(q, b, tab, lens, page, 3))
        r.append(PS.paged_sparse_attention(q, k, v, tab, lens, r[-1]))
        r.append(PE.evict_positions(pool, tab, lens, m, 100, recent=10, sinks=2, return_source=True))
        out.append(r + [b[first:], pool[:, :, first:], m])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(*out, strict=True))
    assert cuda_lib.sn_device_status(1, None) == 0


def test_graphs_that_share_a_workspace(ops):
    """Two captured steps, of other sizes and of both forms of the attention, replayed in turn."""
    PK, PE, PS = ops
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    k, v = r(40, 2, 16, 128), r(40, 2, 16, 128)
    tab = torch.randperm(40, device="cuda", generator=g).to(torch.int32).view(2, 20)
    ws = PE.mass_workspace(2, 16, 2, 128, 320)
    q = [r(2, 16, 128), r(1, 4, 128)]
    lens = [ints([320, 33]), ints([100])]
    mass = [torch.zeros(2, 2, 320, device="cuda"), torch.zeros(1, 2, 320, device="cuda")]
    blocks = [ints([[[0, 3, 19, 7], [1, 2, 18, 19]], [[0, 1, 2, -1]] * 2]), ints([[[5, 6]] * 2])]

    def step(i):
        a = PE.paged_decode_attention_mass(q[i], k, v, tab[:2 - i], lens[i], mass[i], workspace=ws)
        return a, PS.paged_sparse_attention(q[i], k, v, tab[:2 - i], lens[i], blocks[i], workspace=ws)

    want = [[t.clone() for t in step(i)] for i in range(2)]
    once = [m.clone() for m in mass]
    graphs, out = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            out.append(step(i))
    for m in mass:
        m.zero_()
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out[i], want[i]))
    for m, o, times in zip(mass, once, (2, 3)):
        total = sum([o] * times)
        assert ((m - total).abs() <= 2.0 ** -22 * total).all()


def test_another_stream(ops):
    """stream= of every operator: it waits for what was enqueued there, and its results belong to it."""
    PK, PE, PS = ops
    g = torch.Generator(device="cuda").manual_seed(2)
    pool = torch.randn(2, 2, 12, 2, 16, 64, device="cuda", generator=g).to(BF16)
    tab, lens = torch.arange(12, device="cuda", dtype=torch.int32).view(2, 6), ints([90, 33])
    q = torch.randn(2, 8, 64, device="cuda", generator=g).to(BF16)

    def run(stream):
        p, m, b = pool.clone(), torch.zeros(2, 2, 2, 96, device="cuda"), PS.page_bounds(pool[0, 0])
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                torch.cuda._sleep(2_000_000)
        r = [PE.paged_decode_attention_mass(q, p[i, 0], p[i, 1], tab, lens, m[i], stream=stream) for i in range(2)]
        r.append(PE.evict_positions(p, tab, lens, m, 40, recent=4, return_source=True, stream=stream))
        PS.update_page_bounds(p[0, 0], b, tab, lens, cu_seqlens=ints([0, 90, 123]), stream=stream)
        r.append(PS.select_blocks(q, b, tab, lens, 16, 3, stream=stream))
        r.append(PS.paged_sparse_attention(q, p[0, 0], p[0, 1], tab, lens, r[-1], stream=stream))
        (stream or torch.cuda.current_stream()).synchronize()
        return r + [p, m, b]

    want = run(None)
    cu = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = run(cu)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_results_do_not_change_from_call_to_call(ops):
    """Many CTAs a row, cut streams, ties: the same bits every time."""
    PK, PE, PS = ops
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = torch.randn(1, 2, 1300, 2, 16, 128, device="cuda", generator=g).to(BF16)
    tab, lens = torch.randperm(1300, device="cuda", generator=g)[:1280].to(torch.int32).view(2, 640), ints([10237, 9001])
    q = torch.randn(2, 16, 128, device="cuda", generator=g).to(BF16)
    weights = torch.rand(1, 2, 2, 10240, device="cuda", generator=g).mul(8).round()  # eight values
    b = PS.page_bounds(pool[0, 0])
    PS.update_page_bounds(pool[0, 0], b, tab, lens, cu_seqlens=ints([0, 10237, 19238]))
    b = (b * 2).round().clamp(-1, 1)  # few values, many equal sums
    ws = PE.mass_workspace(2, 16, 2, 128, 10240)
    first = None
    for _ in range(5):
        p, m, z = pool.clone(), weights.clone(), torch.zeros(2, 2, 10240, device="cuda")
        r = [PE.paged_decode_attention_mass(q, p[0, 0], p[0, 1], tab, lens, z, workspace=ws), z]
        r += [PS.select_blocks(q, b, tab, lens, 16, 100, first=1, last=1)]
        r += [PS.paged_sparse_attention(q, p[0, 0], p[0, 1], tab, lens, r[-1], workspace=ws)]
        r += [PE.evict_positions(p, tab, lens, m, 5000, recent=77, sinks=3, return_source=True), p, m]
        torch.cuda.synchronize()
        first = first or r
        assert all(torch.equal(x, y) for x, y in zip(r, first, strict=True))
