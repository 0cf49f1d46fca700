"""Ragged serving end to end: prompts, steps, forks and frees of several streams against the dense decode step taken
token by token, one stream at a time (the same weights; its cache holds one common position).

Both sides round to bf16 after every op of every layer, in other orders inside the ops, so logits (rms about 1) agree
to some bf16 rounding steps of the hidden state: relative norm 3e-2 over 4 layers, and the same top choice wherever the
dense path's two best logits are further apart than twice the largest difference."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _dense_logits(seed, cfg, tokens):
    """Logits after each token of one stream, by the dense decode step."""
    from sonata_b200.kernels import decode_step as DS
    m = DS.SyntheticZonos(cfg, batch=1, context=0, max_seqlen=256, seed=seed)
    out = []
    with torch.no_grad():
        for t in range(tokens.shape[0]):
            m.pos = t
            m.cos, m.sin = DS.rotary_cos_sin(t, cfg.head_dim, "cuda")
            out.append(m.step(tokens[t:t + 1]).clone())
    torch.cuda.synchronize()
    return out


def _close(got, want):
    d = (got - want).double()
    assert (d.norm() / want.double().norm()).item() <= 3e-2, (d.norm() / want.double().norm()).item()
    two = want.topk(2, dim=-1).values
    sure = (two[..., 0] - two[..., 1]) > 2 * d.abs().max()
    assert torch.equal(got.argmax(-1)[sure], want.argmax(-1)[sure])


def test_prompts_steps_and_forks(cuda_lib):
    from sonata_b200.kernels import decode_step as DS, serve
    cfg = DS.ZonosBackboneConfig(n_layer=4, attn_layer_idx=[1, 3])
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 180, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    want = [_dense_logits(7, cfg, x[i, :n]) for i, n in enumerate((42, 140, 20))]
    m = DS.SyntheticZonos(cfg, batch=3, context=0, max_seqlen=8, seed=7)
    r = serve.RaggedZonos(m, num_pages=60, max_len=256)
    # stream 0: 37 tokens; 1: 130; 2: nothing yet
    lg = r.prompt(torch.cat([x[0, :37], x[1, :130]]), [37, 130, 0])
    _close(lg[:, 0:1], want[0][36])
    _close(lg[:, 1:2], want[1][129])
    assert not lg[:, 2].any()
    # stream 0 goes on by a second piece while stream 2 starts
    lg = r.prompt(torch.cat([x[0, 37:40], x[2, :17]]), [3, 0, 17])
    _close(lg[:, 0:1], want[0][39])
    _close(lg[:, 2:3], want[2][16])
    for i in range(2):  # one token of every stream at its own position
        lg = r.step(torch.stack([x[0, 40 + i], x[1, 130 + i], x[2, 17 + i]]))
        for s, t in ((0, 40 + i), (1, 130 + i), (2, 17 + i)):
            _close(lg[:, s:s + 1], want[s][t])
    # stream 2 ends, stream 1 is continued twice: both give what one gives; then the pages are compacted
    r.free(2)
    r.fork(1, 2)
    assert r.cache.pages[2][:8] == r.cache.pages[1][:8] and r.cache.pages[2][8] != r.cache.pages[1][8]
    for i in range(2, 5):
        lg = r.step(torch.stack([x[0, 41], x[1, 130 + i], x[1, 130 + i]]))
        assert torch.equal(lg[:, 1], lg[:, 2])
        _close(lg[:, 1:2], want[1][130 + i])
        if i == 3:
            r.free(0)
            assert r.cache.compact() > 0
    assert cuda_lib.sn_device_status(1, None) == 0


def test_refusals(cuda_lib):
    from sonata_b200.kernels import decode_step as DS, serve
    cfg = DS.ZonosBackboneConfig(n_layer=2, attn_layer_idx=[0])
    m = DS.SyntheticZonos(cfg, batch=2, context=0, max_seqlen=8, seed=0)
    r = serve.RaggedZonos(m, num_pages=3, max_len=64)
    x = torch.zeros(60, cfg.d_model, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        r.prompt(x[:5], [5])
    with pytest.raises(ValueError):
        r.prompt(x[:5], [2, 2])
    with pytest.raises(ValueError):
        r.step(x[:1])
    with pytest.raises(RuntimeError):
        r.prompt(x, [30, 30])  # 4 pages of 3
    assert r.cache.lens == [0, 0]


def test_max_len_inside_a_page(cuda_lib):
    """max_len positions and no more, whether or not it ends a page: the last one is right, the next one is refused and
    changes nothing."""
    from sonata_b200.kernels import decode_step as DS, serve
    cfg = DS.ZonosBackboneConfig(n_layer=2, attn_layer_idx=[1])
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(22, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    want = _dense_logits(9, cfg, x[:20])
    m = DS.SyntheticZonos(cfg, batch=1, context=0, max_seqlen=8, seed=9)
    r = serve.RaggedZonos(m, num_pages=10, max_len=20)  # pages of 16: two of them would hold 32
    with pytest.raises(ValueError):
        r.prompt(x[:21], [21])
    assert r.cache.lens == [0] and r.cache.free_pages == 10
    r.prompt(x[:18], [18])
    with pytest.raises(ValueError):
        r.prompt(x[18:21], [3])
    for t in (18, 19):
        _close(r.step(x[t:t + 1])[:, 0:1], want[t])
    with pytest.raises(ValueError):
        r.step(x[20:21])
    assert r.cache.lens == [20]
    assert cuda_lib.sn_device_status(1, None) == 0


def test_states_are_its_own(cuda_lib):
    """Two of them on one model, and the model's own decode step between: none sees another's states."""
    from sonata_b200.kernels import decode_step as DS, serve
    cfg = DS.ZonosBackboneConfig(n_layer=2, attn_layer_idx=[1])
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(2, 12, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    want = [_dense_logits(4, cfg, x[i]) for i in range(2)]
    m = DS.SyntheticZonos(cfg, batch=1, context=0, max_seqlen=64, seed=4)
    mixer = m.backbone.layers[0].mixer
    own = mixer.conv_state, mixer.ssm_state
    with torch.no_grad():
        first = m.step(x[0, :1]).clone()
    held = [t.clone() for t in own]
    a = serve.RaggedZonos(m, num_pages=8, max_len=64)
    a.prompt(x[0, :9], [9])
    b = serve.RaggedZonos(m, num_pages=8, max_len=64)
    b.prompt(x[1, :5], [5])
    for t in range(9, 12):
        _close(a.step(x[0, t:t + 1])[:, 0:1], want[0][t])
        _close(b.step(x[1, t - 4:t - 3])[:, 0:1], want[1][t - 4])
    # the model's states are the tensors they were, as they were
    assert mixer.conv_state is own[0] and mixer.ssm_state is own[1]
    assert torch.equal(own[0], held[0]) and torch.equal(own[1], held[1])
    for t in own:
        t.zero_()
    with torch.no_grad():
        assert torch.equal(m.step(x[0, :1]), first)


def test_idle_streams(cuda_lib):
    """A freed slot and one that never started stay empty through the others' steps, and a prompt or a fork into them is as
    good as in a new one; steps of some of the streams leave the others where they are."""
    from sonata_b200.kernels import decode_step as DS, serve
    cfg = DS.ZonosBackboneConfig(n_layer=4, attn_layer_idx=[1, 3])
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(3, 40, cfg.d_model, device="cuda", generator=g).to(torch.bfloat16)
    want = [_dense_logits(11, cfg, x[i]) for i in range(3)]
    m = DS.SyntheticZonos(cfg, batch=4, context=0, max_seqlen=8, seed=11)
    r = serve.RaggedZonos(m, num_pages=12, max_len=64)
    junk = torch.full((cfg.d_model,), float("nan"), device="cuda", dtype=torch.bfloat16)
    rows = lambda **k: torch.stack([k.get(f"s{s}", junk) for s in range(4)])
    with pytest.raises(ValueError):  # no stream holds anything
        r.step(rows())
    r.prompt(torch.cat([x[0, :20], x[1, :9]]), [20, 9, 0, 0])
    r.free(0)
    for t in range(9, 12):
        lg = r.step(rows(s1=x[1, t]))
        _close(lg[:, 1:2], want[1][t])
        assert not lg[:, [0, 2, 3]].any()
    assert r.cache.lens == [0, 12, 0, 0] and r.cache.pages[0] == r.cache.pages[2] == []
    r.prompt(x[2, :17], [17, 0, 0, 0])  # another stream in the freed slot
    r.fork(1, 3)
    for t in range(3):
        lg = r.step(rows(s0=x[2, 17 + t], s1=x[1, 12 + t], s3=x[1, 12 + t]))
        _close(lg[:, 0:1], want[2][17 + t])
        _close(lg[:, 1:2], want[1][12 + t])
        _close(lg[:, 3:4], want[1][12 + t])
    # stream 0 alone, then a first token by name in the slot that never started, then all of them
    lg = r.step(rows(s0=x[2, 20]), active=[True, False, False, False])
    _close(lg[:, 0:1], want[2][20])
    lg = r.step(rows(s2=x[0, 0]), active=[0, 0, 1, 0])
    _close(lg[:, 2:3], want[0][0])
    lg = r.step(rows(s0=x[2, 21], s1=x[1, 15], s2=x[0, 1], s3=x[1, 15]))
    for s, i, t in ((0, 2, 21), (1, 1, 15), (2, 0, 1), (3, 1, 15)):
        _close(lg[:, s:s + 1], want[i][t])
    assert r.cache.lens == [22, 16, 2, 16]
    for bad in ([True], [False] * 4):
        with pytest.raises(ValueError):
            r.step(rows(), active=bad)
    assert r.cache.lens == [22, 16, 2, 16]
    assert cuda_lib.sn_device_status(1, None) == 0
