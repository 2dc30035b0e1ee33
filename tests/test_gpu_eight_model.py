"""A model served in 8 bits (`model.eight_bit_params`): layer, forward, decode, generation.

The bf16 layer on weights rounded to 8 bits and on rows rounded to 8 bits (bf16 holds both exactly)
makes the same products but for the order and cuts of their sums, so what the scan leaves is held to
the bf16 noise of that: 1e-2 of the states' norm. Behind the scan rows are rounded again, half a step
of e4m3 (2^-4) at most, 2^-4 / sqrt(3) = 0.036 of the norm where every value takes the largest step and
errors are even, and a product passes that ratio on. A block's output so differs by a few of these; a
model's logits, whose stream is the embedding plus such outputs, are held to 0.15 of their norm.
"""

import pytest
import torch

from test_gpu_eight import round8, rounded_weight

BF16, F32 = torch.bfloat16, torch.float32
STATE_REL, ROWS_REL, LOGITS_REL = 1e-2, 0.036, 0.15

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert bool(torch.isfinite(a).all())
    return float((a - b).norm() / b.norm())


def siso(m3, d_model=128, expand=2, chunk=64, d_state=64, headdim=64):
    return m3.SISOConfig(d_model=d_model, d_state=d_state, headdim=headdim, expand=expand, chunk=chunk)


def lm(m3, dtype, vocab=61, n_layers=2, d_intermediate=200, seed=0, **kw):
    cfg = m3.model.LMConfig(vocab_size=vocab, n_layers=n_layers, siso=siso(m3, **kw), d_intermediate=d_intermediate)
    params = m3.model.init_lm(cfg, seed)
    # ids that mean something: a stream of the blocks' own size
    params = params._replace(embed=params.embed * 25)
    return cfg, m3.model.lm_map(lambda t: t.to(dtype).cuda(), params)


def rounded_params(m3, params):
    """The bf16 model whose projections hold the values of the packed ones."""
    w = lambda t: rounded_weight(t.cpu()).to(BF16).cuda()  # noqa: E731
    blocks = [b._replace(siso=b.siso._replace(in_proj=w(b.siso.in_proj), out_proj=w(b.siso.out_proj)),
                         mlp=None if b.mlp is None else m3.model.MLPParams(w(b.mlp.fc1), w(b.mlp.fc2)))
              for b in params.blocks]
    return params._replace(blocks=blocks)


@pytest.mark.parametrize("seqlen", [64, 192])
@pytest.mark.parametrize("carried", [False, True])
def test_layer(m3, dev, seqlen, carried):
    """With an identity as out_proj (expand 1) the layer's output is the scan's rows in 8 bits."""
    cfg = siso(m3, expand=1)
    gen = torch.Generator().manual_seed(seqlen + carried)
    p = m3.init_params(cfg, gen, device=dev)
    eye = torch.eye(cfg.d_inner, device=dev)
    p8 = p._replace(in_proj=m3.pack8(p.in_proj), out_proj=m3.pack8(eye))
    ref = p._replace(in_proj=rounded_weight(p.in_proj.cpu()).to(BF16).cuda(), out_proj=eye.to(BF16))
    u = torch.randn(3, seqlen, cfg.d_model, generator=gen).to(BF16)
    ur = round8(u.double()).to(BF16).cuda()
    st = None
    with torch.no_grad():
        if carried:
            _, st = m3.mamba3_siso_layer(ref, ur, cfg)
        got, s8 = m3.mamba3_siso_layer(p8, u.cuda(), cfg, state=st)
        again, _ = m3.mamba3_siso_layer(p8, m3.quantize8(u.cuda()), cfg, state=st)
        want, s16 = m3.mamba3_siso_layer(ref, ur, cfg, state=st)
    assert got.shape == want.shape and got.dtype == BF16 and torch.equal(got, again)
    for a, b in zip(s8, s16):
        if a is s8.phi:   # angles: apart by whole turns at most
            a, b = torch.sin(a.double()), torch.sin(b.double())
        assert rel(a, b) < STATE_REL
    assert rel(got, round8(want.double().cpu())) < ROWS_REL
    assert rel(got, want) < ROWS_REL


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d_intermediate", [0, 200])
def test_forward(m3, dev, dtype, d_intermediate):
    cfg, params = lm(m3, dtype, d_intermediate=d_intermediate)
    p8, ref = m3.model.eight_bit_params(params, cfg), rounded_params(m3, params)
    xs = torch.randint(0, 61, (2, 192), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        got, want = m3.model.lm_forward(p8, xs, cfg), m3.model.lm_forward(ref, xs, cfg)
        assert got.dtype == F32 and got.shape == want.shape
        assert rel(got, want) < LOGITS_REL
        # in two segments with a carried state
        a, st = m3.model.lm_forward(p8, xs[:, :64], cfg, states=m3.model.zero_states(cfg, 2, device=dev))
        b, st = m3.model.lm_forward(p8, xs[:, 64:], cfg, states=st)
        assert rel(torch.cat([a, b], 1), got) < LOGITS_REL


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch", [1, 3, 40])
def test_decode(m3, dev, dtype, batch):
    """Tokens one by one against the prompt at once, and a recorded step against eager ones."""
    cfg, params = lm(m3, dtype)
    p8 = m3.model.eight_bit_params(params, cfg)
    xs = torch.randint(0, 61, (batch, 64), generator=torch.Generator().manual_seed(batch)).cuda()
    with torch.no_grad():
        want = m3.model.lm_forward(p8, xs, cfg)
        st, graph = m3.model.zero_states(cfg, batch, device=dev), m3.train.DecodeGraph(p8, cfg, batch)
        for i in range(64):
            got, st = m3.model.lm_decode_step(p8, xs[:, i], st, cfg)
            assert torch.equal(graph.step(xs[:, i]), got)
            assert rel(got, want[:, i]) < LOGITS_REL, i


def test_generate(m3, dev):
    cfg, params = lm(m3, F32)
    p8 = m3.model.eight_bit_params(params, cfg)
    prompt = list(range(61)) + list(range(30))
    a = m3.train.generate(p8, cfg, 3, prompt, n_tokens=20, graph=True)
    b = m3.train.generate(p8, cfg, 3, prompt, n_tokens=20, graph=False)
    assert a == b and len(a) == len(prompt) + 20


def test_sub_heads(m3, dev):
    """A head width that decodes as sub-heads, through the composed step."""
    cfg, params = lm(m3, BF16, headdim=128)
    p8 = m3.model.eight_bit_params(params, cfg)
    xs = torch.randint(0, 61, (2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        want = m3.model.lm_forward(p8, xs, cfg)
        st = m3.model.zero_states(cfg, 2, device=dev)
        for i in range(64):
            got, st = m3.model.lm_decode_step(p8, xs[:, i], st, cfg)
        assert rel(got, want[:, -1]) < LOGITS_REL


def test_refusals(m3, dev, tmp_path):
    M = m3.model
    cfg, params = lm(m3, F32)
    p8 = M.eight_bit_params(M.lm_map(lambda t: t.requires_grad_(), params), cfg)
    xs = torch.zeros(1, 64, dtype=torch.int64, device=dev)
    M.lm_forward(p8, xs, cfg)                          # packed weights and detached vectors: no gradient to take
    assert M.decode_params(p8, cfg) is p8
    train = p8._replace(embed=p8.embed.clone().requires_grad_())
    bad_gain = p8._replace(blocks=[b._replace(norm_gain=b.norm_gain.clone().requires_grad_()) for b in p8.blocks])
    scfg = m3.SISOConfig(d_model=64, d_state=16, headdim=16, expand=2, chunk=64, policy_name="f32")
    f32_cfg = M.LMConfig(vocab_size=61, n_layers=2, siso=scfg)
    b0 = p8.blocks[0]
    half = b0.siso._replace(out_proj=params.blocks[0].siso.out_proj)
    u = torch.zeros(1, 64, 128, device=dev, dtype=BF16)
    for call, what in (
            (lambda: M.lm_forward(train, xs, cfg), "gradient"),
            (lambda: M.lm_loss(bad_gain, xs, xs, cfg), "gradient"),
            (lambda: M.lm_leaves(p8), "for serving"),
            (lambda: M.lm_to(p8, dtype=BF16), "for serving"),
            (lambda: m3.train.make_optimizer(p8), "for serving"),
            (lambda: m3.checkpoint.save(str(tmp_path / "a"), p8, cfg), "for serving"),
            (lambda: m3.convert.lm_state_dict(p8, cfg), "for serving"),
            (lambda: M.eight_bit_params(params, f32_cfg), "bf16 policy"),
            (lambda: m3.mamba3_siso_layer(half, u, cfg.siso), "both be packed"),
            (lambda: m3.mamba3_siso_layer(b0.siso, u[0], cfg.siso), r"\(B, L, d_model\)"),
            (lambda: m3.mamba3_siso_layer(b0.siso, u[:, :, :64], cfg.siso), "rows of 64"),
            (lambda: m3.mamba3_siso_layer(b0.siso, u, cfg.siso, state=M.zero_states(cfg, 2, device=dev)[0]), "state must"),
            (lambda: m3.mamba3_siso_decode_step(params.blocks[0].siso, u[:, 0], cfg.siso, None, residual=u[:, 0]),
             "in 8 bits")):
        with pytest.raises(ValueError, match=what):
            call()


def test_wide_heads_without_a_gradient(m3, dev):
    """The bf16 layer of head width 128 under no_grad, against the same call with a gradient."""
    cfg = siso(m3, headdim=128)
    p = m3.init_params(cfg, 0, device=dev)
    p = p._replace(in_proj=p.in_proj.to(BF16), out_proj=p.out_proj.to(BF16))
    u = torch.randn(2, 128, cfg.d_model, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    with torch.no_grad():
        got, _ = m3.mamba3_siso_layer(p, u, cfg)
    want, _ = m3.mamba3_siso_layer(p, u.clone().requires_grad_(), cfg)
    assert rel(got, want.detach()) < STATE_REL
