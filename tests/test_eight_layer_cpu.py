"""What a layer in 8 bits refuses before any launch: vectors that its kernels would read by address."""

import pytest
import torch


def packed(m3, k, n):
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    tiles, steps = -(-n // 64) * 4, -(-k // 128)
    return m3.Weight8(torch.zeros(tiles, steps, 2, 64, 16, dtype=f8),
                      torch.zeros(steps, tiles // 4, 64, 4, dtype=torch.uint8).view(e8), k, n, False)


@pytest.fixture(scope="module")
def layer(m3):
    cfg = m3.SISOConfig(d_model=128, d_state=64, headdim=64, expand=2, chunk=64)
    p = m3.init_params(cfg, 0)
    return cfg, p._replace(in_proj=packed(m3, cfg.d_model, cfg.d_in_proj), out_proj=packed(m3, cfg.d_inner, cfg.d_model))


def calls(m3, cfg, p):
    st = m3.model.zero_states(m3.model.LMConfig(vocab_size=7, n_layers=1, siso=cfg), 2, device="cpu")[0]
    u = torch.zeros(2, 64, cfg.d_model, dtype=torch.bfloat16)
    return (lambda: m3.mamba3_siso_layer(p, u, cfg), lambda: m3.mamba3_siso_layer(p, u, cfg, state=st),
            lambda: m3.mamba3_siso_decode_step(p, u[:, 0], cfg, st))


@pytest.mark.parametrize("field", ["dt_bias", "b_norm_weight", "c_norm_weight", "b_bias", "c_bias", "d_skip"])
@pytest.mark.parametrize("change", [
    lambda t: t[:-1], lambda t: t[:1], lambda t: torch.cat([t, t]), lambda t: t[None], lambda t: t.to("meta")],
    ids=["short", "one", "long", "axis", "device"])
def test_vectors_of_another_shape_or_device(m3, layer, field, change):
    """A short vector would be read past its end, and one elsewhere through an address of another device."""
    cfg, p = layer
    for call in calls(m3, cfg, p._replace(**{field: change(getattr(p, field))})):
        with pytest.raises(ValueError, match=f"{field} must be"):
            call()


def test_vectors_that_are_missing(m3, layer):
    cfg, p = layer
    for call in calls(m3, cfg, p._replace(b_bias=None)):
        with pytest.raises(ValueError, match="b_bias must be"):
            call()
    # no skip is a layer's right: the call goes on, to the products, which the CPU does not do
    for call in calls(m3, cfg, p._replace(d_skip=None)):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


@pytest.mark.parametrize("shape", [(0, 64), (2, 0)])
def test_no_tokens(m3, layer, shape):
    """As the layer in bf16, a ValueError of its own."""
    cfg, p = layer
    with pytest.raises(ValueError, match="a token at least"):
        m3.mamba3_siso_layer(p, torch.zeros(*shape, cfg.d_model, dtype=torch.bfloat16), cfg)


def test_packed_weights_are_not_packed_again(m3, layer):
    cfg, p = layer
    M = m3.model
    lm = M.LMConfig(vocab_size=7, n_layers=1, siso=cfg)
    params = M.init_lm(lm, 0)
    params = params._replace(blocks=[b._replace(siso=p) for b in params.blocks])
    for short in (False, True):
        with pytest.raises(ValueError, match="for serving"):
            M.eight_bit_params(params, lm, short_sums=short)
