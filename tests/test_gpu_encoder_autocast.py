"""The encoder's channels-last option under autocast: positions and background keep float32, whatever the features' type."""

import pytest
import torch

from gaussian_splat_encoder import efficient_encoder as EE

pytestmark = pytest.mark.gpu

VARIANTS = [("free", {}), ("adaptive", dict(fine_stride=4, residual_grid=32)),
            ("adaptive", dict(fine_stride=4, residual_grid=32, fine_reader_heads=4))]


def encoder(variant, kw, offsets):
    torch.manual_seed(3)
    enc = EE.EfficientGaussianEncoder(d_feature=32, variant=variant, channels_last=True, **kw).cuda()
    if offsets:   # the heads that move splats start at zero
        for m in enc.modules():
            if isinstance(m, EE._SplatHead):
                torch.nn.init.normal_(m.mu_head.weight, std=0.02)
    return enc


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant,kw", VARIANTS)
def test_centres_under_autocast(variant, kw, dt):
    """Without offsets the splats sit on the cells' centres: the float32 encoder's, to the bit."""
    enc, img = encoder(variant, kw, False), torch.rand(1, 3, 512, 384, device="cuda")
    with torch.no_grad():
        ref = enc(img)
        with torch.autocast("cuda", dtype=dt):
            out = enc(img)
    assert out["mu"].dtype is torch.float32 and torch.equal(out["mu"], ref["mu"])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant,kw", VARIANTS)
def test_positions_under_autocast(variant, kw, dt):
    """Offsets of a few pixels from bfloat16 features: 2^-8 of a feature after three stages of bfloat16 products, heads of
    about 0.02 * sqrt(33) per unit of it and offsets of up to 32 pixels make 0.02 pixels of standard deviation, five of
    which and the offset's own rounding (2^-9 of 32 pixels at most) stay below a quarter of a pixel."""
    enc, img = encoder(variant, kw, True), torch.rand(1, 3, 512, 384, device="cuda")
    with torch.no_grad():
        ref = enc(img)
        with torch.autocast("cuda", dtype=dt):
            out = enc(img)
    moved = (ref["mu"] - encoder(variant, kw, False)(img)["mu"]).abs().max().item() * 512
    err = (out["mu"] - ref["mu"]).abs().max().item() * 512
    print(f"offsets up to {moved:.1f} px, error {err:.3f} px", flush=True)
    assert out["mu"].dtype is torch.float32 and moved > 1 and err < 0.25
    # the mean over all cells is taken in float32, and so is the product behind it: what is left are the features' own
    # roundings, 2^-8 of values of order one through a sigmoid's slope of a quarter
    assert out["bg"].dtype is torch.float32 and (out["bg"] - ref["bg"]).abs().max().item() < 2.0 ** -8


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("variant,kw", VARIANTS)
def test_training_under_autocast(variant, kw, dt):
    """A step's gradients are float32 and finite, and the renderer takes the splats as they are."""
    from gaussian_splat_encoder.render_hip import render_alpha_octave
    enc, img = encoder(variant, kw, True), torch.rand(2, 3, 64, 48, device="cuda")
    with torch.autocast("cuda", dtype=dt):
        o = enc(img)
    r = render_alpha_octave(o["mu"], o["log_scale"], o["color"], o["opacity"], o["bg"], 64, 48, theta=o["theta"])
    (r.float() - img).square().mean().backward()
    grads = [p.grad for p in enc.parameters() if p.grad is not None]
    assert grads and all(g.dtype is torch.float32 and torch.isfinite(g).all() for g in grads)
