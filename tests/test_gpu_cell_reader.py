"""The operators together: CellReader and the encoder's channels-last and reading options against plain float64 modules,
forward and backward."""

import pytest
import torch
import torch.nn.functional as TF

import _feature_ref as R
from gaussian_splat_encoder import efficient_encoder as EE
from gaussian_splat_encoder.cell_reader import CellReader

pytestmark = pytest.mark.gpu


def plain_reader(m, x, states, lengths=None, mask=None):
    """CellReader in float64: P holds its parameters."""
    P = {k: v.detach().double().requires_grad_(True) for k, v in m.named_parameters()}
    lin = lambda t, n: t @ P[n + ".weight"].t() + P[n + ".bias"]   # noqa: E731
    norm = lambda t, n: R.group_norm_act(t, m.norm1.num_groups, P[n + ".weight"], P[n + ".bias"], 1e-5, "none",  # noqa: E731
                                         False)
    B, h, d = x.shape[0], m.heads, m.head_dim
    kv = lin(states, "to_kv").reshape(B, -1, 2, m.kv_heads, d)
    q = lin(norm(x, "norm1"), "to_q").reshape(B, -1, h, d)
    a = R.cross_attention(q, kv[:, :, 0], kv[:, :, 1], lengths, mask, d ** -0.5)
    x = x + lin(a.reshape(x.shape[:-1] + (h * d,)), "to_out")
    return x + lin(R.act(lin(norm(x, "norm2"), "fc1"), "gelu"), "fc2"), P


def reader(*a, **kw):
    torch.manual_seed(0)
    m = CellReader(*a, **kw).cuda()
    for layer in (m.to_out, m.fc2):
        torch.nn.init.normal_(layer.weight, std=layer.in_features ** -0.5)
        torch.nn.init.normal_(layer.bias, std=0.1)
    return m


@pytest.mark.parametrize("masked", [False, True])
def test_reader_forward_backward(masked):
    """float32 through ten operators in a row: their bounds (64 * 2^-24 each) add up."""
    m = reader(48, 40, heads=6, kv_heads=2)
    x = torch.randn(3, 9, 7, 48, device="cuda", requires_grad=True)
    st = torch.randn(3, 5, 6, 40, device="cuda", requires_grad=True)
    lengths = torch.tensor([30, 0, 11], device="cuda") if masked else None
    y = m(x, st, kv_lengths=lengths)
    xd, sd = x.detach().double().requires_grad_(True), st.detach().double().requires_grad_(True)
    z, P = plain_reader(m, xd, sd, lengths)
    g = torch.randn_like(y)
    names = [k for k, _ in m.named_parameters()]
    got = torch.autograd.grad(y, [x, st, *m.parameters()], g)
    want = torch.autograd.grad(z, [xd, sd, *[P[k] for k in names]], g.double())
    bound = 10 * R.BOUND[torch.float32]
    errs = {n: R.rel(a, b) for n, a, b in zip(["y", "x", "states", *names], [y, *got], [z, *want])}
    assert all(e <= bound for e in errs.values()), errs


def test_new_reader_is_the_identity():
    m = CellReader(32, 16).cuda()
    x, st = torch.randn(2, 4, 5, 32, device="cuda"), torch.randn(2, 3, 16, device="cuda")
    with torch.no_grad():
        assert torch.equal(m(x, st), x)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_tokens_read_splat_latents(dt):
    """A few query tokens read the latents of all splats of an image, dead ones masked, from keys and values that are kept:
    the same bits as from the states, and one step of a training program."""
    enc = EE.EfficientGaussianEncoder(d_feature=32, variant="free", gaussians_per_cell=2, channels_last=True).cuda()
    out = enc(torch.rand(2, 3, 64, 48, device="cuda"), return_latents=True)
    lat = enc.gather_splat_latents(out)
    m = reader(64, lat.shape[-1], heads=4)
    tokens = torch.randn(2, 5, 64, device="cuda").to(dt)
    live = out["opacity"] > 0.5
    with torch.no_grad():
        kv = m.keys_values(lat.to(dt))
        y = m(tokens, lat.to(dt), key_mask=live)
        assert torch.equal(m(tokens, kv=kv, key_mask=live), y)
    ref, _ = plain_reader(m, tokens.double(), lat.double(), mask=live)
    assert R.rel(y, ref) <= 10 * R.BOUND[dt]
    m(tokens, lat.to(dt), key_mask=live).float().square().mean().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in [*m.parameters(), *enc.backbone.parameters()])


@pytest.mark.parametrize("variant,kw", [("free", {}), ("adaptive", dict(fine_stride=4, residual_grid=32)),
                                        ("adaptive", dict(fine_stride=4, residual_grid=32, fine_reader_heads=4))])
def test_channels_last_encoder_is_the_same_encoder(variant, kw):
    """The same weights with and without channels_last: the same splats and gradients up to rounding. The convolutions of
    the two layouts may sum in other orders, and stages multiply such differences: 1e-4 of an output's norm."""
    torch.manual_seed(1)
    a = EE.EfficientGaussianEncoder(d_feature=64, variant=variant, **kw).cuda()
    b = EE.EfficientGaussianEncoder(d_feature=64, variant=variant, channels_last=True, **kw).cuda()
    b.load_state_dict(a.state_dict(), strict=True)
    img = torch.rand(2, 3, 72, 56, device="cuda")
    oa, ob = a(img), b(img)
    for k in ("mu", "log_scale", "color", "opacity", "theta", "bg"):
        assert oa[k].shape == ob[k].shape and R.rel(ob[k], oa[k]) <= 1e-4, k
    keys = ("log_scale", "color", "opacity", "theta", "bg")
    g = [torch.randn_like(oa[k]) for k in keys]
    ga = torch.autograd.grad([oa[k] for k in keys], list(a.parameters()), g, allow_unused=True)
    gb = torch.autograd.grad([ob[k] for k in keys], list(b.parameters()), g, allow_unused=True)
    for (n, _), x, y in zip(a.named_parameters(), ga, gb):
        assert (x is None) == (y is None), n
        if x is not None and x.any():
            assert R.rel(y, x) <= 1e-3, n
    if variant == "adaptive":   # a training step: render, loss, backward
        from gaussian_splat_encoder.render_hip import render_alpha_octave
        ob = b(img)
        r = render_alpha_octave(ob["mu"], ob["log_scale"], ob["color"], ob["opacity"], ob["bg"], 72, 56, theta=ob["theta"])
        b.zero_grad()
        TF.mse_loss(r, img).backward()
        assert all(torch.isfinite(p.grad).all() for p in b.parameters() if p.grad is not None)


def test_channels_last_encoder_under_autocast():
    """bfloat16 convolutions feed bfloat16 operators; parameters stay float32 and get finite gradients."""
    torch.manual_seed(2)
    enc = EE.EfficientGaussianEncoder(d_feature=32, variant="free", channels_last=True).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = enc(torch.rand(1, 3, 64, 64, device="cuda"))
    ref = enc(torch.rand(1, 3, 64, 64, device="cuda"))
    assert out["log_scale"].dtype is torch.bfloat16 and out["mu"].shape == ref["mu"].shape
    sum(out[k].float().sum() for k in ("mu", "log_scale", "color", "opacity", "bg")).backward()
    assert all(p.grad is None or (p.grad.dtype is torch.float32 and torch.isfinite(p.grad).all()) for p in enc.parameters())
