"""TokenReader on the GPU: against a plain float64 layer with its gradients, dense and cached, frame by frame, captured, and on
the encoder's splats."""

import math

import pytest
import torch

import _feature_ref as FR
import _token_ref as R
from gaussian_splat_encoder.token_ops import RotaryAxes
from gaussian_splat_encoder.token_reader import TokenReader

pytestmark = pytest.mark.gpu


def rand(*shape, dt=torch.float32, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)


def make(channels=96, state=56, heads=6, kv_heads=2, kind="rms"):
    torch.manual_seed(3)
    r = TokenReader(channels, state, RotaryAxes((4, 6, 6), base=100.0, scale=(1.0, 20.0, 20.0)), heads=heads, kv_heads=kv_heads,
                    kind=kind).cuda()
    with torch.no_grad():       # a trained one's: gates open, norms not all ones
        for i, n in enumerate(("gate1", "gate2", "norm1", "post1", "norm2", "post2")):
            getattr(r, n).copy_(1 + 0.3 * torch.randn(channels, generator=torch.Generator().manual_seed(i)))
    return r


def where(B, L, t, seed):
    """Positions (time, y, x) of a frame's splats."""
    p = torch.rand(B, L, 2, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
    return torch.cat([torch.full((B, L, 1), float(t), device="cuda"), p], -1)


def plain(r, p, x, pos, s, spos, mask):
    """The layer r in float64 with the parameters p."""
    lin = lambda v, n: v @ p[n + ".weight"].t() + p[n + ".bias"]   # noqa: E731
    B, L, C = x.shape
    heads, kv, D, ax, kind = r.heads, r.kv_heads, r.head_dim, r.axes, r.kind
    q = lin(R.norm(x, p["norm1"], None, kind, 1e-6), "to_q").reshape(B, L, heads, D)
    k, v = lin(s, "to_kv").reshape(B, s.shape[1], 2, kv, D).unbind(2)
    a = FR.cross_attention(R.rotary(q, pos, ax), R.rotary(k, spos, ax), v, None, mask, D ** -0.5)
    y = x + p["gate1"] * R.norm(lin(a.reshape(B, L, heads * D), "to_out"), p["post1"], None, kind, 1e-6)
    h = lin(FR.act(lin(R.norm(y, p["norm2"], None, kind, 1e-6), "fc1"), "gelu"), "fc2")
    return y + p["gate2"] * R.norm(h, p["post2"], None, kind, 1e-6)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_reader_and_its_gradients(kind):
    """Float32: each of the layer's nine steps has the operators' bound, the gradients pass them twice."""
    r = make(kind=kind)
    B, L, N = 2, 9, 150
    x, s = rand(B, L, 96, seed=1).requires_grad_(True), rand(B, N, 56, seed=2).requires_grad_(True)
    pos, spos = where(B, L, 4, 5).requires_grad_(True), where(B, N, 2, 6).requires_grad_(True)
    mask = rand(B, N, seed=7) < 0.8
    names = [n for n, _ in r.named_parameters()]
    y = r(x, pos, s, spos, key_mask=mask)
    g = rand(*y.shape, seed=8)
    ga = torch.autograd.grad(y, [x, s, pos, spos] + list(r.parameters()), g)
    d = [t.detach().double().requires_grad_(True) for t in (x, s, pos, spos)]
    p = {n: t.detach().double().requires_grad_(True) for n, t in r.named_parameters()}
    z = plain(r, p, d[0], d[2], d[1], d[3], mask)
    gd = torch.autograd.grad(z, d + [p[n] for n in names], g.double())
    assert FR.rel(y, z) <= 9 * R.bound_of(torch.float32)
    for n, a, b in zip(["x", "states", "positions", "state positions"] + names, ga, gd):
        if n == "to_kv.bias":   # keys' biases move all scores alike where nothing turns: their part is a difference of sums
            continue
        assert FR.rel(a, b) <= 18 * R.bound_of(torch.float32), n


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_frames_one_by_one_are_frames_together(dt):
    """Three frames appended in turn and read by tokens, against the dense layer over all states. The layer rounds nine results
    in turn either way (the dense path the turned queries as well): ten roundings on each side."""
    r = make()
    B, T, L, page = 2, 130, 5, 48
    cache, tables = r.new_cache(B, 3 * T, page=page, dtype=dt, masked=True)
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    frames, places, masks = [], [], []
    for f in range(3):
        frames.append(rand(B, T, 56, dt=dt, seed=10 + f))
        places.append(where(B, T, f, 20 + f))
        masks.append(rand(B, T, seed=30 + f) < 0.5)
        lengths += T
        r.append(cache, tables, lengths, frames[-1], places[-1], key_mask=masks[-1])
        x, pos = rand(B, L, 96, dt=dt, seed=40 + f), where(B, L, f, 50 + f)
        got = r.read(x, pos, cache, tables, lengths)
        with torch.no_grad():
            want = r(x, pos, torch.cat(frames, 1), torch.cat(places, 1), key_mask=torch.cat(masks, 1))
        assert got.dtype is dt
        bound = R.bound_of(dt) * 2 * 10
        assert FR.rel(got, want) <= bound
        for t in range(L):     # tokens one by one
            one = r.read(x[:, t:t + 1], pos[:, t:t + 1], cache, tables, lengths)
            assert FR.rel(one, got[:, t:t + 1]) <= bound


def test_tokens_that_read_themselves_in_order():
    """Causal reading: tokens appended one at a time see what they see when they are appended together."""
    r = make(state=96)
    n = 70
    x, pos = rand(1, n, 96, seed=1), where(1, n, 0, 2)
    cache, tables = r.new_cache(1, n, page=16, dtype=torch.float32)
    all_, lens = torch.tensor([n], device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    r.append(cache, tables, all_, x, pos)
    want = r.read(x, pos, cache, tables, all_, causal=True)
    again, tables = r.new_cache(1, n, page=16, dtype=torch.float32)
    for t in range(n):
        lens += 1
        r.append(again, tables, lens, x[:, t:t + 1], pos[:, t:t + 1])
        one = r.read(x[:, t:t + 1], pos[:, t:t + 1], again, tables, lens, causal=True)
        assert FR.rel(one, want[:, t:t + 1]) <= 10 * R.bound_of(torch.float32)
    assert FR.rel(again.k, cache.k) <= R.bound_of(torch.float32)


def test_new_reader_is_the_identity():
    r = TokenReader(64, 64, RotaryAxes((8, 8))).cuda()
    x = rand(1, 3, 64, dt=torch.bfloat16)
    assert torch.equal(r(x, torch.zeros(3, 2, device="cuda"), rand(1, 9, 64, dt=torch.bfloat16, seed=1),
                         torch.zeros(9, 2, device="cuda")), x)


def test_a_captured_serving_step():
    """Append and read of a frame in one graph, replayed over new frames with eager work in between."""
    r = make()
    B, T, L = 1, 40, 3
    dt = torch.bfloat16

    def fresh():
        c, t = r.new_cache(B, 5 * T, page=16, dtype=dt)
        return c, t, torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(state, s, spos, x, pos):
        c, t, n = state
        n.add_(T)
        r.append(c, t, n, s, spos)
        return r.read(x, pos, c, t, n)

    frames = [(rand(B, T, 56, dt=dt, seed=i), where(B, T, i, i), rand(B, L, 96, dt=dt, seed=60 + i), where(B, L, i, 70 + i))
              for i in range(4)]
    eager = fresh()
    want = [step(eager, *f).clone() for f in frames]
    state, args = fresh(), [t.clone() for t in frames[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(), *args)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(state, *args)
    for f, w in zip(frames, want):
        for a, b in zip(args, f):
            a.copy_(b)
        g.replay()
        other = fresh()
        assert torch.equal(step(other, *frames[0]), want[0])
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_reader_over_the_encoders_splats():
    """Splats of two images, at their own centres: positions and latents take gradients back into the encoder."""
    from gaussian_splat_encoder.efficient_encoder import EfficientGaussianEncoder
    torch.manual_seed(0)
    enc = EfficientGaussianEncoder(d_feature=64, variant="adaptive", fine_stride=4, residual_grid=32, channels_last=True).cuda()
    img = torch.rand(2, 3, 64, 64, device="cuda")
    out = enc(img, return_latents=True)
    lat = enc.gather_splat_latents(out)
    r = TokenReader(64, lat.shape[-1], RotaryAxes((8, 8), scale=16.0)).cuda()
    with torch.no_grad():
        r.gate1.fill_(1.0), r.gate2.fill_(1.0)
    x = rand(2, 4, 64)
    y = r(x, torch.full((4, 2), 0.5, device="cuda"), lat, out["mu"], key_mask=out["opacity"] > 0.1)
    y.square().mean().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in r.parameters())
    mu = enc.fine_head.mu_head.weight.grad
    assert mu is not None and bool(torch.isfinite(mu).all()) and bool(mu.any())
    cache, tables = r.new_cache(2, lat.shape[1], dtype=torch.float32, masked=True)
    n = torch.full((2,), lat.shape[1], device="cuda")
    r.append(cache, tables, n, lat, out["mu"].detach(), key_mask=out["opacity"] > 0.1)
    got = r.read(x, torch.full((2, 4, 2), 0.5, device="cuda"), cache, tables, n)
    assert FR.rel(got, y) <= 20 * R.bound_of(torch.float32)
    assert math.isfinite(got.sum().item())
