"""The feature operators on the GPU where sizes, types and values are at an end of their range."""

import math

import pytest
import torch

import _feature_ref as R
from gaussian_splat_encoder import feature_ops as F
from gaussian_splat_encoder.cell_reader import CellReader

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def rand(*shape, dt=torch.float32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,G", [((70000, 24), 4), ((65536, 3, 16), 2), ((92160, 1, 20), 20)])
def test_norm_of_many_images(dt, shape, G):
    """More images than a grid's second and third dimensions hold: one norm per token."""
    x, w, b = rand(*shape, dt=dt, shift=0.2), rand(shape[-1], seed=1, scale=0.3, shift=1.0), rand(shape[-1], seed=2)
    a = [t.requires_grad_(True) for t in (x, w, b)]
    d = [t.detach().double().requires_grad_(True) for t in (x, w, b)]
    y, z = F.group_norm_act(a[0], G, a[1], a[2], act="gelu"), R.group_norm_act(*d[:1], G, *d[1:], 1e-5, "gelu", False)
    g = rand(*shape, dt=dt, seed=3)
    got, want = torch.autograd.grad(y, a, g), torch.autograd.grad(z, d, g.double())
    errs = [R.rel(p, q) for p, q in zip((y, *got), (z, *want))]
    assert all(e <= R.BOUND[dt] for e in errs), errs
    if dt is torch.float32:   # the far end, element by element
        assert torch.allclose(y[-5:].double(), z[-5:], atol=1e-5)


@pytest.mark.parametrize("dt", TYPES)
def test_reader_of_no_images(dt):
    """An empty batch gives an empty batch, forward and backward, as the operators do."""
    m = CellReader(32, 16).cuda()
    x = torch.zeros(0, 4, 5, 32, device="cuda", dtype=dt, requires_grad=True)
    y = m(x, torch.zeros(0, 3, 16, device="cuda", dtype=dt))
    gx, = torch.autograd.grad(y.sum(), x)
    assert y.shape == x.shape and y.dtype is dt and gx.shape == x.shape
    none = m(torch.randn(2, 0, 32, device="cuda").to(dt), torch.randn(2, 0, 16, device="cuda").to(dt))
    assert none.shape == (2, 0, 32)


@pytest.mark.parametrize("M", [4096, 16384])
def test_slopes_keep_their_mean(M):
    """The bias gradient of tanh over bfloat16 rows, against its formula, in the mean over 1,024 columns of different sizes.
    Rounding the kept input to the nearest half goes either way and leaves that mean; the results' own rounding to bfloat16
    moves it by 2^-8 / sqrt(12) / sqrt(1024) = 3.5e-5 of standard deviation at most, and 1.5e-4 is four times that. Cutting
    bits of the input off would move every slope one way, by 2 tanh(z) 2^-12 = 3e-4 for inputs from 0.5 to 1."""
    z = torch.rand(M, 1024, generator=torch.Generator("cuda").manual_seed(4), device="cuda") * 0.5 + 0.5
    hi = z.bfloat16()
    lo = (z - hi.float()).bfloat16()   # the product adds the two exactly: inputs of more bits than a half's 11
    w = torch.eye(64, device="cuda", dtype=torch.bfloat16).repeat(1, 2)
    up = (1 + torch.arange(1024, device="cuda") % 128 / 128).bfloat16()
    got = []
    for c in range(0, 1024, 64):
        b = torch.zeros(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = F.linear_act(torch.cat([hi[:, c:c + 64], lo[:, c:c + 64]], 1), w, b, act="tanh")
        got.append(torch.autograd.grad(y, b, up[c:c + 64].expand_as(y))[0].double())
    want = (up.double() * (1 - torch.tanh(hi.double() + lo.double()) ** 2)).sum(0)
    off = (torch.cat(got) / want - 1).mean().abs().item()
    print(f"mean error of the slopes {off:.1e}", flush=True)
    assert off < 1.5e-4


def test_kept_inputs_hold_nan_and_infinities():
    """NaN in a row reaches its gradient; infinite inputs of gelu and silu have the limits' slopes, past a half's range too."""
    w = torch.eye(4, device="cuda", dtype=torch.bfloat16)
    for name, want in (("gelu", (1, 0)), ("silu", (1, 0)), ("relu", (1, 0)), ("tanh", (0, 0)), ("sigmoid", (0, 0))):
        for dt in TYPES:
            x = torch.tensor([[7e4, -7e4, 3e38, -3e38], [0, 0, math.nan, 0]], device="cuda", dtype=dt).requires_grad_(True)
            y = F.linear_act(x, w.to(dt), act=name)
            g, = torch.autograd.grad(y, x, torch.ones_like(y))
            assert g[0].tolist() == [want[0], want[1]] * 2, (name, dt, g)
            if name != "relu":
                assert torch.isnan(g[1]).all(), (name, dt, g)


@pytest.mark.parametrize("name", ["gelu", "silu", "relu", "tanh", "sigmoid"])
def test_activations_point_by_point(name):
    """float32 activations over a fine grid, the product being the value itself. An error of 2^-20 (9.5e-7) at most: half a
    unit of results up to 8 (2.4e-7), a unit of the reciprocal times x (6e-8 * 8), half of one of its argument, and 7e-8 of
    gelu's fit."""
    x = torch.linspace(-8, 8, 1 << 20, device="cuda")[:, None]
    y = F.linear_act(x, torch.ones(1, 1, device="cuda"), act=name)
    err = (y.double() - R.act(x.double(), name)).abs()
    print(f"{name}: {err.max().item():.2e} at x = {x[err.argmax()].item():.3f}", flush=True)
    assert err.max().item() <= 2.0 ** -20


def test_norm_offsets_past_32_bits():
    """One image of more than 2^31 values, whose last 4,000 rows are values of their own and, negated, the rows of the first
    half's end: outputs and gradients there are the negated ones exactly, as the mean is zero and all sums are alike."""
    M = 2 ** 31 // 32 + 4099
    half = M // 2 + 1
    x = torch.empty(1, 2 * half, 32, device="cuda", dtype=torch.bfloat16)
    x[0, :half] = rand(1, 32, dt=torch.bfloat16)
    x[0, half - 4000:half] = rand(4000, 32, dt=torch.bfloat16, seed=1)
    x[0, half:] = -x[0, :half]
    assert (2 * half - 4000) * 32 > 2 ** 31
    x.requires_grad_(True)
    y = F.group_norm_act(x, 1, act="none")
    far, near = y[0, -4000:].float(), y[0, half - 4000:half].float()
    # the sums of the two halves come in other orders: a mean of 2^-24 of the deviation may be left
    ref = rand(4000, 32, dt=torch.bfloat16, seed=1).float() / x.detach()[0, :half].float().square().mean().sqrt()
    assert (far + near).abs().max() <= 2.0 ** -7 * near.abs().max() and R.rel(near, ref) <= R.BOUND[torch.bfloat16]
    assert R.rel(far, -ref) <= R.BOUND[torch.bfloat16]
    g = torch.zeros_like(y)
    g[0, -4000:] = rand(4000, 32, dt=torch.bfloat16, seed=2)
    g[0, half - 4000:half] = -g[0, -4000:]
    dx, = torch.autograd.grad(y, x, g)
    # the gradient's sums vanish against 2^31 values: dx is g / deviation but for 4,000 * 32 terms over them
    rstd = 1 / x.detach()[0, :half].float().square().mean().sqrt()
    want = g[0, -4000:].float() * rstd
    assert R.rel(dx[0, -4000:], want) <= R.BOUND[torch.bfloat16]
    assert R.rel(dx[0, half - 4000:half], -want) <= R.BOUND[torch.bfloat16]
    assert dx[0, :half - 4000].abs().max() <= 1e-3


def test_linear_gradient_offsets_past_32_bits():
    """Rows and their gradients of more than 2^31 values: the far end gives what the same rows give alone."""
    M = 2 ** 31 // 32 + 4099
    x = torch.zeros(M, 32, device="cuda", dtype=torch.bfloat16)
    x[-300:] = rand(300, 32, dt=torch.bfloat16, seed=3)
    w = rand(32, 32, dt=torch.bfloat16, seed=1, scale=0.2)
    g = torch.zeros(M, 32, device="cuda", dtype=torch.bfloat16)
    g[-300:] = rand(300, 32, dt=torch.bfloat16, seed=5)

    def grads(x, g):
        a = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
        return torch.autograd.grad(F.linear_act(*a, act="gelu"), a, g)

    (dx, dw), (tx, tw) = grads(x, g), grads(x[-300:].clone(), g[-300:].clone())
    bound = R.BOUND[torch.bfloat16]
    assert R.rel(dx[-300:], tx) <= bound and R.rel(dw, tw) <= bound and not dx[:-300].any()


def test_attention_gradient_offsets_past_32_bits():
    """Queries, keys, values and the output's gradient whose rows lie 40,000 values apart, over 2^31 values in all: the bits
    of dense copies, forward and backward."""
    big = torch.zeros(60000, 40000, device="cuda", dtype=torch.bfloat16)
    big[:, :256] = rand(60000, 256, dt=torch.bfloat16, seed=5)
    views = [big[None, :, None, i:i + 64] for i in (0, 64, 128, 192)]

    def grads(q, k, v, g):
        a = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = F.cross_attention(*a)
        return [y, *torch.autograd.grad(y, a, g)]

    assert all(torch.equal(a, b) for a, b in zip(grads(*views), grads(*[t.contiguous() for t in views])))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,full", [(80, 96), (88, 96), (112, 128), (120, 128)])
def test_attention_of_part_heads_costs_no_more(dt, D, full):
    """Heads that fill a part of their blocks of 32 values do a part of the full heads' work, forward and backward. (Rows
    kept in memory instead of registers took 1.9 times as long; half as long again is left for noise.)"""
    def step(d):
        a = [rand(1, 4096, 4, d, dt=dt, seed=i).requires_grad_(True) for i in range(3)]
        g = rand(1, 4096, 4, d, dt=dt, seed=3)
        return lambda: torch.autograd.grad(F.cross_attention(*a), a, g)

    times = {D: [], full: []}
    calls = {d: step(d) for d in times}
    for i in range(12):
        for d, call in calls.items():
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            call()
            start.record()
            for _ in range(4):
                call()
            end.record()
            torch.cuda.synchronize()
            times[d].append(start.elapsed_time(end))
    part, whole = min(times[D]), min(times[full])
    print(f"{dt}: heads of {D} {part / 4:.3f} ms, of {full} {whole / 4:.3f} ms", flush=True)
    assert part < 1.5 * whole


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,scale", [(2, 300, 8, 4, 4, 32, 1.5), (2, 300, 70, 4, 2, 32, 4.0),
                                                  (3, 600, 71, 4, 2, 40, 1.5), (1, 1000, 2000, 4, 4, 16, 1.5)])
def test_attention_gradients_round_twice(B, Lq, Lk, H, Hk, D, scale):
    """bfloat16 results carry two roundings: the probabilities' or score gradients' before the second product, and their
    own. A rounding is 1.66e-3 in the 2-norm of normal values, two are 2.35e-3, three (the output's, which the score
    gradients are taken against) 2.9e-3, and more where a few keys hold most of the weight: 2.6e-3 lies between."""
    dt = torch.bfloat16
    kv = rand(B, Lk, 2, Hk, D, dt=dt, seed=1)
    a = [t.requires_grad_(True) for t in (rand(B, Lq, H, D, dt=dt, scale=scale), kv[:, :, 0].clone(), kv[:, :, 1].clone())]
    d = [t.detach().double().requires_grad_(True) for t in a]
    y, z, g = F.cross_attention(*a), R.cross_attention(*d, None, None, D ** -0.5), rand(B, Lq, H, D, dt=dt, seed=3)
    got, want = torch.autograd.grad(y, a, g), torch.autograd.grad(z, d, g.double())
    errs = [R.rel(p, q) for p, q in zip((y, *got), (z, *want))]
    print(" ".join(f"{e:.2e}" for e in errs), flush=True)
    assert max(errs) <= 2.6e-3


@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", [(3, 1, 3000, 4, 4, 16), (2, 1, 102, 2, 2, 32), (4, 7, 613, 2, 2, 96),
                                            (5, 1, 300, 8, 2, 64), (3, 2, 8, 16, 4, 64), (1, 64, 33, 1, 1, 40)])
def test_attention_of_few_rows_rounds_once(B, Lq, Lk, H, Hk, D):
    """Few rows' roundings do not average out: there bfloat16 results and gradients carry their own alone, to a tenth of it."""
    dt = torch.bfloat16
    kv = rand(B, Lk, 2, Hk, D, dt=dt, seed=1)
    a = [t.requires_grad_(True) for t in (rand(B, Lq, H, D, dt=dt, scale=1.5), kv[:, :, 0].clone(), kv[:, :, 1].clone())]
    d = [t.detach().double().requires_grad_(True) for t in a]
    y, z, g = F.cross_attention(*a), R.cross_attention(*d, None, None, D ** -0.5), rand(B, Lq, H, D, dt=dt, seed=3)
    got, want = torch.autograd.grad(y, a, g), torch.autograd.grad(z, d, g.double())
    errs = [(R.rel(p, q), R.rel(q.to(dt), q)) for p, q in zip((y, *got), (z, *want))]
    print(" ".join(f"{e:.2e}/{o:.2e}" for e, o in errs), flush=True)
    assert all(e <= 1.1 * o for e, o in errs), errs


def test_attention_rows_keep_their_sums():
    """One row's probabilities share its statistics: taken from the logarithm of their sum (about 20, whose last bit is 2e-6,
    7e-7 of a probability after 2^x) each row's gradients would be off by that together. Over 24 rows of as many images the
    mean of it stays below a third of it: a float32 gradient's other roundings go either way."""
    B, Lk, D = 24, 30000, 40
    q, k, v, g = (rand(*s, seed=i) for i, s in enumerate([(B, 1, 1, D), (B, Lk, 1, D), (B, Lk, 1, D), (B, 1, 1, D)]))
    a = [t.requires_grad_(True) for t in (q, k, v)]
    dv = torch.autograd.grad(F.cross_attention(*a), a, g)[2].double()
    p = torch.softmax((q.double() * k.double()).sum(-1) * D ** -0.5, 1)
    # dv = p g: the factor that a whole row is off by, in the least squares
    want = p * g.double()[:, :, 0]
    off = (dv[:, :, 0] * want).sum((1, 2)) / (want * want).sum((1, 2)) - 1
    print(f"rows off by {off.abs().mean().item():.1e}, {off.abs().max().item():.1e} at most", flush=True)
    assert off.abs().mean().item() <= 2.3e-7


@pytest.mark.parametrize("M,K,N,name", [(76, 17, 9, "sigmoid"), (3, 212, 525, "silu"), (1304, 16, 16, "tanh"), (1, 64, 5, "gelu"),
                                        (8, 797, 17, "tanh"), (300, 400, 400, "gelu"), (9000, 24, 130, "silu")])
def test_linear_gradients_of_few_rows_or_weights_round_once(M, K, N, name):
    """Where few terms or few results do not average roundings, bfloat16 gradients carry their own alone, to a tenth of it:
    the kept input's (2^-11, in slopes that change by up to 2 z of it) is a quarter of a result's at most."""
    dt = torch.bfloat16
    a = [t.requires_grad_(True) for t in (rand(M, K, dt=dt), rand(N, K, dt=dt, seed=1, scale=K ** -0.5),
                                          rand(N, dt=dt, seed=2, scale=0.2))]
    d = [t.detach().double().requires_grad_(True) for t in a]
    y, z, g = F.linear_act(*a, act=name), R.linear_act(*d, name, None), rand(M, N, dt=dt, seed=3)
    got, want = torch.autograd.grad(y, a, g), torch.autograd.grad(z, d, g.double())
    errs = [(R.rel(p, q), R.rel(q.to(dt), q)) for p, q in zip((y, *got), (z, *want))]
    print(" ".join(f"{e:.2e}/{o:.2e}" for e, o in errs), flush=True)
    assert all(e <= 1.1 * o for e, o in errs), errs
