"""The feature operators on the GPU against plain float64 implementations: types, ragged sizes, strides, masks that leave
rows empty, NaN in what is left out, gradients, repeatability."""

import math

import pytest
import torch

import _feature_ref as R
from gaussian_splat_encoder import feature_ops as F

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
ACTS = ["none", "gelu", "silu", "relu", "tanh", "sigmoid"]


def rand(*shape, dt=torch.float32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)


def compare(fn, ref, inputs, dt, seed=99, bound=None):
    """Outputs and every gradient of fn against ref in float64 on the same inputs; returns the outputs."""
    bound = R.BOUND[dt] if bound is None else bound
    a = [None if t is None else t.detach().requires_grad_(True) for t in inputs]
    d = [None if t is None else t.detach().double().requires_grad_(True) for t in inputs]
    y, z = fn(*a), ref(*d)
    assert y.dtype is dt
    g = rand(*y.shape, dt=dt, seed=seed)
    names = [i for i, t in enumerate(a) if t is not None]
    ga = torch.autograd.grad(y, [a[i] for i in names], g)
    gd = torch.autograd.grad(z, [d[i] for i in names], g.double())
    errs = {"y": R.rel(y, z)}
    errs.update((i, R.rel(p, q)) for i, p, q in zip(names, ga, gd))
    assert all(e <= bound for e in errs.values()), errs
    with torch.no_grad():
        assert torch.equal(fn(*a), y)   # the inference path, and a second run
    return [y, *ga]


# ------------------------------------------------------------------------------------------------ group norm
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("name", ACTS)
def test_norm_activations(dt, first, name):
    x, w, b = rand(2, 9, 7, 24, dt=dt, shift=0.3), rand(24, seed=1, scale=0.3, shift=1.0), rand(24, seed=2, scale=0.3)
    compare(lambda x, w, b: F.group_norm_act(x, 4, w, b, act=name, act_first=first),
            lambda x, w, b: R.group_norm_act(x, 4, w, b, 1e-5, name, first), [x, w, b], dt)


# positions and channels around the chunk (4 or 8 values), the workgroup's rows, the register path's end, one group to
# groups of one channel, groups wider than a workgroup's channels
NORM_SHAPES = [(1, 1, 16, 2), (2, 2, 3, 1), (3, 5, 33, 11), (1, 4097, 8, 8), (2, 1000, 64, 8), (1, 20000, 64, 8),
               (5, 513, 20, 4), (1, 300, 132, 12), (2, 7, 4608, 1), (1, 31, 9000, 2), (1, 17, 5000, 5), (40, 50, 12, 3)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,L,C,G", NORM_SHAPES)
def test_norm_shapes(dt, B, L, C, G):
    x, w, b = rand(B, L, C, dt=dt, shift=-0.2), rand(C, seed=1, scale=0.3, shift=1.0), rand(C, seed=2, scale=0.3)
    compare(lambda x, w, b: F.group_norm_act(x, G, w, b, act="gelu", act_first=True),
            lambda x, w, b: R.group_norm_act(x, G, w, b, 1e-5, "gelu", True), [x, w, b], dt)
    compare(lambda x, w: F.group_norm_act(x, G, w, None, eps=1e-3, act="silu"),
            lambda x, w: R.group_norm_act(x, G, w, None, 1e-3, "silu", False), [x, w], dt)
    compare(lambda x: F.group_norm_act(x, G, act="none"), lambda x: R.group_norm_act(x, G, None, None, 1e-5, "none", False),
            [x], dt)


def test_norm_far_mean():
    """A mean a thousand deviations from zero: the statistics may not cancel. The inputs themselves carry 2^-24 of the
    mean, the same in the reference; the kernel's sums may add a few more units of it per value of deviation 1."""
    for L in (64, 30000):
        x = rand(1, L, 32, shift=1000.0)
        y = F.group_norm_act(x, 4, act="none")
        ref = R.group_norm_act(x.double(), 4, None, None, 1e-5, "none", False)
        assert (y.double() - ref).abs().max().item() < 1000 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dt", TYPES)
def test_norm_strides(dt):
    """NCHW tensors in channels-last memory, channel slices, cropped maps and expanded gradients."""
    x = rand(2, 24, 10, 12, dt=dt).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    big = rand(2, 10, 12, 40, dt=dt)
    for v in (x, big[..., 7:31], big[:, 1:9, 2:7, 3:27], big.transpose(1, 3)[:, :24].transpose(1, 3)[..., :8]):
        C = v.shape[-1]
        y = F.group_norm_act(v, 4, act="gelu")
        assert torch.equal(y, F.group_norm_act(v.contiguous(), 4, act="gelu"))
        assert R.rel(y, R.group_norm_act(v.double(), 4, None, None, 1e-5, "gelu", False)) <= R.BOUND[dt], C
    v = big[..., 7:31].detach().requires_grad_(True)
    y = F.group_norm_act(v, 4, act="gelu")
    one, = torch.autograd.grad(y, v, torch.ones_like(y), retain_graph=True)
    two, = torch.autograd.grad(y.sum(), v)   # an expanded gradient of strides zero
    assert torch.equal(one, two)


def test_norm_nan_stays_in_its_group():
    x = rand(2, 2000, 16)
    x[1, 700, 5] = math.nan
    y = F.group_norm_act(x, 4, act="none")
    bad = torch.isnan(y)
    assert bad[1, :, 4:8].all() and bad.sum() == 2000 * 4
    x[1, 700, 5] = math.inf
    assert torch.isnan(F.group_norm_act(x, 4, act="none")[1, :, 4:8]).all()


@pytest.mark.parametrize("shape", [(0, 5, 8), (3, 0, 8), (2, 0, 4, 8)])
def test_norm_empty(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = F.group_norm_act(x, 2, w, w)
    assert y.shape == shape
    gx, gw = torch.autograd.grad(y.sum(), [x, w])
    assert gx.shape == shape and torch.equal(gw, torch.zeros_like(w))


def test_norm_of_single_values():
    """Groups of one value normalise to zero exactly, and have a zero gradient."""
    x = rand(3, 1, 8).requires_grad_(True)
    w, b = rand(8, seed=1), rand(8, seed=2)
    y = F.group_norm_act(x, 8, w, b, act="none")
    assert torch.equal(y, b.expand(3, 1, 8))
    assert torch.equal(torch.autograd.grad(y, x, rand(3, 1, 8, seed=3))[0], torch.zeros_like(x))


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_linear_activations(dt, name):
    x, w, b, r = rand(3, 50, 48, dt=dt), rand(40, 48, dt=dt, seed=1, scale=0.14), rand(40, dt=dt, seed=2), \
        rand(3, 50, 40, dt=dt, seed=3)
    # the saved input of the activation is rounded too (2^-9 of it at most), which its slope's slope carries on
    bound = R.BOUND[dt] * (1.5 if dt is torch.bfloat16 else 1)
    compare(lambda *t: F.linear_act(*t[:3], act=name, residual=t[3]), lambda *t: R.linear_act(*t[:3], name, t[3]),
            [x, w, b, r], dt, bound=bound)


LINEAR_SHAPES = [(1, 1, 1), (1, 256, 1024), (2, 7, 3), (5, 33, 31), (17, 64, 129), (33, 257, 32), (130, 133, 18),
                 (300, 512, 40), (1000, 40, 300), (129, 1030, 127), (5000, 24, 5), (2048, 128, 2048), (257, 65, 4096)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,N", LINEAR_SHAPES)
def test_linear_shapes(dt, M, K, N):
    x, w, b = rand(M, K, dt=dt), rand(N, K, dt=dt, seed=1, scale=K ** -0.5), rand(N, dt=dt, seed=2)
    compare(lambda *t: F.linear_act(*t), lambda *t: R.linear_act(*t, "none", None), [x, w, b], dt)
    r = rand(M, N, dt=dt, seed=4)
    compare(lambda x, w, r: F.linear_act(x, w, None, residual=r), lambda x, w, r: R.linear_act(x, w, None, "none", r),
            [x, w, r], dt)


@pytest.mark.parametrize("dt", TYPES)
def test_linear_strides_and_partial_gradients(dt):
    big, res = rand(70, 3, 100, dt=dt), rand(70, 90, dt=dt, seed=5)
    w, b = rand(36, 64, dt=dt, seed=1, scale=0.1), rand(36, dt=dt, seed=2)
    for x in (big[:, 1, 5:69], big[:, 2, :64], big.permute(2, 1, 0)[:64, 0].t(), big[:, :1, 3:67].expand(70, 3, 64)[:, 2]):
        y = F.linear_act(x, w, b, act="gelu", residual=res[:, 11:47])
        ref = R.linear_act(x.double(), w.double(), b.double(), "gelu", res[:, 11:47].double())
        assert R.rel(y, ref) <= R.BOUND[dt]
    x = big[:, 0, 1:65]
    full = None
    for which in ((0, 1, 2), (0,), (1,), (2,), (1, 2)):
        a = [t.detach().clone().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
        y = F.linear_act(*a, act="silu")
        got = dict(zip(which, torch.autograd.grad(y, [a[i] for i in which], rand(70, 36, dt=dt, seed=8))))
        full = full or got
        assert all(torch.equal(got[i], full[i]) for i in which)
    wt = rand(64, 36, dt=dt, seed=1, scale=0.1).t()   # a weight that is not laid out row by row
    assert torch.equal(F.linear_act(x, wt), F.linear_act(x, wt.contiguous()))
    one = rand(70, 1, dt=dt, seed=3).expand(70, 64)
    assert torch.equal(F.linear_act(one, w), F.linear_act(one.contiguous(), w))


@pytest.mark.parametrize("dt", TYPES)
def test_linear_empty_and_nan(dt):
    w = rand(5, 8, dt=dt).requires_grad_(True)
    b = rand(5, dt=dt).requires_grad_(True)
    x = torch.zeros(0, 8, device="cuda", dtype=dt, requires_grad=True)
    y = F.linear_act(x, w, b, act="gelu")
    gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == (0, 5) and gx.shape == (0, 8) and not gw.any() and not gb.any()
    x = rand(40, 8, dt=dt)
    x[7, 3] = math.nan
    y = F.linear_act(x, w, b)
    assert torch.isnan(y[7]).all() and torch.isnan(y).sum() == 5


def test_linear_activation_inputs_out_of_the_kept_range():
    """Inputs of the activation past a half's range, and positive ones below it: the slopes are the limits', 1 for a relu of
    any positive value."""
    w = torch.eye(8, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    x = torch.tensor([[1e30, -1e30, 1e5, -1e5, 1e-30, -1e-30, 3.0, -3.0]], device="cuda").bfloat16().requires_grad_(True)
    for name, want in (("relu", [1, 0, 1, 0, 1, 0, 1, 0]), ("gelu", [1, 0, 1, 0, 0.5, 0.5, 1.0119, -0.0119]),
                       ("sigmoid", [0, 0, 0, 0, 0.25, 0.25, 0.0452, 0.0452])):
        y = F.linear_act(x, w, act=name)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.allclose(g.float()[0], torch.tensor(want, device="cuda", dtype=torch.float32), atol=2.0 ** -8), name


# ------------------------------------------------------------------------------------------------ cross attention
def qkv(B, Lq, Lk, H, Hk, D, dt, scale=1.5):
    kv = rand(B, Lk, 2, Hk, D, dt=dt, seed=1)
    return rand(B, Lq, H, D, dt=dt, scale=scale), kv[:, :, 0], kv[:, :, 1]


# one token to several tiles of rows and keys (32, 64, 128), either side longer, shared heads, head widths around the
# chunk and the 32-wide blocks
ATTN_SHAPES = [(1, 1, 1, 1, 1, 8), (1, 1, 1000, 4, 4, 64), (3, 1, 77, 6, 2, 40), (2, 5, 3, 2, 1, 33), (1, 16, 5000, 8, 2, 64),
               (2, 32, 129, 3, 3, 32), (1, 33, 64, 2, 2, 96), (1, 200, 130, 4, 1, 128), (2, 300, 31, 2, 2, 1),
               (1, 1025, 65, 1, 1, 16), (1, 70, 1500, 4, 2, 100), (1, 2000, 2000, 2, 1, 64)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D", ATTN_SHAPES)
def test_attention_shapes(dt, B, Lq, Lk, H, Hk, D):
    q, k, v = qkv(B, Lq, Lk, H, Hk, D, dt)
    if Lk > 1:
        compare(lambda *t: F.cross_attention(*t), lambda *t: R.cross_attention(*t, None, None, D ** -0.5), [q, k, v], dt,
                bound=attn_bound(dt, Lk))
    else:   # a softmax over one key is constant: zero gradients of q and k up to rounding
        y = F.cross_attention(q, k, v)
        assert R.rel(y, v.double().expand(q.shape)) <= R.BOUND[dt]


def attn_bound(dt, Lk):
    """Gradients take dp - rowsum(do o) from an output rounded to bf16: with few keys that difference is of the output's
    own size, and its rounding (2^-9) counts beside the score gradient's."""
    return R.BOUND[dt] * (2 if dt is torch.bfloat16 and Lk < 200 else 1)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Lq", [1, 45, 200])
@pytest.mark.parametrize("kind", ["lengths", "mask", "both"])
def test_attention_masks(dt, Lq, kind):
    """Images with all, one, some and no keys; what is left out holds NaN and infinities; gradients there are zero."""
    B, Lk, H, Hk, D = 5, 390, 4, 2, 48
    q, k, v = qkv(B, Lq, Lk, H, Hk, D, dt)
    lengths = torch.tensor([390, 64, 0, 129, 385], device="cuda", dtype=torch.int64) if kind != "mask" else None
    mask = None
    if kind != "lengths":
        mask = torch.rand(B, Lk, generator=torch.Generator("cuda").manual_seed(3), device="cuda") < 0.5
        mask[2] = False
        mask[0, 64:192] = False   # whole tiles without keys
    ok = R.valid(q, k, lengths, mask)
    bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=dt)
    pick = torch.arange(Lk, device="cuda") % 3
    k = torch.where(ok[:, :, None, None], k, bad[pick][None, :, None, None].expand_as(k))
    v = torch.where(ok[:, :, None, None], v, bad[pick][None, :, None, None].expand_as(v))
    y, dq, dk, dv = compare(lambda *t: F.cross_attention(*t, kv_lengths=lengths, key_mask=mask, scale=0.2),
                            lambda *t: R.cross_attention(*t, lengths, mask, 0.2), [q, k, v], dt, bound=attn_bound(dt, 64))
    assert not y[2].any() and not dq[2].any()
    off = ~ok[:, :, None, None].expand_as(dk)
    assert not dk[off].any() and not dv[off].any()


def test_attention_lengths_past_the_keys():
    q, k, v = qkv(2, 3, 50, 2, 2, 16, torch.float32)
    n = torch.tensor([10 ** 6, -5], device="cuda", dtype=torch.int32)
    y = F.cross_attention(q, k, v, kv_lengths=n)
    assert torch.equal(y[0], F.cross_attention(q, k, v)[0]) and not y[1].any()
    big = F.cross_attention(q, k, v, kv_lengths=torch.tensor([2 ** 32, -2 ** 40], device="cuda"))
    assert torch.equal(big, y)


@pytest.mark.parametrize("dt", TYPES)
def test_attention_strides(dt):
    """Heads before tokens, odd offsets, expanded keys, a strided mask: the same bits as contiguous copies."""
    q = rand(2, 4, 70, 41, dt=dt).transpose(1, 2)[..., 1:]
    k = rand(2, 4, 130, 43, dt=dt, seed=1).transpose(1, 2)[..., 2:42]
    v = rand(1, 130, 1, 45, dt=dt, seed=2).expand(2, 130, 4, 45)[..., 3:43]
    mask = (rand(130, 4, seed=3) > 0)[:, ::2].t()
    y = F.cross_attention(q, k, v, key_mask=mask)
    assert torch.equal(y, F.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), key_mask=mask.contiguous()))
    assert R.rel(y, R.cross_attention(q.double(), k.double(), v.double(), None, mask, 40 ** -0.5)) <= R.BOUND[dt]
    flip = rand(2, 40, 130, 4, dt=dt, seed=1).permute(0, 2, 3, 1)   # head vectors that are not dense
    assert torch.equal(F.cross_attention(q, flip, v), F.cross_attention(q, flip.contiguous(), v))


@pytest.mark.parametrize("B,Lq,Lk", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_attention_empty(B, Lq, Lk):
    q, k, v = (t.detach().requires_grad_(True) for t in qkv(B, Lq, Lk, 2, 1, 16, torch.float32))
    y = F.cross_attention(q, k, v)
    assert y.shape == q.shape and not y.any()
    for t, g in zip((q, k, v), torch.autograd.grad(y.sum(), [q, k, v])):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dt", TYPES)
def test_attention_large_scores(dt):
    """Scores of some thousands, where exp overflows: the running maximum keeps the softmax finite."""
    q, k, v = qkv(1, 40, 300, 2, 2, 32, dt, scale=100.0)
    y = F.cross_attention(q, k, v, scale=10.0)
    ref = R.cross_attention(q.double(), k.double(), v.double(), None, None, 10.0)
    # a score of 1e4 carries 2^-24 of itself into the exponent, about 1e-3 of a probability
    assert torch.isfinite(y).all() and R.rel(y, ref) <= (4e-3 if dt is torch.float32 else 8e-3)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
def test_attention_scales(dt, scale):
    """A negative scale turns the order of the scores round; zero weighs all keys alike."""
    q, k, v = qkv(2, 70, 333, 4, 2, 40, dt)
    ins = [q, k, v]
    if scale == -0.3:
        compare(lambda *t: F.cross_attention(*t, scale=scale), lambda *t: R.cross_attention(*t, None, None, scale), ins, dt)
    else:   # the gradients of q and k vanish with the scale
        y = F.cross_attention(*ins, scale=scale)
        assert R.rel(y, v.double().mean(1, keepdim=True).repeat_interleave(2, 2).expand(q.shape)) <= R.BOUND[dt]


def test_second_derivatives_are_refused():
    x = rand(4, 8).requires_grad_(True)
    w = rand(8, 8, seed=1).requires_grad_(True)
    g, = torch.autograd.grad(F.linear_act(x, w, act="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_saved_tensors_that_come_back_dense():
    """Hooks that move what a backward keeps may give strided views back as dense tensors; the gradients stay the same."""
    big = rand(2, 10, 12, 40)
    calls = {"norm": (lambda v: F.group_norm_act(v, 4, act="gelu"), big[:, 1:9, 2:7, 3:27]),
             "linear": (lambda v: F.linear_act(v, rand(8, 24, seed=1), act="silu"), big[:, :, 3, 3:27]),
             "attention": (lambda v: F.cross_attention(rand(2, 7, 4, 24, seed=2), v, v), big[:, :, 2:4, 3:27])}
    for name, (fn, view) in calls.items():
        v = view.detach().requires_grad_(True)
        assert not v.is_contiguous(), name
        y = fn(v)
        up = rand(*y.shape, seed=3)
        want, = torch.autograd.grad(y, v, up)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.cuda()):
            y = fn(v)
        got, = torch.autograd.grad(y, v, up)
        assert torch.equal(got, want), name


def test_gradients_against_differences():
    """Directional differences of the float32 kernels' own outputs, in the middle of their precision: a step of 2^-9 leaves
    an error of order 2^-18 from the curvature and 2^-24 * 2^9 from rounding, relative to the output's norm."""
    x, w, b = rand(2, 30, 24, shift=0.1), rand(24, seed=1, scale=0.2, shift=1), rand(24, seed=2)
    q, k, v = (t.contiguous() for t in qkv(1, 20, 40, 2, 1, 16, torch.float32, scale=1.0))
    calls = [(lambda x, w, b: F.group_norm_act(x, 4, w, b, act="gelu"), [x, w, b]),
             (lambda x, w, b: F.group_norm_act(x, 4, w, b, act="silu", act_first=True), [x, w, b]),
             (lambda x, w, b: F.linear_act(x, w, b, act="tanh"), [x, rand(10, 24, seed=3, scale=0.2), rand(10, seed=4)]),
             (lambda *t: F.cross_attention(*t), [q, k, v])]
    for fn, ins in calls:
        for i in range(len(ins)):
            a = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(ins)]
            y = fn(*a)
            g, d = rand(*y.shape, seed=5), rand(*ins[i].shape, seed=6)
            want = (torch.autograd.grad(y, a[i], g)[0].double() * d.double()).sum().item()
            h = 2.0 ** -9
            with torch.no_grad():
                up = fn(*[t + h * d if j == i else t for j, t in enumerate(ins)]).double()
                dn = fn(*[t - h * d if j == i else t for j, t in enumerate(ins)]).double()
            got = ((up - dn) * g.double()).sum().item() / (2 * h)
            size = y.double().norm().item() * g.double().norm().item()
            assert abs(got - want) <= 1e-3 * size, (i, got, want, size)


def test_another_stream():
    """Calls on a side stream, with inputs made there: the same bits as on the default stream."""
    s = torch.cuda.Stream()
    q, k, v = qkv(1, 64, 700, 2, 2, 64, torch.bfloat16)
    x, w = rand(1, 5000, 64, dt=torch.bfloat16), rand(96, 64, dt=torch.bfloat16, seed=1)
    want = [F.cross_attention(q, k, v), F.group_norm_act(x, 8), F.linear_act(x, w, act="gelu")]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [F.cross_attention(q.clone(), k.clone(), v.clone()), F.group_norm_act(x.clone(), 8),
               F.linear_act(x.clone(), w.clone(), act="gelu")]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: their far ends give what the same rows give alone."""
    M = 2 ** 31 // 32 + 4099
    x = torch.empty(M, 32, device="cuda", dtype=torch.bfloat16)
    x.copy_(rand(1, 32, dt=torch.bfloat16).expand(M, 32))
    tail = rand(300, 32, dt=torch.bfloat16, seed=3)
    x[-300:] = tail
    w = rand(40, 32, dt=torch.bfloat16, seed=1)
    y = F.linear_act(x, w, act="gelu")
    assert torch.equal(y[-300:], F.linear_act(tail, w, act="gelu")) and torch.equal(y[:1], F.linear_act(x[:1], w, act="gelu"))
    del y
    # one image whose far half is the near one negated: the mean is zero, and the far end is the near one negated
    half = M // 2
    x[half:2 * half] = -x[:half]
    x[2 * half:] = 0
    y = F.group_norm_act(x[None, :2 * half], 1, act="none")[0]
    assert torch.isfinite(y[-1]).all() and (y[half:half + 100].float() + y[:100].float()).abs().max() <= 2.0 ** -6
    del x, y
    # a cache whose keys lie 40,000 elements apart
    big = torch.zeros(60000, 40000, device="cuda", dtype=torch.bfloat16)
    big[:, :128] = rand(60000, 128, dt=torch.bfloat16, seed=5)
    k, v = big[None, :, None, :64], big[None, :, None, 64:128]
    q = rand(1, 2, 1, 64, dt=torch.bfloat16)
    assert torch.equal(F.cross_attention(q, k, v), F.cross_attention(q, k.contiguous(), v.contiguous()))


def test_graph_replays():
    """A captured chain of the operators gives the eager result on every replay, with eager work in between."""
    q, k, v = qkv(2, 40, 3000, 4, 2, 64, torch.bfloat16)
    w = rand(256, 256, dt=torch.bfloat16, seed=4, scale=0.1)
    mask = torch.rand(2, 3000, generator=torch.Generator("cuda").manual_seed(3), device="cuda") < 0.5

    def chain():
        a = F.cross_attention(q, k, v, key_mask=mask).reshape(2, 40, 256)
        return F.linear_act(F.group_norm_act(a, 8, act="silu"), w, act="gelu", residual=a)

    want = chain()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = chain()
    for _ in range(4):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(chain(), want)
