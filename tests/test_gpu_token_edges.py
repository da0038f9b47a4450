"""The token operators on the GPU where sizes, positions and values are at the ends of what they accept."""

import math

import pytest
import torch

import _token_ref as R
from _feature_ref import rel
from gaussian_splat_encoder import token_ops as F

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def rand(*shape, dt=torch.float32, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)


# ------------------------------------------------------------------------------------------------ positions
# nanoseconds of a clock, the ends of the types, both sides of where a 64-bit product has no quarter turns left (2^51 of them)
FAR = {torch.int64: [1765000000000000001, 2 ** 62 - 12345, -2 ** 62 + 7, 2 ** 63 - 1, -2 ** 63, 2 ** 52 + 3, -2 ** 52 - 3,
                     2 ** 50 + 11, 2 ** 53 + 2, 2 ** 31],
       torch.float32: [1e20, -1e20, 3.4e38, -3.4e38, 2.0 ** 51, -2.0 ** 53, 1e15, 6e15, -7e25, 1.5]}


def pair_norms(x, dims, interleaved):
    out, at = [], 0
    for d in dims:
        v = x[..., at:at + d].double()
        v = v.unflatten(-1, (d // 2, 2)) if interleaved else v.unflatten(-1, (2, d // 2)).transpose(-1, -2)
        out.append(v.norm(dim=-1))
        at += d
    return torch.cat(out, -1)


@pytest.mark.parametrize("kind", list(FAR))
@pytest.mark.parametrize("inter", [False, True])
def test_far_positions_still_turn(kind, inter):
    """Past 2^31 radians the angle loses its accuracy, but what comes out is a rotation: pairs keep their length. Cosines and
    sines are 1.5e-7 off at most, so that their squares' sum is 4.3e-7 off one and a length 2.2e-7; two products and a sum of
    pairs add 2 sqrt(2) 2^-24 of it."""
    p = torch.tensor(FAR[kind], dtype=kind, device="cuda")[:, None]
    n, dims = p.shape[0], (8, 6)
    p = torch.cat([p, p.flip(0)], 1).contiguous()
    ax = F.RotaryAxes(dims, base=100.0, scale=(1.0, 40.0), interleaved=inter)
    bound = 2.2e-7 + 2 * math.sqrt(2) * 2.0 ** -24
    x, g = rand(1, n, 3, 16), rand(1, n, 3, 16, seed=1)

    def same(a, b):
        return bool(((pair_norms(a, dims, inter) / pair_norms(b, dims, inter) - 1).abs() <= bound).all())

    a = x.clone().requires_grad_(True)
    y = F.rotary(a, p, ax)
    assert same(y, x) and torch.equal(y[..., 14:], x[..., 14:])
    assert same(torch.autograd.grad(y, a, g)[0], g)
    if kind is torch.float32:       # |dp| is at most the sum over pairs of rate |g| |x|
        q = p.clone().requires_grad_(True)
        dx, dp = torch.autograd.grad(F.rotary(a, q, ax), [a, q], g)
        assert same(dx, g)
        top = (pair_norms(x, dims, inter) * pair_norms(g, dims, inter)).sum((0, 2, 3))
        assert bool((dp.abs().double() <= 1.0001 * 40.0 * top.sum()).all())
    c = F.PagedCache.empty(1, n, 3, 16, dtype=torch.float32)
    tables, lengths = c.tables(1), torch.tensor([n], device="cuda")
    F.cache_append(c, tables, lengths, x, x, positions=p, axes=ax)
    assert torch.equal(c.k[0], y.detach()[0])
    o = F.cached_attention(x, c, tables, lengths, positions=p, axes=ax)
    want = R.attention(y.detach().double(), c.k, c.v, None, tables, lengths, None, True, 0.25)
    assert rel(o, want) <= R.bound_of(torch.float32)


def test_positions_that_are_no_number_stay_in_their_token():
    p = torch.tensor([[1.0], [math.inf], [2.0], [math.nan], [-math.inf], [3.0]], device="cuda")
    x = rand(1, 6, 2, 8)
    y = F.rotary(x, p, F.RotaryAxes((4,)))
    bad = torch.tensor([1, 3, 4], device="cuda")
    assert bool(torch.isnan(y[:, bad, :, :4]).all()) and torch.equal(y[..., 4:], x[..., 4:])
    good = torch.tensor([0, 2, 5], device="cuda")
    assert torch.equal(y[:, good], F.rotary(x[:, good], p[good], F.RotaryAxes((4,))))


# ------------------------------------------------------------------------------------------------ pieces
def test_one_sequence_of_nearly_2_31_tokens_among_many():
    """The most tokens that a table may have room for, cut into 4,096 pieces of 2^19, of which the last one ends past 2^31. All
    pages but the last seven of the table are one page of small values; the last seven, of other values, have most of the
    weight. Scores are sums of 8 products, exact to 2^-24 of themselves."""
    page, width, B, D, last = 65536, 32767, 65, 8, 7
    k = torch.zeros(2, page, 1, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    k[1, :, :, 0] = 10.0                     # scores: 10 in the last pages, 0 elsewhere
    v[0], v[1] = 0.25, rand(page, 1, D, dt=torch.bfloat16)
    tables = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    tables[0, -last:] = 1
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    lengths[0], lengths[B - 1] = page * width, 5
    q = torch.zeros(B, 1, 1, D, dtype=torch.bfloat16, device="cuda")
    q[:, :, :, 0] = 1.0
    c = F.PagedCache(k, v)
    for causal in (True, False):
        o = F.cached_attention(q, c, tables, lengths, causal=causal, scale=1.0)
        far, near = last * page * math.exp(10.0), (width - last) * page * 1.0
        want = (v[1, :, 0].double().mean(0) * far + 0.25 * near) / (far + near)
        assert rel(o[0, 0, 0], want) <= R.bound_of(torch.bfloat16)
        assert torch.equal(o[B - 1, 0, 0], torch.full_like(o[0, 0, 0], 0.25)) and not bool(o[1:B - 1].any())


# ------------------------------------------------------------------------------------------------ the cache and autograd
def test_an_append_under_a_saved_page_is_noticed():
    """A dense attention over a page saves it for its backward, which must not run on what an append wrote over it."""
    from gaussian_splat_encoder import feature_ops
    c = F.PagedCache.empty(1, 32, 2, 16, dtype=torch.float32)
    c.k.copy_(rand(*c.k.shape)), c.v.copy_(rand(*c.v.shape, seed=1))
    q = rand(1, 3, 2, 16, seed=2).requires_grad_(True)
    o = feature_ops.cross_attention(q, c.k, c.v)
    F.cached_attention(q.detach(), c, c.tables(1), torch.tensor([9], device="cuda"))      # only reads
    torch.autograd.grad(o.sum(), q, retain_graph=True)
    F.cache_append(c, c.tables(1), torch.tensor([9], device="cuda"), rand(1, 1, 2, 16), rand(1, 1, 2, 16))
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o.sum(), q)


# ------------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("T", [1, 6])
def test_infinite_values_that_count(T, causal):
    """Float32: an infinite value makes its column infinite in every row that sees it, also where dead tokens lie beside it, and
    leaves the other columns as they are. Scores differ by 20 at most, so that no probability vanishes."""
    H, Hk, D, page, width = 4, 2, 40, 16, 20
    g = torch.Generator("cuda").manual_seed(3)
    k, v = rand(width, page, Hk, D, seed=1), rand(width, page, Hk, D, seed=2)
    live = torch.rand(width, page, generator=g, device="cuda") < 0.5
    c = F.PagedCache(k, v, live)
    tables, lengths = c.tables(1), torch.tensor([303], device="cuda")
    q = rand(1, T, H, D, seed=4)
    clean = F.cached_attention(q, c, tables, lengths, causal=causal)
    for i, (j, d, bad) in enumerate([(0, 3, math.inf), (37, 0, -math.inf), (100, 39, math.inf), (211, 17, -math.inf),
                                     (290, 20, math.inf)]):
        p, at = j // page, j % page
        live[p, at] = True
        want = F.cached_attention(q, c, tables, lengths, causal=causal).clone()
        old = v[p, at, 0, d].clone()
        v[p, at, 0, d] = bad
        o = F.cached_attention(q, c, tables, lengths, causal=causal)
        want[:, :, :H // Hk, d] = bad
        hit = torch.isinf(want)
        assert torch.equal(o[hit], want[hit]), (j, d)
        assert rel(o[~hit], want[~hit]) <= R.bound_of(torch.float32), (j, d)
        v[p, at, 0, d] = old
    assert bool(torch.isfinite(clean).all())


# ------------------------------------------------------------------------------------------------ plans
def plan(B, H, Hk, D, T, lengths, page, width):
    """How cached_attention cuts its sequences: the way, the pieces aimed at, the units (128 tokens) and those of a piece."""
    R_ = T * H // Hk
    two = R_ > 16
    held = {32: (4, 3), 64: (3, 2), 96: (2, 1), 128: (2, 1)}[-(-D // 32) * 32][two]
    each = Hk * -(-R_ // (32 if two else 16))
    once = max(1, 256 * held // each)
    fit = B <= 64 and 2 * B <= once
    pieces = once if fit else -(-4 * 256 * held // each)
    cut = "whole" if page * width <= 128 or pieces <= 1 else "scanned" if B <= 64 else "mapped"
    units = sum(-(-n // 128) for n in lengths)
    return cut, fit, pieces, units, max(1, -(-units // pieces))


def workspace(cut, pieces, B, H, Hk, D, T):
    if cut == "whole":
        return 0
    return (16 * (pieces + B) if cut == "mapped" else 0) + 8 * B + 4 * 2 * pieces * T * H * (D + 2)


def attention(q, c, tables, lengths):
    """One token of each sequence over all its tokens in float64, sequences of a length near each other at a time."""
    B, _, H, D = q.shape
    o = torch.zeros(B, 1, H, D, dtype=torch.float64, device="cuda")
    order = sorted((n, b) for b, n in enumerate(lengths.tolist()) if n > 0)
    rep = H // c.heads
    while order:
        m = order[-1][0]
        some = [b for n, b in order if 2 * n > m][-max(1, (1 << 22) // (m * H * D)):]
        gone = set(some)
        order = [x for x in order if x[1] not in gone]
        b = torch.tensor(some, device="cuda")
        j = torch.arange(m, device="cuda")
        at = tables[b].long()[:, j.clamp(max=tables.shape[1] * c.page - 1) // c.page]
        k, v = (t[at, j % c.page].double().repeat_interleave(rep, 2) for t in (c.k, c.v))        # [n, m, H, D]
        s = (q[b].double() * k).sum(-1) * D ** -0.5
        s = s.masked_fill((j >= lengths[b][:, None])[..., None], -math.inf)
        w = torch.exp(s - s.amax(1, keepdim=True))
        o[b, 0] = (w[..., None] * v).sum(1) / w.sum(1)[..., None]
    return o


def spread(B, most, long, n):
    """B lengths of 0 to `most` tokens, every `long`-th one of n."""
    return [n - i % 77 if i % long == long // 2 else (i * 7919) % (most + 1) for i in range(B)]


# (sequences, heads, key heads, D, lengths), and the plan: how they are cut, whether all pieces fit the card at once, pieces of
# one unit of 128 tokens or of more
PLANS = [
    (2500, 2, 1, 64, spread(2500, 130, 400, 9000), "mapped", False, False),       # three rounds of 1,024 sequences
    (2500, 2, 1, 64, spread(2500, 300, 300, 60000), "mapped", False, True),
    (1025, 1, 1, 32, [0] * 1024 + [40000], "mapped", False, False),               # all in the second round's only one
    (3000, 4, 4, 128, spread(3000, 40, 1500, 20000), "mapped", False, True),
    (17000, 1, 1, 16, spread(17000, 60, 8000, 3000), "mapped", False, True),      # more than workgroups join
    (100, 8, 8, 128, spread(100, 700, 9, 3000), "mapped", False, True),
    (200, 16, 8, 64, spread(200, 300, 50, 5000), "mapped", False, True),
    (65, 8, 8, 128, spread(65, 200, 30, 500), "mapped", False, False),
    (40, 8, 8, 128, spread(40, 900, 11, 1500), "scanned", False, False),
    (40, 8, 8, 128, spread(40, 900, 11, 12000), "scanned", False, True),
    (64, 4, 4, 64, spread(64, 500, 60, 30000), "scanned", True, True),
    (64, 32, 8, 96, spread(64, 2000, 20, 9000), "scanned", False, True),
    (30, 8, 8, 128, spread(30, 900, 11, 3000), "scanned", True, True),
    (3, 2, 1, 64, [300000, 0, 5000], "scanned", True, True),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,H,Hk,D,lengths,cut,fit,longer", PLANS)
def test_every_way_of_cutting(dt, B, H, Hk, D, lengths, cut, fit, longer):
    import ctypes

    from gaussian_splat_encoder import _lib
    page = 64
    width = -(-max(lengths) // page)
    got = plan(B, H, Hk, D, 1, lengths, page, width)
    assert got[:2] == (cut, fit) and (got[4] > 1) == longer
    pages = 97
    g = torch.Generator("cuda").manual_seed(B)
    k, v = (torch.randn(pages, Hk, page, D, generator=g, device="cuda").to(dt).transpose(1, 2) for _ in range(2))
    c = F.PagedCache(k, v)
    tables = torch.randint(0, pages, (B, width), generator=g, device="cuda", dtype=torch.int32)   # pages are only read
    n = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    q = rand(B, 1, H, D, dt=dt, seed=1, scale=1.3)
    d, keep = c._describe(tables, n, None, B, 1)
    assert _lib.load().splat_cached_attention_workspace_bytes(ctypes.byref(d), H, 1) == workspace(cut, got[2], B, H, Hk, D, 1)
    o = F.cached_attention(q, c, tables, n)
    want = attention(q, c, tables, n)
    assert rel(o, want) <= R.bound_of(dt)
    bad = (o.double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1).clamp_min(1e-30)
    full = n > 0                             # each sequence by itself: a lost piece of one does not show among thousands
    assert bool((bad[full] <= R.bound_of(dt)).all()) and not bool(o[~full].any())
    assert torch.equal(F.cached_attention(q, c, tables, n), o)


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("H,Hk,D,n", [(4, 4, 64, 300), (8, 2, 128, 129), (32, 1, 96, 61)])
def test_bfloat16_attention_rounds_its_result_alone(H, Hk, D, n, turned):
    """Probabilities and turned queries are sums of two bfloat16 values, 2^-17 of them off: the result is as far from float64 as
    the exact one rounded, within 5%. (One value for the two: 15% to 82% more, test_token_edges.)"""
    B, page = 12, 32
    width = -(-n // page)
    c = F.PagedCache(rand(B * width, page, Hk, D, dt=torch.bfloat16, seed=1, scale=1.3),
                     rand(B * width, page, Hk, D, dt=torch.bfloat16, seed=2))
    tables, lengths = c.tables(B), torch.full((B,), n, device="cuda")
    q = rand(B, 1, H, D, dt=torch.bfloat16, seed=3, scale=1.3)
    ax, pos = (F.RotaryAxes((D,)), torch.full((B, 1, 1), 12345, device="cuda")) if turned else (None, None)
    o = F.cached_attention(q, c, tables, lengths, positions=pos, axes=ax)
    qd = R.rotary(q.double(), pos.double(), ax) if turned else q.double()
    want = R.attention(qd, c.k, c.v, None, tables, lengths, None, True, D ** -0.5)
    assert rel(o, want) <= 1.05 * rel(want.to(torch.bfloat16), want)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_reader_gradients_of_key_and_value_biases(kind):
    """The values' half of to_kv's bias has the bound of the reader's other parameters. The keys' half is a sum over all states
    that mostly cancels (a bias moves all scores nearly alike): the same bound, of the terms' magnitudes."""
    from test_gpu_token_reader import make, plain, where
    r = make(kind=kind)
    B, L, N = 2, 9, 150
    x, s, pos, spos = rand(B, L, 96, seed=1), rand(B, N, 56, seed=2), where(B, L, 4, 5), where(B, N, 2, 6)
    mask = rand(B, N, seed=7) < 0.8
    y = r(x, pos, s, spos, key_mask=mask)
    g = rand(*y.shape, seed=8)
    got, = torch.autograd.grad(y, r.to_kv.bias, g)
    p = {n: t.detach().double() for n, t in r.named_parameters()}
    each = p["to_kv.bias"].expand(B, N, -1).clone().requires_grad_(True)          # a bias of each state's own
    p["to_kv.bias"] = each
    z = plain(r, p, x.double(), pos.double(), s.double(), spos.double(), mask)
    d, = torch.autograd.grad(z, each, g.double())
    half, bound = r.kv_heads * r.head_dim, 18 * R.bound_of(torch.float32)
    want = d.sum((0, 1))
    assert rel(got[half:], want[half:]) <= bound
    assert (got[:half] - want[:half]).norm().item() <= bound * d[..., :half].abs().sum((0, 1)).norm().item()


def test_the_documented_example_runs():
    """The lines on tokens in the readme, with what its reader has: eight sequences of one new token in bfloat16, a frame's
    latents as the encoder gives them (float32)."""
    import os
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")
    with open(at) as f:
        blocks = [b.split("```")[0] for b in f.read().split("```python\n")[1:]]
    code, = [b for b in blocks if "cached_attention" in b]
    env = dict(torch=torch, q=rand(8, 1, 8, 64, dt=torch.bfloat16), k=rand(8, 1, 4, 64, dt=torch.bfloat16, seed=1),
               v=rand(8, 1, 4, 64, dt=torch.bfloat16, seed=2), positions=rand(8, 1, 3, seed=3), p=rand(8, 1, 3, seed=3),
               x=rand(4, 100, 256), h=rand(4, 100, 256, seed=4), g=rand(256, seed=5), w1=rand(256, seed=6), w2=rand(256, seed=7),
               latents=rand(1, 500, 128, seed=8), splat_positions=rand(1, 500, 3, seed=9), tokens=rand(1, 5, 256, seed=10),
               token_positions=rand(5, 3, seed=11))
    before = env["tokens"]
    exec(compile(code, at, "exec"), env)
    assert torch.equal(env["o"].view(8, 4, 2, 64), env["v"][:, 0, :, None].expand(8, 4, 2, 64))    # one token: its value
    assert torch.equal(env["tokens"], before)                       # a new layer's gates are closed
