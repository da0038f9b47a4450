"""The token operators on the GPU against plain float64 implementations: types, ragged sizes, strides, masks and tables that leave
rows empty, NaN in what is left out, gradients against the formulas' and against differences, repeatability, graphs, streams."""

import math

import pytest
import torch

import _token_ref as R
from _feature_ref import rel
from gaussian_splat_encoder import token_ops as F

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def rand(*shape, dt=torch.float32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dt)


def randint(lo, hi, shape, seed=0, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def close(a, b, what=""):
    """The 2-norm of a's error within its type's bound."""
    e = rel(a, b)
    assert e <= R.bound_of(a.dtype), (what, e)


# ------------------------------------------------------------------------------------------------ rotary
def places(kind, B, L, A, seed=5):
    if kind == "float32":
        return rand(B, L, A, seed=seed, scale=3.0)
    if kind == "shared":
        return randint(0, 500, (L, A), seed)
    if kind == "shared float32":
        return rand(1, L, A, seed=seed, scale=3.0)
    return randint(-1000, 100000, (B, L, A), seed, getattr(torch, kind))


# heads of whole chunks, of half ones, odd; axes that fill the head or a part of it, with halves of 8, 4, 2 and 1 pairs; heads
# side by side up to a workgroup's threads and beyond
ROTARY = [(1, 1, 1, 2, (2,)), (2, 3, 4, 64, (64,)), (2, 37, 3, 64, (32, 32)), (1, 65, 2, 40, (20, 16)), (3, 5, 5, 33, (10, 6)),
          (1, 300, 1, 128, (64, 32, 32)), (2, 9, 40, 128, (126,)), (1, 7, 300, 16, (4, 4, 4, 4)), (2, 130, 6, 96, (16, 24, 24)),
          (1, 2500, 2, 8, (4, 2))]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["float32", "int32", "int64", "shared", "shared float32"])
@pytest.mark.parametrize("B,L,H,D,dims", ROTARY)
def test_rotary(dt, kind, B, L, H, D, dims):
    for inter in (False, True):
        ax = F.RotaryAxes(dims, base=500.0, scale=tuple(0.5 + i for i in range(len(dims))), interleaved=inter)
        x = rand(B, L, H, D, dt=dt).requires_grad_(True)
        p = places(kind, B, L, len(dims))
        real = "float32" in kind
        p.requires_grad_(real)
        y = F.rotary(x, p, ax)
        xd, pd = x.detach().double().requires_grad_(True), p.detach().double().requires_grad_(real)
        yd = R.rotary(xd, pd, ax)
        g = rand(B, L, H, D, dt=dt, seed=9)
        a = torch.autograd.grad(y, [x, p] if real else [x], g)
        d = torch.autograd.grad(yd, [xd, pd] if real else [xd], g.double())
        assert y.dtype is dt and y.shape == x.shape and a[0].dtype is dt
        close(y, yd, "y")
        close(a[0], d[0], "dx")
        if real:
            # sums of terms f g y that may cancel: 64 units of the terms' own magnitude, |g| and |y| of a pair at most their
            # 2-norms, times the rates of the axis
            assert a[1].dtype is torch.float32 and a[1].shape == p.shape
            mag = (g.double().norm(dim=-1) * x.detach().double().norm(dim=-1)).sum(-1)      # [B, L]
            mag = mag.sum(0, keepdim=True) if p.shape[0] == 1 else mag
            top = torch.tensor([abs(s) for s in ax.scale], dtype=torch.float64, device="cuda")
            assert bool(((a[1] - d[1]).abs() <= 64 * 2.0 ** -24 * mag[..., None] * top).all())
        with torch.no_grad():
            assert torch.equal(F.rotary(x, p, ax), y)


def test_rotary_far_positions():
    """Angles of positions up to 2^31: the product of a position and a rate is rounded to 53 bits here and in the reference,
    2^31 * 2^-53 = 2.4e-7 radians each; sines and cosines add 1e-7."""
    p = torch.tensor([[2 ** 31 - 1, -2 ** 31, 2 ** 30 + 7, 16777217, -16777219]], device="cuda", dtype=torch.int64).T.contiguous()
    ax = F.RotaryAxes((128,))
    x = rand(1, 5, 3, 128)
    err = (F.rotary(x, p, ax).double() - R.rotary(x.double(), p.double(), ax)).abs().max().item()
    assert err <= (2 * 2.4e-7 + 2e-7) * x.abs().max().item() * math.sqrt(2)
    assert torch.equal(F.rotary(x, p.clamp(-2 ** 31, 2 ** 31 - 1).int(), ax), F.rotary(x, p, ax))


def test_rotary_of_every_quarter():
    """Angles around multiples of a quarter turn, where the reduction changes over: sines and cosines to 1.5e-7."""
    q = torch.arange(-9, 10, device="cuda", dtype=torch.float64) * (math.pi / 4)
    p = (q[:, None] + torch.linspace(-1e-3, 1e-3, 21, device="cuda", dtype=torch.float64)).reshape(-1, 1).float()
    x = torch.tensor([1.0, 0.0], device="cuda").expand(1, p.shape[0], 1, 2)
    y = F.rotary(x, p, F.RotaryAxes((2,)))[0, :, 0].double()
    w = p.double()[:, 0]
    assert (y - torch.stack([torch.cos(w), torch.sin(w)], -1)).abs().max().item() <= 1.5e-7


@pytest.mark.parametrize("dt", TYPES)
def test_rotary_strides(dt):
    ax = F.RotaryAxes((16, 8))
    big = rand(2, 11, 3, 4, 32, dt=dt)
    pos = rand(2, 11, 5, seed=1)
    want = F.rotary(big[:, :, 1].contiguous(), pos[..., 1:4:2].contiguous(), ax)
    assert torch.equal(F.rotary(big[:, :, 1], pos[..., 1:4:2], ax), want)
    t = big[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2)            # heads first
    assert torch.equal(F.rotary(t, pos[..., 1:4:2], ax), want)
    odd = rand(2, 11, 4, 33, dt=dt)[..., 1:]                                 # rows that start at any element
    assert torch.equal(F.rotary(odd, pos[..., :2], ax), F.rotary(odd.contiguous(), pos[..., :2].contiguous(), ax))
    last = rand(2, 11, 32, 4, dt=dt).transpose(2, 3)                         # no dense heads: copied
    assert torch.equal(F.rotary(last, pos[..., :2], ax), F.rotary(last.contiguous(), pos[..., :2], ax))
    x = big[:, :, 0].detach().requires_grad_(True)
    one, = torch.autograd.grad(F.rotary(x, pos[..., :2], ax).sum(), x)       # an expanded gradient
    two, = torch.autograd.grad(F.rotary(x, pos[..., :2], ax), x, torch.ones_like(x))
    assert torch.equal(one, two)
    p = pos[..., :2].detach().requires_grad_(True)
    one, = torch.autograd.grad(F.rotary(t, p, ax).sum(), p)
    two, = torch.autograd.grad(F.rotary(t.contiguous(), p, ax), p, torch.ones_like(t))
    assert torch.equal(one, two)


@pytest.mark.parametrize("shape", [(0, 4, 2, 8), (2, 0, 2, 8)])
def test_rotary_empty(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    p = torch.zeros(shape[1], 1, device="cuda", requires_grad=True)
    y = F.rotary(x, p, F.RotaryAxes((4,)))
    gx, gp = torch.autograd.grad(y.sum(), [x, p])
    assert y.shape == shape and gx.shape == shape and torch.equal(gp, torch.zeros_like(p))


def test_rotary_gradients_against_differences():
    """d/dt of <g, rotary(x + t u, p + t w)> by central differences in float64 of float32 results. Two roundings of 2^-24 over
    2 t = 2e-3 leave 6e-5 g y a term, of random sign: four times the root of n such terms of size 1 (third derivatives, of
    rates of 1 at most, leave t^2 / 6 = 2e-7 a term)."""
    ax = F.RotaryAxes((12, 8), base=50.0)
    x, p, u, w, g = rand(2, 9, 3, 24), rand(2, 9, 2, seed=1), rand(2, 9, 3, 24, seed=2), rand(2, 9, 2, seed=3), \
        rand(2, 9, 3, 24, seed=4)
    f = lambda t: (F.rotary(x + t * u, p + t * w, ax).double() * g.double()).sum().item()   # noqa: E731
    num = (f(1e-3) - f(-1e-3)) / 2e-3
    x.requires_grad_(True), p.requires_grad_(True)
    gx, gp = torch.autograd.grad(F.rotary(x, p, ax), [x, p], g)
    ana = ((gx.double() * u).sum() + (gp.double() * w).sum()).item()
    assert abs(num - ana) <= 4 * 6e-5 * math.sqrt(x.numel())


def test_second_derivatives_are_refused():
    x = rand(1, 2, 1, 4).requires_grad_(True)
    g, = torch.autograd.grad(F.rotary(x, rand(2, 1), F.RotaryAxes((4,))).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            F.token_norm(torch.autograd.forward_ad.make_dual(rand(2, 4), rand(2, 4)))


# ------------------------------------------------------------------------------------------------ the cache
def make_cache(pages, page, Hk, D, dt, masked=False, seed=3, layout="heads"):
    k, v = rand(pages, Hk, page, D, dt=dt, seed=seed, scale=1.3), rand(pages, Hk, page, D, dt=dt, seed=seed + 1)
    if layout == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    else:                                   # token by token, keys and values in one tensor, a gap between pages
        both = torch.zeros(pages, page + 1, 2, Hk, D, dtype=dt, device="cuda")
        both[:, :page, 0], both[:, :page, 1] = k.transpose(1, 2), v.transpose(1, 2)
        k, v = both[:, :page, 0], both[:, :page, 1]
    live = torch.rand(pages, page, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") < 0.6 if masked else None
    return F.PagedCache(k, v, live)


def make_tables(B, width, pages, seed=7):
    """Rows of different pages in no order (pages >= B width)."""
    ids = torch.randperm(pages, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")[:B * width]
    return ids.int().reshape(B, width)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("page,T,Hk,D,dims", [(1, 1, 1, 3, None), (16, 1, 4, 64, (64,)), (17, 5, 2, 40, (20, 16)),
                                              (7, 30, 3, 33, (32,)), (64, 200, 8, 128, (32, 48, 48)), (5, 3, 300, 8, (4,))])
def test_append(dt, masked, page, T, Hk, D, dims):
    B, width = 4, -(-260 // page) + 1
    for layout in ("heads", "tokens"):
        c = make_cache(B * width + 2, page, Hk, D, dt, masked, layout=layout)
        tables = make_tables(B, width, B * width + 2)
        lengths = torch.tensor([T, 0, 251, width * page + 3], device="cuda", dtype=torch.int32)   # none, and past the table
        counts = torch.tensor([T, T, (T + 1) // 2, T], device="cuda", dtype=torch.int32)
        k, v = rand(B, T, 2, Hk, D, dt=dt, seed=11).unbind(2)
        mask = (rand(B, T, seed=12) < 0.3) if masked else None
        ax = None if dims is None else F.RotaryAxes(dims, interleaved=layout == "tokens")
        p = None if dims is None else randint(0, 3000, (B, T, len(dims)), 13)
        stored = k if dims is None else F.rotary(k, p, ax)
        for n in (None, counts):
            want = R.append(c.k, c.v, c.live, tables, lengths, stored, v, n, mask)
            F.cache_append(c, tables, lengths, k, v, counts=n, positions=p, axes=ax, key_mask=mask)
            assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])
            assert c.live is None or torch.equal(c.live, want[2])


def test_append_without_a_mask_marks_tokens_live():
    c = F.PagedCache.empty(2, 4, 1, 8, dtype=torch.float32, masked=True)
    F.cache_append(c, c.tables(1), torch.tensor([3], device="cuda"), rand(1, 3, 1, 8), rand(1, 3, 1, 8))
    assert c.live.tolist() == [[True, True, True, False], [False] * 4]


def test_append_leaves_bad_places_alone():
    """Tables with entries that are no page, negative lengths and counts: nothing is written for them, and nothing else."""
    c = make_cache(6, 4, 2, 16, torch.float32)
    k0, v0 = c.k.clone(), c.v.clone()
    tables = torch.tensor([[-1, 2], [6, 1 << 30], [-2 ** 31, 3], [4, 5]], device="cuda", dtype=torch.int32)
    lengths = torch.tensor([6, 8, -5, 8], device="cuda", dtype=torch.int32)
    counts = torch.tensor([6, 8, 8, -3], device="cuda", dtype=torch.int32)
    k, v = rand(4, 8, 2, 16, seed=1), rand(4, 8, 2, 16, seed=2)
    F.cache_append(c, tables, lengths, k, v, counts=counts)
    k0[2, :2], v0[2, :2] = k[0, 4:6], v[0, 4:6]
    assert torch.equal(c.k, k0) and torch.equal(c.v, v0)


def check_attention(q, c, tables, lengths, counts=None, causal=True, scale=None, positions=None, axes=None):
    o = F.cached_attention(q, c, tables, lengths, counts=counts, causal=causal, scale=scale, positions=positions, axes=axes)
    qd = q.double() if axes is None else R.rotary(q.double(), positions.double(), axes)
    want = R.attention(qd, c.k, c.v, c.live, tables, lengths.clamp_min(0), counts, causal,
                       q.shape[-1] ** -0.5 if scale is None else scale)
    assert o.dtype is q.dtype and o.shape == q.shape and not bool(torch.isnan(o).any())
    close(o, want)
    empty = want.abs().amax(-1) == 0
    assert not bool(o[empty].any())
    assert torch.equal(F.cached_attention(q, c, tables, lengths, counts=counts, causal=causal, scale=scale,
                                          positions=positions, axes=axes), o)
    return o


# tiles of 16 and 32 tokens, pieces of 128, pages inside and across them, one token, none
LENGTHS = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 255, 257, 700]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("page,H,Hk,D,T", [(16, 4, 4, 64, 1), (1, 2, 1, 16, 3), (7, 6, 2, 40, 5), (64, 8, 1, 128, 2),
                                           (100, 3, 3, 33, 1), (17, 5, 1, 96, 7), (32, 2, 2, 80, 20), (24, 40, 1, 1, 1),
                                           (48, 4, 2, 127, 33), (16, 8, 1, 128, 5), (16, 8, 1, 96, 5), (16, 8, 1, 64, 5),
                                           (16, 8, 1, 32, 5), (16, 8, 1, 24, 5), (16, 8, 1, 56, 3), (16, 8, 1, 112, 3),
                                           (32, 2, 1, 24, 1), (32, 2, 1, 112, 1), (32, 2, 1, 32, 1), (32, 2, 1, 3, 9)])
def test_attention(dt, causal, page, H, Hk, D, T):
    B, width = len(LENGTHS), -(-700 // page)
    for layout, masked in (("heads", False), ("tokens", True)):
        c = make_cache(B * width + 1, page, Hk, D, dt, masked, layout=layout)
        tables = make_tables(B, width, B * width + 1)
        q = rand(B, T, H, D, dt=dt, seed=21, scale=1.3)
        lengths = torch.tensor(LENGTHS, device="cuda", dtype=torch.int32)
        check_attention(q, c, tables, lengths, causal=causal)
        counts = torch.tensor([min(n, T, 1 + i % 4) for i, n in enumerate(LENGTHS)], device="cuda", dtype=torch.int64)
        o = check_attention(q, c, tables, lengths.long(), counts=counts, causal=causal, scale=-0.3)
        for b in range(B):
            assert not bool(o[b, int(counts[b]):].any())      # rows past a sequence's new tokens


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,dims", [(64, (64,)), (40, (20, 16)), (33, (2, 4, 6)), (128, (128,))])
def test_attention_turns_queries(dt, inter, D, dims):
    B, T = 3, 4
    c = make_cache(40, 16, 2, D, dt)
    ax = F.RotaryAxes(dims, base=30.0, interleaved=inter)
    pos = rand(B, T, len(dims), seed=2, scale=20.0)
    check_attention(rand(B, T, 6, D, dt=dt, seed=1), c, make_tables(B, 10, 40), torch.tensor([150, 9, 77], device="cuda"),
                    positions=pos, axes=ax)
    check_attention(rand(B, T, 6, D, dt=dt, seed=1), c, make_tables(B, 10, 40), torch.tensor([150, 9, 77], device="cuda"),
                    positions=pos[0], axes=ax, causal=False)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,n,T,H,Hk", [(1, 50000, 1, 4, 4), (1, 30011, 9, 8, 2), (5, 20000, 1, 16, 4), (150, 800, 1, 2, 1),
                                        (70, 3000, 2, 4, 1)])
def test_attention_of_long_and_many_sequences(dt, B, n, T, H, Hk):
    """Sequences cut into pieces and joined, most of a batch's work in few of them."""
    page, D = 64, 64
    width = -(-n // page)
    c = make_cache(max(8, B * width // 16), page, Hk, D, dt)
    tables = randint(0, c.pages, (B, width), 3)              # pages may be shared where they are only read
    lengths = torch.tensor([n if i % (7 if B < 1000 else 301) == 0 else (i * 37) % (n // 3) if B < 1000 else i % 140
                            for i in range(B)], device="cuda")
    check_attention(rand(B, T, H, D, dt=dt, seed=1, scale=1.5), c, tables, lengths)


@pytest.mark.parametrize("dt", TYPES)
def test_what_is_left_out_has_no_effect(dt):
    """NaN and infinities in dead tokens, behind the lengths, on pages no table names and (causal) in tokens after a query."""
    B, T, H, Hk, D, page, width = 3, 6, 4, 2, 64, 16, 20
    for bad in (math.nan, math.inf, -math.inf):
        c = make_cache(B * width + 4, page, Hk, D, dt, masked=True)
        tables = make_tables(B, width, B * width + 4)
        tables[1, 3], tables[2, 0] = -1, 5000
        lengths = torch.tensor([310, 139, 33], device="cuda")
        q = rand(B, T, H, D, dt=dt, seed=1)
        want = check_attention(q, c, tables, lengths)
        c.live[tables[0, 19], 0:6] = True       # the new tokens of the first sequence count
        want = check_attention(q, c, tables, lengths)
        k, v = c.k.clone(), c.v.clone()
        used = torch.zeros(c.pages, page, dtype=torch.bool, device="cuda")
        for b in range(B):
            j = torch.arange(int(lengths[b]), device="cuda")
            p = tables[b].long()[j // page]
            ok = (p >= 0) & (p < c.pages)
            used[p[ok], (j % page)[ok]] = True
        c.k[~(used & c.live)] = bad
        c.v[~(used & c.live)] = bad
        assert torch.equal(F.cached_attention(q, c, tables, lengths), want)
        # tokens after query 1 of the first sequence: queries 0 and 1 do not see them
        at = [(int(tables[0, (306 + i) // page]), (306 + i) % page) for i in range(4)]
        for p, o in at:
            c.k[p, o], c.v[p, o] = bad, bad
        o = F.cached_attention(q, c, tables, lengths)
        assert rel(o[0, :2], want[0, :2]) <= 2.0 ** -20 and torch.equal(o[1:], want[1:])
        assert bool(torch.isnan(o[0, 2:]).any())
        c.k.copy_(k), c.v.copy_(v)


@pytest.mark.parametrize("dt", TYPES)
def test_lengths_past_the_table(dt):
    """A query's place goes by its sequence's length, also where the table has no room for all of it."""
    c = make_cache(20, 16, 2, 64, dt)
    tables = make_tables(4, 5, 20)
    lengths = torch.tensor([80, 83, 90, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    check_attention(rand(4, 9, 4, 64, dt=dt, seed=1), c, tables, lengths)
    check_attention(rand(4, 9, 4, 64, dt=dt, seed=1), c, tables, lengths, counts=torch.tensor([9, 5, 9, 2], device="cuda"))


def test_attention_of_nothing():
    c = F.PagedCache.empty(4, 8, 2, 16)
    q = rand(3, 2, 4, 16, dt=torch.bfloat16)
    zero = torch.zeros_like(q)
    no = torch.zeros(3, dtype=torch.int32, device="cuda")
    for tables in (c.tables(3), torch.zeros(3, 0, dtype=torch.int32, device="cuda")):
        assert torch.equal(F.cached_attention(q, c, tables, no), zero)
        assert torch.equal(F.cached_attention(q, c, tables, no - 7), zero)
    assert torch.equal(F.cached_attention(q, c, torch.zeros(3, 0, dtype=torch.int32, device="cuda"), no + 9), zero)
    assert F.cached_attention(q[:, :0], c, c.tables(3), no).shape == (3, 0, 4, 16)
    assert F.cached_attention(q[:0], c, c.tables(0), no[:0]).shape == (0, 2, 4, 16)
    nopages = F.PagedCache(c.k[:0], c.v[:0])
    assert torch.equal(F.cached_attention(q, nopages, c.tables(3), no + 5), zero)
    F.cache_append(nopages, c.tables(3), no + 5, q[:, :, :2], q[:, :, :2])


def test_attention_strides():
    c = make_cache(12, 16, 2, 32, torch.bfloat16)
    tables, lengths = make_tables(2, 6, 12), torch.tensor([90, 33], device="cuda")
    q = rand(2, 3, 3, 4, 33, dt=torch.bfloat16)[:, :, 1, :, 1:]
    want = F.cached_attention(q.contiguous(), c, tables, lengths)
    assert torch.equal(F.cached_attention(q, c, tables, lengths), want)
    assert torch.equal(F.cached_attention(q.transpose(1, 2).contiguous().transpose(1, 2), c, tables, lengths), want)
    assert torch.equal(F.cached_attention(q.transpose(2, 3).contiguous().transpose(2, 3), c, tables, lengths), want)
    wide = torch.full((2, 14), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2][:, :6] = tables
    assert torch.equal(F.cached_attention(q, c, wide[:, :12:2], lengths), want)


def test_offsets_past_32_bits():
    """Pages that lie past 2^32 elements of their tensor, and offsets within a page past 2^31."""
    n = (1 << 32) + (1 << 20)
    big = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    step = 1 << 31
    k = big.as_strided((3, 8, 2, 16), (step, 64, 16, 1), 0)
    v = big.as_strided((3, 8, 2, 16), (step, 64, 16, 1), 32)
    far = big.as_strided((2, 3, 2, 16), (64, step, 16, 1), 1 << 19)          # tokens 2^31 elements apart
    for c in (F.PagedCache(k, v), F.PagedCache(far, far.as_strided(far.shape, far.stride(), (1 << 19) + 32))):
        c.k.copy_(rand(*c.k.shape, dt=torch.bfloat16)), c.v.copy_(rand(*c.k.shape, dt=torch.bfloat16, seed=1))
        tables = torch.arange(c.pages, device="cuda", dtype=torch.int32).flip(0)[None].contiguous()
        lengths = torch.tensor([c.pages * c.page], device="cuda")
        check_attention(rand(1, 2, 4, 16, dt=torch.bfloat16, seed=2), c, tables, lengths)
        x = rand(1, 3, 2, 16, dt=torch.bfloat16, seed=4)
        want = R.append(c.k, c.v, None, tables, lengths, x, x, None, None)
        F.cache_append(c, tables, lengths, x, x)
        assert torch.equal(c.k, want[0]) and torch.equal(c.v, want[1])


def test_a_captured_step_follows_its_lengths():
    """Append and attention in one graph, replayed as the sequences grow past a piece and a page, against eager calls; two graphs
    with workspaces of their own in turn."""
    B, Hk, D, page, width = 3, 2, 64, 16, 64
    ax = F.RotaryAxes((64,))
    tables = make_tables(B, width, B * width)
    steps = [(rand(B, 1, 4, D, dt=torch.bfloat16, seed=s), rand(B, 1, Hk, D, dt=torch.bfloat16, seed=s + 50),
              rand(B, 1, Hk, D, dt=torch.bfloat16, seed=s + 90)) for s in range(6)]
    start = torch.tensor([0, 127, 900], device="cuda", dtype=torch.int32)

    def step(c, lengths, q, k, v):
        lengths.add_(1)
        pos = (lengths - 1)[:, None, None]
        F.cache_append(c, tables, lengths, k, v, positions=pos, axes=ax)
        return F.cached_attention(q, c, tables, lengths, positions=pos, axes=ax)

    def eager():
        c, n = make_cache(B * width, page, Hk, D, torch.bfloat16), start.clone()
        return [step(c, n, *s).clone() for s in steps], c, n

    want, cw, nw = eager()
    graphs = []
    for _ in range(2):
        c, n = make_cache(B * width, page, Hk, D, torch.bfloat16), start.clone()
        args = [t.clone() for t in steps[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(c, n, *args)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(c, n, *args)
        fresh = make_cache(B * width, page, Hk, D, torch.bfloat16)
        c.k.copy_(fresh.k), c.v.copy_(fresh.v), n.copy_(start)
        graphs.append((g, c, n, args, out))
    for i, s in enumerate(steps):
        for g, c, n, args, out in graphs:
            for a, b in zip(args, s):
                a.copy_(b)
            g.replay()
        assert torch.equal(eager()[0][i], want[i])            # eager work between the replays
        torch.cuda.synchronize()
        for g, c, n, args, out in graphs:
            assert torch.equal(out, want[i])
    for g, c, n, args, out in graphs:
        assert torch.equal(c.k, cw.k) and torch.equal(c.v, cw.v) and torch.equal(n, nw)


def test_two_streams_at_once():
    c = make_cache(600, 64, 4, 64, torch.bfloat16)
    calls = [(rand(1, 1, 4, 64, dt=torch.bfloat16, seed=i), make_tables(1, 500, 600, seed=i),
              torch.tensor([31000 + i], device="cuda")) for i in range(4)]
    want = [F.cached_attention(q, c, t, n) for q, t, n in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for i, (s, (q, t, n)) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(F.cached_attention(q, c, t, n))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(g, w) for g in gs)


# ------------------------------------------------------------------------------------------------ norms per token
def check_norm(shape, dt, kind="rms", gate=None, act="none", block=True, nxt=True, params="all", scale=0.7, eps=1e-6, use=(0, 1)):
    C = shape[-1]
    x, h = rand(*shape, dt=dt, seed=1, scale=2.0, shift=0.3), rand(*shape, dt=dt, seed=2, shift=-0.2)
    par = [rand(C, seed=3 + i, scale=0.3, shift=float(i % 2 == 0)) for i in range(4)]
    if params == "none":
        par = [None] * 4
    elif params == "weights":
        par[1] = par[3] = None
    if not block:
        par[:2] = [None, None]
    if not nxt:
        par[2:] = [None, None]
    gt = None
    if gate is not None:
        gt = rand(*gate, dt=dt if tuple(gate) == tuple(shape) else torch.float32, seed=8, shift=0.2)
    own = [x, h, par[0], par[1], gt, par[2], par[3]]
    a = [None if t is None else t.detach().requires_grad_(True) for t in own]
    d = [None if t is None else t.detach().double().requires_grad_(True) for t in own]
    ys = F.residual_norm(a[0], a[1], a[2], a[3], gate=a[4], gate_act=act, next_weight=a[5], next_bias=a[6], kind=kind, eps=eps,
                         scale=scale, norm_block=block, norm_next=nxt)
    ys = ys if isinstance(ys, tuple) else (ys,)
    zs = R.residual_norm(d[0], d[1], d[2], d[3], d[4], act, d[5], d[6], kind, eps, scale, block, nxt)
    assert len(ys) == len(zs)
    for y, z in zip(ys, zs):
        assert y.dtype is dt and y.shape == torch.Size(shape)
        close(y, z, "output")
    use = [i for i in use if i < len(ys)]
    up = [rand(*shape, dt=dt, seed=20 + i) for i in use]
    ins = [i for i, t in enumerate(a) if t is not None]
    ga = torch.autograd.grad([ys[i] for i in use], [a[i] for i in ins], up, allow_unused=True)
    gd = torch.autograd.grad([zs[i] for i in use], [d[i] for i in ins], [u.double() for u in up], allow_unused=True)
    for i, p, q in zip(ins, ga, gd):
        if q is None:
            assert p is None or not bool(p.any())
            continue
        assert p.dtype is own[i].dtype and p.shape == own[i].shape
        close(p, q, f"gradient {i}")
    with torch.no_grad():
        again = F.residual_norm(a[0], a[1], a[2], a[3], gate=a[4], gate_act=act, next_weight=a[5], next_bias=a[6], kind=kind,
                                eps=eps, scale=scale, norm_block=block, norm_next=nxt)
    again = again if isinstance(again, tuple) else (again,)
    assert all(torch.equal(y, z) for y, z in zip(ys, again))
    return ga


# rows of one to eight lanes' chunks, of one wave, of four and of sixteen, each with one and two chunks a lane, odd widths
WIDTHS = [4, 8, 31, 64, 100, 200, 256, 333, 512, 517, 1000, 1024, 1500, 2048, 3000, 4096, 5001, 8192]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("C", WIDTHS)
def test_residual_norm_widths(dt, kind, C):
    check_norm((2, 37, C), dt, kind, gate=(C,))
    check_norm((3, 5, C), dt, kind, gate=(3, 5, C), act="sigmoid")
    check_norm((2, 37, C), dt, kind, gate=(2, C), act="silu", params="weights")
    check_norm((1, 9, C), dt, kind, gate=(1, 9, C), act="tanh", params="none")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu", "tanh"])
@pytest.mark.parametrize("gate", ["channel", "image", "rows", "token", None])
def test_residual_norm_gates(dt, act, gate):
    B, h, w, C = 5, 6, 7, 72
    shape = {"channel": (C,), "image": (B, C), "rows": (B, 1, 1, C), "token": (B, h, w, C), None: None}[gate]
    check_norm((B, h, w, C), dt, gate=shape, act=act)
    check_norm((B, h, w, C), dt, "layer", gate=shape, act=act, block=False, params="weights")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("block,nxt", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("params", ["all", "weights", "none"])
def test_residual_norm_parts(dt, block, nxt, params):
    for use in ((0, 1), (0,), (1,)):
        if use == (1,) and not nxt:
            continue
        check_norm((3, 50, 96), dt, "layer", gate=(96,), block=block, nxt=nxt, params=params, use=use)
        check_norm((3, 50, 96), dt, "rms", gate=(3, 1, 96), act="tanh", block=block, nxt=nxt, params=params, use=use, scale=-1.5)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,gate", [((1, 1, 8), (8,)), ((3000, 1, 16), (3000, 1, 16)), ((3000, 2, 16), (3000, 1, 16)),
                                        ((1001, 3, 264), (1001, 264)), ((20000, 24), (24,)), ((2, 9001, 256), (2, 1, 256)),
                                        ((900, 300, 4), (900, 4)), ((64,), (64,)), ((7, 40), (7, 40))])
def test_residual_norm_rows(dt, shape, gate):
    """One token, images of a token or two (many gates), long images, whole and split ranges."""
    check_norm(shape, dt, "layer", gate=gate, act="sigmoid")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("shape", [(1, 5), (40, 33), (3, 100, 256), (2, 3, 5, 1000), (10000, 64), (3, 8192)])
def test_token_norm(dt, kind, shape):
    C = shape[-1]
    x, w, b = rand(*shape, dt=dt, shift=0.5), rand(C, seed=1, shift=1.0, scale=0.2), rand(C, seed=2)
    for p in ([w, b], [w, None], [None, None]):
        a = [None if t is None else t.detach().requires_grad_(True) for t in [x, *p]]
        d = [None if t is None else t.detach().double().requires_grad_(True) for t in [x, *p]]
        y, z = F.token_norm(*a, kind=kind, eps=1e-3), R.norm(*d, kind, 1e-3)
        close(y, z)
        g = rand(*shape, dt=dt, seed=5)
        i = [k for k, t in enumerate(a) if t is not None]
        for p_, q_ in zip(torch.autograd.grad(y, [a[k] for k in i], g), torch.autograd.grad(z, [d[k] for k in i], g.double())):
            close(p_, q_)


def test_token_norm_is_the_layer_norm_of_each_token():
    from gaussian_splat_encoder import feature_ops
    x = rand(50, 96)
    assert rel(F.token_norm(x, kind="layer", eps=1e-5), feature_ops.group_norm_act(x, 1, act="none")) <= 2.0 ** -20


def test_far_means_do_not_cancel():
    """A mean a thousand deviations from zero: the row's own rounding of 2^-24 of the mean, and a few units of it in the sums."""
    x = rand(64, 700, shift=1000.0)
    y = F.token_norm(x, kind="layer", eps=0.0)
    assert (y.double() - R.norm(x.double(), None, None, "layer", 0.0)).abs().max().item() < 1000 * 8 * 2.0 ** -24


@pytest.mark.parametrize("dt", TYPES)
def test_norm_strides(dt):
    big, hid = rand(3, 20, 3, 80, dt=dt), rand(3, 20, 81, dt=dt, seed=1)
    x, h = big[:, :, 1], hid[..., 1:]
    w, g = rand(80, seed=2), rand(3, 20, 2, 80, dt=dt, seed=3)[:, :, 0]
    want = F.residual_norm(x.contiguous(), h.contiguous(), w, gate=g.contiguous(), gate_act="tanh")
    got = F.residual_norm(x, h, w, gate=g, gate_act="tanh")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    col = rand(3, 80, 20, dt=dt).transpose(1, 2)
    assert torch.equal(F.token_norm(col), F.token_norm(col.contiguous()))
    wide = rand(80, 2, seed=4)[:, 0]
    assert torch.equal(F.token_norm(x, wide), F.token_norm(x, wide.contiguous()))
    a, b = x.detach().requires_grad_(True), h.detach().requires_grad_(True)
    one = torch.autograd.grad([t.sum() for t in F.residual_norm(a, b, w)], [a, b])             # expanded gradients
    two = torch.autograd.grad(F.residual_norm(a, b, w), [a, b], [torch.ones_like(x)] * 2)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    # h is x itself, and a row used for all tokens
    c = x.detach().requires_grad_(True)
    s, = torch.autograd.grad(sum(t.float().square().sum() for t in F.residual_norm(c, c)), c)
    cd = c.detach().double().requires_grad_(True)
    t, = torch.autograd.grad(sum(t.square().sum() for t in R.residual_norm(cd, cd, None, None, None, "none", None, None, "rms",
                                                                             1e-6, 1.0, True, True)), cd)
    # two roundings of the upstream gradients 2 y and 2 n, and of the two parts of the sum before and after it
    assert rel(s, t) <= R.bound_of(dt) * (4 if dt is torch.bfloat16 else 1)
    one = rand(1, 1, 80, dt=dt).expand(3, 20, 80).detach()
    assert torch.equal(F.residual_norm(x, one)[0], F.residual_norm(x, one.contiguous())[0])


def test_norm_empty():
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w, g = torch.ones(8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
        y, n = F.residual_norm(x, x, w, gate=g, next_weight=w)
        gx, gw, gg = torch.autograd.grad((y + n).sum(), [x, w, g])
        assert y.shape == shape and gx.shape == shape and not bool(gw.any()) and not bool(gg.any())


def test_norm_of_zeros_and_bad_rows():
    """Zero rows give the bias; NaN and infinities stay in their row."""
    x, b = torch.zeros(9, 40, device="cuda"), rand(40)
    for kind in ("rms", "layer"):
        assert torch.equal(F.token_norm(x, None, b, kind=kind), b.expand(9, 40))
        y = x.clone().normal_()
        good = F.token_norm(y, kind=kind)
        y[4, 7], y[6, 0] = math.nan, math.inf
        got = F.token_norm(y, kind=kind)
        assert bool(torch.isnan(got[4]).all()) and bool(torch.isnan(got[6]).any())
        keep = [i for i in range(9) if i not in (4, 6)]
        assert torch.equal(got[keep], good[keep])


def test_norm_gradients_against_differences():
    """d/dt of <g, (y, n)> along a direction of every input by central differences of float32 results: two roundings of 2^-24 of
    values of up to 10 over 2 t = 4e-3 leave 3e-4 a term, of random sign; the third derivative's part, t^2 / 6 of it, is
    taken from the differences over 3 t (a second time over for the fifth)."""
    C, t = 48, 2e-3
    ins = [rand(6, C, seed=1), rand(6, C, seed=2)] + [rand(C, seed=3 + i, scale=0.3, shift=1.0) for i in range(4)] \
        + [rand(6, C, seed=9)]
    dirs = [rand(*v.shape, seed=30 + i) for i, v in enumerate(ins)]
    g = [rand(6, C, seed=50), rand(6, C, seed=51)]

    def run(v):
        return F.residual_norm(v[0], v[1], v[2], v[3], gate=v[6], gate_act="silu", next_weight=v[4], next_bias=v[5],
                               kind="layer")

    f = lambda s: sum((o.double() * u.double()).sum().item() for o, u in zip(run([v + s * d for v, d in zip(ins, dirs)]), g))  # noqa: E731
    num = (f(t) - f(-t)) / (2 * t)
    a = [v.detach().requires_grad_(True) for v in ins]
    ana = sum((p.double() * d.double()).sum().item() for p, d in zip(torch.autograd.grad(run(a), a, g), dirs))
    third = abs(f(3 * t) - 3 * f(t) + 3 * f(-t) - f(-3 * t)) / (8 * t ** 3) * t * t / 6
    assert abs(num - ana) <= 3e-4 * math.sqrt(2 * 6 * C) + 2 * third


def test_saved_tensors_may_come_back_dense():
    """A hook that stores what the backward needs elsewhere gives dense copies back for strided views."""
    big = rand(2, 30, 3, 4, 32)
    x, h, g = big[:, :, 0].flatten(2), big[:, :, 1].flatten(2), big[:, :, 2].flatten(2)
    v, pos = big.transpose(1, 3)[:, :, 0].transpose(1, 2), rand(2, 30, 5, seed=1)[..., 1:3]
    ax, up = F.RotaryAxes((16, 8)), rand(2, 30, 128, seed=2)

    def grads():
        a = [t.detach().requires_grad_(True) for t in (x, h, g, v, pos)]
        y, n = F.residual_norm(a[0], a[1], gate=a[2], gate_act="silu")
        r = F.rotary(a[3], a[4], ax)
        return torch.autograd.grad([y, n, r], a, [up, 2 * up, rand(*r.shape, seed=3)])

    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda().contiguous()):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_broadcast_inputs():
    """Expanded inputs: their gradients are summed over what they were expanded to."""
    one, row, up = rand(1, 1, 2, 16), rand(1, 1, 48, seed=1), rand(3, 7, 48, seed=2)
    pos, h = rand(3, 7, 1, seed=3), rand(3, 7, 48, seed=4)
    ax = F.RotaryAxes((16,))
    a, b, p = one.requires_grad_(True), row.requires_grad_(True), pos[:1, :1].detach().requires_grad_(True)
    r = F.rotary(a.expand(3, 7, 2, 16), p.expand(3, 7, 1), ax)
    y, n = F.residual_norm(b.expand(3, 7, 48), h)
    got = torch.autograd.grad([r, y, n], [a, b, p], [rand(3, 7, 2, 16, seed=5), up, up])
    d = [t.detach().double().requires_grad_(True) for t in (a, b, p)]
    rd = R.rotary(d[0].expand(3, 7, 2, 16), d[2].expand(3, 7, 1), ax)
    yd, nd = R.residual_norm(d[1].expand(3, 7, 48), h.double(), None, None, None, "none", None, None, "rms", 1e-6, 1.0, True,
                             True)
    want = torch.autograd.grad([rd, yd, nd], d, [rand(3, 7, 2, 16, seed=5).double(), up.double(), up.double()])
    for g, w in zip(got, want):
        close(g, w)


def test_rows_past_2_31_values():
    """Tensors of more than 2^31 values whose last rows are compared: their own values, and gradients."""
    n, C = 8_600_000, 256
    x = torch.empty(n, C, dtype=torch.bfloat16, device="cuda")
    x.view(-1, 1000 * C).copy_(rand(1000 * C, dt=torch.bfloat16))
    x[-3:] = rand(3, C, dt=torch.bfloat16, seed=1)
    w, gate = rand(C, seed=2, shift=1.0), rand(C, seed=3)
    y, m = F.residual_norm(x, x, w, gate=gate, next_weight=w)
    a, b = F.residual_norm(x[-3:], x[-3:], w, gate=gate, next_weight=w)
    assert torch.equal(y[-3:], a) and torch.equal(m[-3:], b)
    xs, = torch.autograd.grad(F.token_norm(x.requires_grad_(True), w), x, x.detach())
    part = x[-3:].detach().requires_grad_(True)
    assert torch.equal(xs[-3:], torch.autograd.grad(F.token_norm(part, w), part, part.detach())[0])
    del xs, y, m
    x = x.detach()
    pos = torch.arange(n, device="cuda", dtype=torch.int32)[:, None]
    ax = F.RotaryAxes((64,))
    r = F.rotary(x.view(1, n, 4, 64), pos, ax)
    assert torch.equal(r[0, -3:], F.rotary(x[-3:].view(1, 3, 4, 64), pos[-3:], ax)[0])


def test_a_captured_training_step():
    """Forward and backward in a graph, replayed over new values with eager work between, against the eager result."""
    x, h = rand(700, 128, dt=torch.bfloat16), rand(700, 128, dt=torch.bfloat16, seed=1)
    w, gate, pos = rand(128, seed=2, shift=1.0), rand(128, seed=3), rand(1, 700, 2, seed=4)
    ax = F.RotaryAxes((16, 16))

    def step(x, h, w, gate, pos):
        a = [t.detach().requires_grad_(True) for t in (x, h, w, gate, pos)]
        y, n = F.residual_norm(a[0], a[1], a[2], gate=a[3], gate_act="sigmoid", next_weight=a[2])
        r = F.rotary(n.view(1, 700, 4, 32), a[4], ax)
        return torch.autograd.grad([y, r], a, [torch.ones_like(y), torch.full_like(r, 0.5)])

    args = [x.clone(), h.clone(), w, gate, pos.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*args)
    for s in range(4):
        for t, seed in ((args[0], s), (args[1], s + 10), (args[4], s + 20)):
            t.copy_(rand(*t.shape, dt=t.dtype, seed=seed))
        g.replay()
        want = step(*[t.clone() for t in args])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
