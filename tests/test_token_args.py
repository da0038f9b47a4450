"""Host-side refusals of the token operators (CPU; no kernel runs), and the C entry points' own argument checks."""

import ctypes
import math

import pytest
import torch

from gaussian_splat_encoder import _lib
from gaussian_splat_encoder import token_ops as F


class Dev(torch.Tensor):
    """A host tensor that says it is on a device: the checks before any launch are what is tested."""
    is_cuda = True


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Dev)


def ints(*shape):
    return t(*shape, dtype=torch.int32)


def cache(pages=4, page=8, heads=2, D=16, dtype=torch.float32, masked=False):
    return F.PagedCache(t(pages, page, heads, D, dtype=dtype), t(pages, page, heads, D, dtype=dtype),
                        t(pages, page, dtype=torch.bool) if masked else None)


AX = F.RotaryAxes((8, 4))


def test_cpu_tensors_are_refused():
    z = torch.zeros
    for call in (lambda: F.rotary(z(1, 2, 1, 16), z(2, 2), AX), lambda: F.token_norm(z(2, 4)),
                 lambda: F.residual_norm(z(2, 4), z(2, 4)), lambda: F.PagedCache(z(2, 2, 1, 4), z(2, 2, 1, 4)),
                 lambda: F.cached_attention(z(1, 1, 2, 16), cache(), ints(1, 2), ints(1)),
                 lambda: F.cache_append(cache(), ints(1, 2), ints(1), z(1, 1, 2, 16), z(1, 1, 2, 16))):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()


@pytest.mark.parametrize("call,what", [
    (lambda: F.RotaryAxes(()), "axes are needed"),
    (lambda: F.RotaryAxes((2, 2, 2, 2, 2)), "axes are needed"),
    (lambda: F.RotaryAxes((3,)), "even"),
    (lambda: F.RotaryAxes((0, 4)), "even"),
    (lambda: F.RotaryAxes((64, 66)), "even"),
    (lambda: F.RotaryAxes((4, 4), base=(10.0,)), "base needs"),
    (lambda: F.RotaryAxes((4,), base=0.0), "positive"),
    (lambda: F.RotaryAxes((4,), scale=math.inf), "finite"),
    (lambda: F.RotaryAxes((4,), scale=math.nan), "finite"),
    (lambda: F.rotary(t(1, 2, 16), t(2, 2), AX), r"\[B, L, H, D\]"),
    (lambda: F.rotary(t(1, 2, 1, 160), t(2, 2), AX), "1 to 128"),
    (lambda: F.rotary(t(1, 2, 1, 8), t(2, 2), AX), "do not fit"),
    (lambda: F.rotary(t(1, 2, 1, 16), t(2, 3), AX), "positions must be"),
    (lambda: F.rotary(t(2, 2, 1, 16), t(3, 2, 2), AX), "positions must be"),
    (lambda: F.rotary(t(1, 2, 1, 16), t(2, 2, dtype=torch.float64), AX), "float32, int32 or int64"),
    (lambda: F.rotary(t(1, 2, 1, 16), None, AX), "axes need positions"),
    (lambda: F.rotary(t(1, 2, 1, 16), t(2, 2), (8, 4)), "RotaryAxes"),
    (lambda: F.rotary(t(1, 2, 1, 16, dtype=torch.float16), t(2, 2), AX), "float32 or bfloat16"),
    (lambda: F.PagedCache(t(4, 8, 2, 16), t(4, 8, 2, 8)), r"\[pages, page, Hk, D\]"),
    (lambda: F.PagedCache(t(4, 0, 2, 16), t(4, 0, 2, 16)), r"\[pages, page, Hk, D\]"),
    (lambda: F.PagedCache(t(4, 8, 2, 129), t(4, 8, 2, 129)), "1 to 128"),
    (lambda: F.PagedCache(t(4, 8, 16, 2).transpose(2, 3), t(4, 8, 2, 16)), "dense"),
    (lambda: F.PagedCache(t(4, 8, 2, 16), t(4, 8, 2, 16), t(4, 8)), "live must be"),
    (lambda: F.PagedCache(t(4, 8, 2, 16), t(4, 8, 2, 16), t(8, 4, dtype=torch.bool)), "live must be"),
    (lambda: F.PagedCache(t(4, 8, 2, 16), t(4, 8, 2, 16, dtype=torch.bfloat16)), "one type"),
    (lambda: F.PagedCache(t(4, 8, 2, 16).requires_grad_(True), t(4, 8, 2, 16)), "gradient"),
    (lambda: F.cache_append("cache", ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16)), "PagedCache"),
    (lambda: F.cache_append(cache(), ints(1, 2), ints(1), t(1, 1, 1, 16), t(1, 1, 1, 16)), "k and v must be"),
    (lambda: F.cache_append(cache(), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 2, 2, 16)), "k and v must be"),
    (lambda: F.cache_append(cache(), ints(2, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16)), "tables must be"),
    (lambda: F.cache_append(cache(), t(1, 2, dtype=torch.int64), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16)), "tables must be"),
    (lambda: F.cache_append(cache(), ints(1, 2), t(1), t(1, 1, 2, 16), t(1, 1, 2, 16)), "lengths must be"),
    (lambda: F.cache_append(cache(), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16), counts=ints(2)), "counts must be"),
    (lambda: F.cache_append(cache(), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16),
                            key_mask=t(1, 1, dtype=torch.bool)), "live"),
    (lambda: F.cache_append(cache(masked=True), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16), key_mask=t(1, 1)),
     "key_mask must be"),
    (lambda: F.cache_append(cache(), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16), axes=AX), "axes need positions"),
    (lambda: F.cache_append(cache(dtype=torch.bfloat16), ints(1, 2), ints(1), t(1, 1, 2, 16), t(1, 1, 2, 16)), "one type"),
    (lambda: F.cached_attention(t(1, 1, 3, 16), cache(), ints(1, 2), ints(1)), "q must be"),
    (lambda: F.cached_attention(t(1, 1, 2, 8), cache(), ints(1, 2), ints(1)), "q must be"),
    (lambda: F.cached_attention(t(1, 2, 16), cache(), ints(1, 2), ints(1)), "q must be"),
    (lambda: F.cached_attention(t(1, 1, 2, 16), cache(), ints(1, 2), ints(1), scale=math.inf), "scale"),
    (lambda: F.cached_attention(t(1, 1, 2, 16), cache(), ints(1, 2), ints(1), scale=math.nan), "scale"),
    (lambda: F.cached_attention(t(1, 1, 2, 16), cache(), ints(1, 2), ints(1), positions=t(1, 2), axes="xy"), "RotaryAxes"),
    (lambda: F.token_norm(t(2, 4), kind="batch"), "unknown norm"),
    (lambda: F.token_norm(t(2, 4), eps=-1.0), "eps"),
    (lambda: F.token_norm(t(2, 4), eps=math.nan), "eps"),
    (lambda: F.token_norm(t(2, 8193)), "1 to 8192"),
    (lambda: F.token_norm(t(2, 0)), "1 to 8192"),
    (lambda: F.token_norm(t(2, 4), t(3)), "weight must be"),
    (lambda: F.residual_norm(t(2, 4), t(2, 5)), "h must be"),
    (lambda: F.residual_norm(t(2, 4), t(2, 4, dtype=torch.bfloat16)), "one type"),
    (lambda: F.residual_norm(t(2, 4), t(2, 4), gate_act="gelu"), "unknown activation"),
    (lambda: F.residual_norm(t(2, 4), t(2, 4), scale=math.inf), "scale"),
    (lambda: F.residual_norm(t(2, 4), t(2, 4), t(4), norm_block=False), "weight and bias"),
    (lambda: F.residual_norm(t(2, 4), t(2, 4), next_bias=t(4), norm_next=False), "next_weight"),
    (lambda: F.residual_norm(t(2, 3, 4), t(2, 3, 4), gate=t(3, 4)), "gate must be"),
    (lambda: F.residual_norm(t(2, 3, 4), t(2, 3, 4), gate=t(2, 3, 1)), "gate must be"),
    (lambda: F.residual_norm(t(2, 3, 4, dtype=torch.bfloat16), t(2, 3, 4, dtype=torch.bfloat16), gate=t(2, 3, 4)),
     "gate for each token"),
])
def test_wrong_arguments_are_refused(call, what):
    with pytest.raises(ValueError, match=what):
        call()


def test_the_cache_has_no_gradients():
    k = t(1, 1, 2, 16).requires_grad_(True)
    with pytest.raises(NotImplementedError, match="inference"):
        F.cache_append(cache(), ints(1, 2), ints(1), k, t(1, 1, 2, 16))
    with pytest.raises(NotImplementedError, match="inference"):
        F.cached_attention(k, cache(), ints(1, 2), ints(1))


def test_rates():
    a = F.RotaryAxes((4, 2), base=(100.0, 7.0), scale=(1.0, 3.0))
    got = list(a._c.quarters)
    assert got[:3] == pytest.approx([2 / math.pi, 2 / math.pi / 10, 6 / math.pi], rel=1e-15) and not any(got[3:])


def test_axes_are_copied_and_stored_with_their_module():
    import copy
    import pickle

    from gaussian_splat_encoder.token_reader import TokenReader
    a = F.RotaryAxes((8, 4), base=(100.0, 7.0), scale=(1.0, 3.0), interleaved=True)
    for b in (copy.deepcopy(a), pickle.loads(pickle.dumps(a)), copy.deepcopy(TokenReader(48, 8, a)).axes):
        assert bytes(b._c) == bytes(a._c) and repr(b) == repr(a)


def test_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    ref = ctypes.byref
    r = _lib.SplatRotation(2, 0, (ctypes.c_int * 4)(8, 4, 0, 0))
    p = _lib.SplatPositions(256, 0, 0, 2, 1)
    turn = lambda **kw: lib.splat_rotary(*dict(dict(  # noqa: E731
        r=ref(r), p=ref(p), x=256, xb=64, xl=16, xh=16, dt=0, B=1, L=2, H=1, D=16, back=0, y=256, st=None), **kw).values())
    assert turn(dt=2) == 1 and turn(x=None) == 1 and turn(r=None) == 1 and turn(p=None) == 1 and turn(H=0) == 1
    assert turn(D=8) == 1 and turn(D=129) == 3 and turn(B=0) == 0 and turn(L=0) == 0 and turn(B=4, L=1 << 30) == 3
    for field, value in (("axes", 5), ("axes", -1)):
        old = getattr(r, field)
        setattr(r, field, value)
        assert turn() == 1
        setattr(r, field, old)
    for bad in (3, -2, 0):
        r.dims[0] = bad
        assert turn() == 1
    r.dims[0] = 8
    bwd = lambda **kw: lib.splat_rotary_bwd(*dict(dict(  # noqa: E731
        r=ref(r), p=ref(p), x=256, xb=64, xl=16, xh=16, g=256, gb=64, gl=16, gh=16, dt=0, B=2, L=2, H=1, D=16, dx=256, dp=256,
        shared=1, ws=None, n=0, st=None), **kw).values())
    assert bwd() == 5 and bwd(dp=None) == 1 and bwd(g=None) == 1
    assert lib.splat_rotary_bwd_workspace_bytes(2, 5, 3, 1) == 4 * 30 and lib.splat_rotary_bwd_workspace_bytes(1, 5, 3, 1) == 0
    none = _lib.SplatRotation()
    assert bwd(r=ref(none)) == 1

    c = _lib.SplatCache(0, 2, 2, 16, 8, 4, 9, 256, 256, None, 256, 32, 16, 256, 32, 16, 0, 0, 256, 4, 256, None)
    put = lambda **kw: lib.splat_cache_append(*dict(dict(  # noqa: E731
        c=ref(c), r=None, p=None, k=256, kb=1, kl=1, kh=1, v=256, vb=1, vl=1, vh=1, mask=None, mb=0, ml=0, T=0, st=None),
        **kw).values())
    ask = lambda **kw: lib.splat_cached_attention(*dict(dict(  # noqa: E731
        c=ref(c), r=None, p=None, q=256, qb=1, ql=1, qh=1, H=4, T=1, scale=1.0, causal=1, o=256, ws=256, n=1 << 30, st=None),
        **kw).values())
    assert put() == 0 and ask(T=0) == 0
    assert put(T=-1) == 1 and put(T=1 << 31) == 3 and put(T=1, k=None) == 1 and put(T=1, mask=256) == 1
    assert put(T=1, r=ref(r)) == 1       # no positions
    assert ask(H=3) == 1 and ask(scale=math.nan) == 1 and ask(q=None) == 1 and ask(T=-1) == 1 and ask(T=1 << 30) == 3
    for field, value, rc in (("dtype", 2, 1), ("Hk", 0, 1), ("D", 0, 1), ("D", 130, 3), ("page", 0, 1), ("width", -1, 1),
                             ("pages", -1, 1), ("pages", 1 << 31, 3), ("width", 1 << 30, 3), ("lengths", None, 1),
                             ("tables", None, 1), ("k", None, 1)):
        old = getattr(c, field)
        setattr(c, field, value)
        assert put(T=1) == rc and ask() == rc, field
        setattr(c, field, old)
    c.width = 1000
    assert ask(ws=None, n=0) == 5 and b"workspace" in lib.splat_last_error()

    a = _lib.SplatTokenNorm(0, 8, 4, 0, 1, 1, 0, 0, 0, 1e-6, 1.0, 8, 8)
    fwd = lambda **kw: lib.splat_token_norm_fwd(*dict(dict(  # noqa: E731
        a=ref(a), x=256, h=256, gate=None, w1=None, b1=None, w2=None, b2=None, y=256, n=256, stat=None, st=None), **kw).values())
    assert fwd(x=None) == 1 and fwd(y=None) == 1 and fwd(n=None) == 1 and fwd(h=None) == 1 and fwd(a=None) == 1
    for field, value, rc in (("dtype", 3, 1), ("C", 0, 1), ("C", 8193, 3), ("M", -1, 1), ("gate", 3, 1), ("gate", 2, 1),
                             ("gate", 1, 1), ("act", 1, 1), ("eps", -1.0, 1), ("M", 1 << 31, 3), ("M", 0, 0)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert fwd() == rc, field
        setattr(a, field, old)
    back = lambda **kw: lib.splat_token_norm_bwd(*dict(dict(  # noqa: E731
        a=ref(a), x=256, h=256, gate=None, w1=256, b1=None, w2=None, dy=256, dn=256, stat=256, dx=256, dh=256, dgate=None,
        dw1=256, db1=None, dw2=None, db2=None, ws=None, n=0, st=None), **kw).values())
    assert back() == 5 and back(dy=None, dn=None) == 1 and back(stat=None) == 1 and back(dgate=256) == 1
    assert back(dn=None, dw2=256) == 1 and back(h=None) == 1
    a.gate, a.segs = 1, 3                # four tokens
    assert fwd(gate=256) == 1 and b"divide" in lib.splat_last_error()


def test_attention_workspaces_are_bounded():
    """Partial rows of split sequences only, however many sequences there are."""
    lib = _lib.load()
    c = _lib.SplatCache(1, 1, 8, 128, 64, 2, 9, 256, 256, None, 1, 1, 1, 1, 1, 1, 0, 0, 256, 4, 256, None)
    ask = lambda: lib.splat_cached_attention_workspace_bytes(ctypes.byref(c), 32, 1)  # noqa: E731
    assert ask() == 0            # 128 tokens at most: no split
    c.width = 512
    # two slots a piece, of four rows a key head with their two statistics; at most four rounds of 512 workgroups
    pieces = 4 * 512 // 8
    rows = 2 * pieces * 8 * 4 * (128 + 2) * 4
    assert 0 < ask() <= rows + 8
    c.B = 4096                            # two numbers a sequence and a list of pieces besides
    assert 0 < ask() <= rows + 8 * 4096 + 16 * (pieces + 4096)
