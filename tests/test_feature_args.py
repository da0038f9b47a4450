"""Host-side refusals of the feature operators (CPU; no kernel runs), and the C entry points' own argument checks."""

import ctypes

import pytest
import torch

from gaussian_splat_encoder import _lib
from gaussian_splat_encoder import feature_ops as F


class Dev(torch.Tensor):
    """A host tensor that says it is on a device: the checks before any launch are what is tested."""
    is_cuda = True


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Dev)


def test_cpu_tensors_are_refused():
    z = torch.zeros
    for call in (lambda: F.group_norm_act(z(1, 4, 8), 2), lambda: F.linear_act(z(2, 4), z(3, 4)),
                 lambda: F.cross_attention(z(1, 2, 1, 8), z(1, 3, 1, 8), z(1, 3, 1, 8))):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()


@pytest.mark.parametrize("call,what", [
    (lambda: F.group_norm_act(t(1, 4, 8), 3), "divide"),
    (lambda: F.group_norm_act(t(1, 4, 8), 0), "divide"),
    (lambda: F.group_norm_act(t(8), 2), r"\[B, ..., C\]"),
    (lambda: F.group_norm_act(t(1, 4, 8), 2, act="swish"), "unknown activation"),
    (lambda: F.group_norm_act(t(1, 4, 8), 2, eps=-1.0), "eps"),
    (lambda: F.group_norm_act(t(1, 4, 8), 2, weight=t(4)), "weight must be"),
    (lambda: F.group_norm_act(t(1, 4, 8), 2, bias=t(1, 8)), "bias must be"),
    (lambda: F.group_norm_act(t(1, 4, 8, dtype=torch.float16), 2), "float32 or bfloat16"),
    (lambda: F.linear_act(t(2, 4), t(3, 5)), "weight"),
    (lambda: F.linear_act(t(2, 4), t(0, 4)), "empty"),
    (lambda: F.linear_act(t(2, 4), t(3, 4), t(4)), "bias must be"),
    (lambda: F.linear_act(t(2, 4), t(3, 4), residual=t(3)), "residual must be"),
    (lambda: F.linear_act(t(2, 4), t(3, 4, dtype=torch.bfloat16)), "one type"),
    (lambda: F.linear_act(t(2, 4), t(3, 4), act=None), "unknown activation"),
    (lambda: F.cross_attention(t(1, 2, 8), t(1, 3, 1, 8), t(1, 3, 1, 8)), "are needed"),
    (lambda: F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 4, 1, 8)), "are needed"),
    (lambda: F.cross_attention(t(2, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8)), "are needed"),
    (lambda: F.cross_attention(t(1, 2, 3, 8), t(1, 3, 2, 8), t(1, 3, 2, 8)), "do not divide"),
    (lambda: F.cross_attention(t(1, 2, 1, 160), t(1, 3, 1, 160), t(1, 3, 1, 160)), "1 to 128"),
    (lambda: F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8), kv_lengths=torch.zeros(2, dtype=torch.int32)),
     "kv_lengths"),
    (lambda: F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8), kv_lengths=torch.zeros(1)), "kv_lengths"),
    (lambda: F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8), key_mask=torch.zeros(1, 3)), "key_mask"),
    (lambda: F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8), key_mask=torch.zeros(3, dtype=torch.bool)),
     "key_mask"),
])
def test_wrong_arguments_are_refused(call, what):
    with pytest.raises(ValueError, match=what):
        call()


def test_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    norm = lambda **kw: lib.splat_group_norm_fwd(*dict(dict(  # noqa: E731
        x=256, xsb=64, xsl=8, w=None, b=None, dt=0, B=1, L=8, C=8, G=2, eps=1e-5, act=1, first=0, y=256, mean=None,
        rstd=None, ws=None, n=0, st=None), **kw).values())
    assert norm(G=3) == 1 and norm(act=6) == 1 and norm(dt=2) == 1 and norm(x=None) == 1 and norm(mean=256) == 1
    assert norm(L=1 << 20) == 5 and b"workspace" in lib.splat_last_error()
    assert norm(B=0) == 0 and norm(L=0) == 0
    lin = lambda **kw: lib.splat_linear_fwd(*dict(dict(  # noqa: E731
        x=256, ldx=8, w=256, b=None, r=None, ldr=0, dt=0, M=4, N=8, K=8, act=0, y=256, z=None, st=None), **kw).values())
    assert lin(K=0) == 1 and lin(N=0) == 1 and lin(M=-1) == 1 and lin(act=9) == 1 and lin(w=None) == 1 and lin(M=0) == 0
    assert lin(M=1 << 33) == 3
    assert lib.splat_linear_bwd(256, 8, 256, 256, None, 0, 4, 8, 8, 1, 256, None, None, 256, 1 << 20, None) == 1   # no z
    assert lib.splat_linear_bwd(256, 8, 256, 256, None, 0, 4, 8, 8, 0, 256, 256, None, 256, 8, None) == 5
    a = _lib.SplatAttention(0, 1, 4, 2, 64, 0.125, 2, 5000)   # few rows, many keys: split, so a workspace is due
    fwd = lambda: lib.splat_attention_fwd(ctypes.byref(a), 256, 256, 256, 256, None, None, 0, None)  # noqa: E731
    assert fwd() == 5
    for field, value, rc in (("H", 3, 1), ("D", 129, 3), ("D", 0, 1), ("dtype", 7, 1), ("Lk", 1 << 33, 3), ("Lq", -1, 1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert fwd() == rc, field
        setattr(a, field, old)
    assert lib.splat_attention_fwd(None, *[256] * 4, None, None, 0, None) == 1
    assert lib.splat_attention_fwd(ctypes.byref(a), None, 256, 256, 256, None, 256, 1 << 20, None) == 1
    a.B = 0
    assert fwd() == 0


def test_workspaces_are_what_the_plans_need():
    lib = _lib.load()
    assert lib.splat_group_norm_workspace_bytes(0, 1, 576, 64, 8) == 0          # one launch, no partial sums
    assert lib.splat_group_norm_workspace_bytes(1, 1, 384 * 384, 64, 8) > 0
    assert lib.splat_group_norm_workspace_bytes(1, 0, 5, 64, 8) == 0
    a = _lib.SplatAttention(1, 1, 4, 4, 64, 0.125, 36864, 100)
    assert lib.splat_attention_workspace_bytes(ctypes.byref(a)) == 0            # few keys: no split
    a.Lq, a.Lk = 1, 92160
    assert lib.splat_attention_workspace_bytes(ctypes.byref(a)) > 0
