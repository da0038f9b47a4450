"""Calls that the feature operators refuse, and layouts that they promise, at the edges (CPU; no kernel runs)."""

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

from gaussian_splat_encoder import _lib
from gaussian_splat_encoder import feature_ops as F


class Dev(torch.Tensor):
    """A host tensor that says it is on a device: the checks before any launch are what is tested."""
    is_cuda = True


def t(*shape):
    return torch.zeros(*shape).as_subclass(Dev)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call,n", [
    (lambda *a: F.group_norm_act(a[0], 2, a[1], a[2]), 3),
    (lambda *a: F.linear_act(a[0], a[1], a[2], residual=a[3]), 4),
    (lambda *a: F.cross_attention(*a), 3)])
def test_forward_mode_is_refused(call, n, grad):
    """A tangent on any input: a result without one would be a wrong derivative."""
    norm = call.__code__.co_names[1] == "group_norm_act"
    shapes = ([(1, 4, 8), (8,), (8,)] if norm else [(2, 4), (3, 4), (3,), (2, 3)] if n == 4 else
              [(1, 2, 1, 8), (1, 3, 1, 8), (1, 3, 1, 8)])
    for i in range(n):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            a = [t(*s) for s in shapes]
            a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i])).as_subclass(Dev)
            assert forward_ad.unpack_dual(a[i]).tangent is not None
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*a)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_attention_scale_has_to_be_finite(scale):
    with pytest.raises(ValueError, match="scale"):
        F.cross_attention(t(1, 2, 1, 8), t(1, 3, 1, 8), t(1, 3, 1, 8), scale=scale)
    a = _lib.SplatAttention(0, 1, 1, 1, 8, scale, 2, 3)
    lib = _lib.load()
    assert lib.splat_attention_fwd(ctypes.byref(a), 256, 256, 256, 256, None, None, 0, None) == 1
    assert b"scale" in lib.splat_last_error()


def test_products_that_a_launch_cannot_hold():
    """2^32 threads and more: an answer before any launch."""
    lib = _lib.load()
    lin = lambda M, N, K: lib.splat_linear_fwd(256, K, 256, None, None, 0, 1, M, N, K, 0, 256, None, None)  # noqa: E731
    assert lin(1, 1 << 28, 1) == 3 and lin(32, 1 << 30, 8) == 3
    bwd = lambda M, N, K: lib.splat_linear_bwd(256, K, 256, 256, None, 1, M, N, K, 0, None, 256, None, 256,  # noqa: E731
                                               1 << 60, None)
    assert bwd(1, 1 << 18, 1 << 17) == 3


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D,Lq", [(33, 77), (1, 301), (127, 3), (64, 16)])
def test_attention_statistics_are_aligned(dtype, D, Lq):
    """The workspace holds two statistics of every split and row, then (from a multiple of 256 bytes) D values of each:
    neither depends on how the other divides."""
    a = _lib.SplatAttention(dtype, 1, 1, 1, D, 0.125, Lq, 20001)
    n = _lib.load().splat_attention_workspace_bytes(ctypes.byref(a))
    splits = [s for s in range(2, 513) if n == (8 * s * Lq + 255) // 256 * 256 + 4 * s * Lq * D]
    assert len(splits) == 1


def test_norm_of_many_images():
    """An image per token: 92,160 splat latents, and as many as a launch holds."""
    lib = _lib.load()
    assert lib.splat_group_norm_bwd_workspace_bytes(0, 92160, 1, 64, 8) > 0
    norm = lambda B, C: lib.splat_group_norm_fwd(256, C, C, None, None, 0, B, 1, C, 1, 1e-5, 0, 0, 256, None,  # noqa: E731
                                                 None, None, 0, None)
    assert norm(1 << 23, 8) == 3 and norm((1 << 31) - 1, 8) == 3
