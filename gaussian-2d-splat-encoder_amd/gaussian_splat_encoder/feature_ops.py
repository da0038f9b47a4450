"""Operators of channels-last feature maps and of models that read them, on hand-written HIP kernels (gfx950), forward and
backward: group norm with an activation, products with an epilogue, cross attention.

Tensors are float32 or bfloat16 on a HIP device, the last dimension dense (anything else is copied first); sums, softmax
statistics and norms are float32 whatever the type. Results are deterministic: no atomics, fixed orders of summation.
Everything runs on the current stream and returns without waiting. Gradients are reverse-mode, of first order (forward-mode
and second derivatives are refused). Device work goes through libsplat_hip.so (include/splat_render.h). The reference has
no counterpart: its network runs on stock torch operations.

Activations: "none", "gelu" (x Phi(x)), "silu", "relu", "tanh", "sigmoid".
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import SplatAttention, check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_KEPT = {torch.float32: torch.float32, torch.bfloat16: torch.float16}   # type of an activation's input for its backward
_ACTS = {"none": 0, "gelu": 1, "silu": 2, "relu": 3, "tanh": 4, "sigmoid": 5}
MAX_HEAD = 128   # values of a head at most
_MAX_FLOAT = torch.finfo(torch.float32).max


def _args(act, x, *others):
    """Type and activation codes of a call; x's type and device are every other tensor's too."""
    if not x.is_cuda:
        raise RuntimeError("the HIP feature operators need device tensors (got a CPU tensor)")
    dtype, dev = x.dtype, x.get_device()
    for t in others:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("the HIP feature operators need device tensors (got a CPU tensor)")
        if t.dtype is not dtype:
            raise ValueError(f"tensors of one type are needed, got {dtype} and {t.dtype}")
        if t.get_device() != dev:
            raise ValueError(f"tensors of one device are needed, got {x.device} and {t.device}")
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"float32 or bfloat16 is needed, got {dtype}")
    code = _ACTS.get(act)
    if code is None:
        raise ValueError(f"unknown activation {act!r}: one of {sorted(_ACTS)}")
    return dt, code


def _ptr(t):
    return None if t is None else t.data_ptr()


def _scratch(nbytes, x):
    """(tensor that keeps the workspace, its pointer); the caller's stream owns it like any torch tensor."""
    if not nbytes:
        return None, None
    t = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    return t, t.data_ptr()


def _launch(x, name, *args):
    """Calls the library's entry point on the current stream of x's device (the library launches on the current device,
    which is made x's where it is another)."""
    fn, i = getattr(_lib.load(), name), x.get_device()
    if i == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        check(rc, name)


def _wants_grad(*ts):
    """Whether a backward may follow. Tangents, which say nothing in requires_grad, are refused."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the HIP feature operators have no forward-mode derivatives")
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ------------------------------------------------------------------------------------------------ group norm
def _positions(x):
    """x [B, ..., C] with dense channels and positions at one distance (itself where its strides allow that), and B, L, C and
    the distances of images and positions."""
    shape = x.shape
    B, C = shape[0], shape[-1]
    L = math.prod(shape[1:-1])
    if x.is_contiguous():
        return x, B, L, C, L * C, C
    x = x.reshape(B, L, C)
    if C != 1 and x.stride(2) != 1:
        x = x.contiguous()
    return x, B, L, C, x.stride(0), x.stride(1)


def _norm_fwd(x, weight, bias, G, eps, dt, act, first, save):
    """(result like x, x as _positions has it, statistics or None)"""
    at = xp, B, L, C, sb, sl = _positions(x)
    y = x.new_empty(x.shape)
    stat = x.new_empty((2, B, G), dtype=torch.float32) if save else None
    if B and L:
        n = _lib.load().splat_group_norm_workspace_bytes(dt, B, L, C, G)
        keep, ws = _scratch(n, x)
        sp = _ptr(stat)
        _launch(x, "splat_group_norm_fwd", xp.data_ptr(), sb, sl, _ptr(weight), _ptr(bias), dt, B, L, C, G, eps, act, first,
                y.data_ptr(), sp, sp + 4 * B * G if save else None, ws, n)
    return y, at, stat


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, G, eps, dt, act, first):
        y, at, stat = _norm_fwd(x, weight, bias, G, eps, dt, act, first, True)
        ctx.save_for_backward(at[0], weight, bias, stat)
        ctx.args = (x.shape, G, dt, act, first)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stat = ctx.saved_tensors
        shape, G, dt, act, first = ctx.args
        x, B, L, C, xb, xl = _positions(x)          # what a saved-tensor hook gives back may lie differently
        need = ctx.needs_input_grad
        new = x.new_empty if B and L else x.new_zeros
        dx = x.new_empty(shape)
        dw = new(C, dtype=torch.float32) if need[1] else None
        db = new(C, dtype=torch.float32) if need[2] else None
        if B and L:
            g, _, _, _, gb, gl = _positions(dy)
            n = _lib.load().splat_group_norm_bwd_workspace_bytes(dt, B, L, C, G)
            keep, ws = _scratch(n, x)
            sp = stat.data_ptr()
            _launch(x, "splat_group_norm_bwd", x.data_ptr(), xb, xl, g.data_ptr(), gb, gl, _ptr(weight), _ptr(bias), sp,
                    sp + 4 * B * G, dt, B, L, C, G, act, first, dx.data_ptr(), _ptr(dw), _ptr(db), ws, n)
        return dx if need[0] else None, dw, db, None, None, None, None, None


def _norm_param(name, t, C, x):
    """A norm parameter as dense float32 (itself where it is that)."""
    if t is None:
        return None
    if t.shape != (C,):
        raise ValueError(f"{name} must be [{C}], got {list(t.shape)}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if t.dtype is not torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="gelu", act_first=False):
    """Group norm and an activation on a channels-last map: x [B, ..., C] -> the same shape and type.

    act_first=False: act(weight * norm(x) + bias). act_first=True: weight * norm(act(x)) + bias, the order of the encoder's
    stages (conv -> GELU -> norm). The mean and the biased variance run over the C / num_groups channels of a group and all
    positions of an image (a norm per token: B tokens of no positions, [B, C]; millions of images fit a launch). weight and
    bias [C] may be None; they are used, and their gradients returned, in float32."""
    dt, code = _args(act, x)
    if x.dim() < 2:
        raise ValueError(f"x must be [B, ..., C], got {list(x.shape)}")
    C, G = x.shape[-1], int(num_groups)
    if G < 1 or C < 1 or C % G:
        raise ValueError(f"{C} channels do not divide into {num_groups} groups")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    weight, bias = _norm_param("weight", weight, C, x), _norm_param("bias", bias, C, x)
    first = 1 if act_first else 0
    if _wants_grad(x, weight, bias):
        return _GroupNormAct.apply(x, weight, bias, G, float(eps), dt, code, first)
    return _norm_fwd(x, weight, bias, G, float(eps), dt, code, first, False)[0]


# ------------------------------------------------------------------------------------------------ products
def _rows(x):
    """x [..., K] as [M, K] with dense rows (a view where the strides allow it)."""
    if x.dim() != 2:
        x = x.reshape(math.prod(x.shape[:-1]), x.shape[-1])
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _linear_fwd(x, weight, bias, residual, out, dt, act, save):
    """(result of shape `out`, x as [M, K], the activation's input or None)"""
    x2 = _rows(x)
    M, K = x2.shape
    N = out[-1]
    y = x.new_empty(out)
    z = x.new_empty((M, N), dtype=_KEPT[x.dtype]) if save and act else None
    if M:
        r2 = None if residual is None else _rows(residual)
        _launch(x, "splat_linear_fwd", x2.data_ptr(), x2.stride(0), weight.data_ptr(), _ptr(bias), _ptr(r2),
                0 if r2 is None else r2.stride(0), dt, M, N, K, act, y.data_ptr(), _ptr(z))
    return y, x2, z


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, out, dt, act):
        y, x2, z = _linear_fwd(x, weight, bias, residual, out, dt, act, True)
        ctx.save_for_backward(x2, weight, z)
        ctx.args = (x.shape, dt, act)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x2, weight, z = ctx.saved_tensors
        shape, dt, act = ctx.args
        need = ctx.needs_input_grad
        M, K = x2.shape
        N = weight.shape[0]
        new = x2.new_empty if M else x2.new_zeros
        dx = x2.new_empty(shape) if need[0] else None
        dw = new((N, K)) if need[1] else None
        db = new(N) if need[2] else None
        if M and (need[0] or need[1] or need[2]):
            g = dy.contiguous()
            n = _lib.load().splat_linear_bwd_workspace_bytes(dt, M, N, K, act)
            keep, ws = _scratch(n, x2)
            _launch(x2, "splat_linear_bwd", x2.data_ptr(), x2.stride(0), weight.data_ptr(), g.data_ptr(), _ptr(z), dt, M, N,
                    K, act, _ptr(dx), _ptr(dw), _ptr(db), ws, n)
        return dx, dw, db, dy if need[3] else None, None, None, None


def linear_act(x, weight, bias=None, act="none", residual=None):
    """act(x weight^T + bias) + residual in one kernel: x [..., K], weight [N, K] (nn.Linear's, or a 1x1 convolution's
    flattened), bias [N] or None, residual [..., N] or None -> [..., N]. All of one type; the product, the bias, the
    activation and the residual are added in float32 and rounded once."""
    dt, code = _args(act, x, weight, bias, residual)
    xs, ws = x.shape, weight.shape
    if len(xs) < 1 or len(ws) != 2 or xs[-1] != ws[1]:
        raise ValueError(f"x [..., K] and weight [N, K] are needed, got {list(xs)} and {list(ws)}")
    N, K = ws
    if N < 1 or K < 1:
        raise ValueError(f"weight must not be empty, got {list(ws)}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must be [{N}], got {list(bias.shape)}")
    out = xs[:-1] + (N,)
    if residual is not None and residual.shape != out:
        raise ValueError(f"residual must be {list(out)}, got {list(residual.shape)}")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if _wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, out, dt, code)
    return _linear_fwd(x, weight, bias, residual, out, dt, code, False)[0]


# ------------------------------------------------------------------------------------------------ cross attention
def _dense(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _describe(q, k, v, lengths, mask, scale, dt):
    B, Lq, H, D = q.shape
    a = SplatAttention(dt, B, H, k.shape[2], D, scale, Lq, k.shape[1], *q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    if lengths is not None:
        a.kv_lengths = lengths.data_ptr()
    if mask is not None:
        a.key_mask = mask.data_ptr()
        a.mb, a.ml = mask.stride()
    return a


def _attention_fwd(q, k, v, lengths, mask, scale, dt, save):
    """(result, log sums, what rounding to bfloat16 left of the result or, for float32, inverse sums; the two None where no
    backward follows)"""
    B, Lq, H, D = q.shape
    o = q.new_empty((B, Lq, H, D))
    lse = q.new_empty(B * Lq * H, dtype=torch.float32) if save else None
    rest = None if not save else torch.empty_like(o) if dt else torch.empty_like(lse)
    if o.numel():
        a = _describe(q, k, v, lengths, mask, scale, dt)
        a.rest = _ptr(rest)
        ref = ctypes.byref(a)
        n = _lib.load().splat_attention_workspace_bytes(ref)
        keep, ws = _scratch(n, q)
        _launch(q, "splat_attention_fwd", ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(lse), ws, n)
    return o, lse, rest


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale, dt):
        q, k, v = _dense(q), _dense(k), _dense(v)
        o, lse, rest = _attention_fwd(q, k, v, lengths, mask, scale, dt, True)
        ctx.save_for_backward(q, k, v, o, lse, rest, lengths, mask)
        ctx.args = (scale, dt)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q, k, v, o, lse, rest, lengths, mask = ctx.saved_tensors
        scale, dt = ctx.args
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if dq.numel() or dk.numel():
            g = _dense(g)
            a = _describe(q, k, v, lengths, mask, scale, dt)
            a.gb, a.gl, a.gh = g.stride()[:3]
            a.rest = _ptr(rest)
            ref = ctypes.byref(a)
            n = _lib.load().splat_attention_bwd_workspace_bytes(ref)
            keep, ws = _scratch(n, q)
            _launch(q, "splat_attention_bwd", ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(),
                    g.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ws, n)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def cross_attention(q, k, v, kv_lengths=None, key_mask=None, scale=None):
    """Attention of one sequence's queries over another's keys and values: q [B, Lq, H, D], k and v [B, Lk, Hk, D] ->
    [B, Lq, H, D]. H is a multiple of Hk (each key head serves H / Hk neighbouring query heads), D at most 128; the three
    may be views (halves of one projection, transposed heads) as long as the head vectors are dense.

    kv_lengths [B] (integers, on the device): an image's keys past its length do not count. key_mask [B, Lk] (bool): keys
    that are False do not count. What such keys hold has no effect, and their gradients are zero; a query without any key
    gives zeros. scale defaults to D ** -0.5."""
    dt, _ = _args("none", q, k, v)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q [B, Lq, H, D] and k, v [B, Lk, Hk, D] are needed, got {list(q.shape)}, {list(k.shape)} and "
                         f"{list(v.shape)}")
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    if H < 1 or Hk < 1 or H % Hk:
        raise ValueError(f"{H} query heads do not divide over {Hk} key heads")
    if not 1 <= D <= MAX_HEAD:
        raise ValueError(f"heads of 1 to {MAX_HEAD} values are needed, got {D}")
    if kv_lengths is not None:
        if kv_lengths.shape != (B,) or kv_lengths.dtype not in (torch.int32, torch.int64) or kv_lengths.device != q.device:
            raise ValueError(f"kv_lengths must be [{B}] int32 or int64 on {q.device}, got {list(kv_lengths.shape)} "
                             f"{kv_lengths.dtype} on {kv_lengths.device}")
        if kv_lengths.dtype is torch.int64:
            kv_lengths = kv_lengths.clamp(0, Lk).to(torch.int32)
        kv_lengths = kv_lengths.contiguous()
    if key_mask is not None and (key_mask.shape != (B, Lk) or key_mask.dtype is not torch.bool
                                 or key_mask.device != q.device):
        raise ValueError(f"key_mask must be [{B}, {Lk}] bool on {q.device}, got {list(key_mask.shape)} {key_mask.dtype} on "
                         f"{key_mask.device}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _MAX_FLOAT:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    if _wants_grad(q, k, v):
        return _CrossAttention.apply(q, k, v, kv_lengths, key_mask, scale, dt)
    return _attention_fwd(_dense(q), _dense(k), _dense(v), kv_lengths, key_mask, scale, dt, False)[0]
