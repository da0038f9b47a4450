"""Operators of tokens that read splats frame by frame, on hand-written HIP kernels (gfx950): rotary positions of several axes,
a paged cache of keys and values with the attention that reads it, norms per token with a block's gate and residual.

They stand beside feature_ops and follow it: float32 or bfloat16 on a HIP device, the last dimension dense (anything else is
copied first), sums and softmax statistics in float32, fixed orders of summation, the current stream, no waits. rotary,
residual_norm and token_norm have gradients (reverse-mode, of first order); the cache is for inference and refuses inputs that
require one. All may be captured into a graph (a backward pass only while no eager graph of the same leaves is alive: torch's
engine would wait for the eager one's stream). The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import SplatCache, SplatPositions, SplatRotation, SplatTokenNorm
from .feature_ops import _MAX_FLOAT, MAX_HEAD, _args, _dense, _launch, _norm_param, _ptr, _rows, _scratch, _wants_grad

MAX_CHANNELS = 8192   # of a norm per token
MAX_AXES = 4
_POSITIONS = {torch.float32: 0, torch.int32: 1, torch.int64: 2}
_KINDS = {"rms": 0, "layer": 1}
_GATE_CODES = {"none": 0, "sigmoid": 5, "silu": 2, "tanh": 4}


# ------------------------------------------------------------------------------------------------ rotary positions
class RotaryAxes:
    """Rates of a rotation by positions of several axes (time, row, column; a splat's centre).

    dims: values of a head that each axis turns, even, one axis after another; values past them pass. Pair i of axis a turns by
    position[a] * scale[a] * base[a] ** (-2 i / dims[a]) radians. base and scale: one number, or one for each axis.
    interleaved: an axis' pairs are neighbours (2 i, 2 i + 1), not (i, i + dims[a] / 2)."""

    def __init__(self, dims, base=10000.0, scale=1.0, interleaved=False):
        self.dims = tuple(int(d) for d in dims)
        if not 1 <= len(self.dims) <= MAX_AXES:
            raise ValueError(f"1 to {MAX_AXES} axes are needed, got {len(self.dims)}")
        if any(d < 2 or d % 2 for d in self.dims) or sum(self.dims) > MAX_HEAD:
            raise ValueError(f"dims must be even, at least 2 and {MAX_HEAD} at most together, got {list(self.dims)}")
        self.base, self.scale = self._each("base", base), self._each("scale", scale)
        if not all(0 < b < math.inf for b in self.base) or not all(abs(s) < math.inf for s in self.scale):
            raise ValueError(f"base must be positive and both finite, got {self.base} and {self.scale}")
        self.interleaved = bool(interleaved)
        try:
            rates = [s * b ** (-2 * i / d) for d, b, s in zip(self.dims, self.base, self.scale) for i in range(d // 2)]
        except OverflowError:
            rates = [math.inf]
        if not all(abs(r) <= _MAX_FLOAT for r in rates):
            raise ValueError(f"rates scale * base ** (-2 i / dims) must be finite float32, got base {self.base}, scale "
                             f"{self.scale}")
        self._c = SplatRotation(len(self.dims), int(self.interleaved), (ctypes.c_int * 4)(*self.dims),
                                (ctypes.c_double * 64)(*(r * 2 / math.pi for r in rates)))

    def __reduce__(self):
        return type(self), (self.dims, self.base, self.scale, self.interleaved)

    def _each(self, name, v):
        v = tuple(float(x) for x in v) if isinstance(v, (tuple, list)) else (float(v),) * len(self.dims)
        if len(v) != len(self.dims):
            raise ValueError(f"{name} needs one number or {len(self.dims)}, got {len(v)}")
        return v

    def __repr__(self):
        return f"RotaryAxes({self.dims}, base={self.base}, scale={self.scale}, interleaved={self.interleaved})"


def _positions(positions, axes, B, L, D, x):
    """C description of positions [B, L, axes] or [L, axes] of x's tokens."""
    if not isinstance(axes, RotaryAxes):
        raise ValueError(f"axes must be RotaryAxes, got {type(axes).__name__}")
    if sum(axes.dims) > D:
        raise ValueError(f"axes of {list(axes.dims)} values do not fit heads of {D}")
    if positions is None:
        raise ValueError("axes need positions")
    A = len(axes.dims)
    shape, kind = positions.shape, _POSITIONS.get(positions.dtype)
    if len(shape) not in (2, 3) or shape[-2:] != (L, A) or (len(shape) == 3 and shape[0] not in (1, B)):
        raise ValueError(f"positions must be [{B}, {L}, {A}] or [{L}, {A}], got {list(shape)}")
    if kind is None:
        raise ValueError(f"positions must be float32, int32 or int64, got {positions.dtype}")
    if positions.get_device() != x.get_device():
        raise ValueError(f"positions are on {positions.device}, the tokens on {x.device}")
    st = positions.stride()
    return SplatPositions(positions.data_ptr(), kind, st[0] if len(shape) == 3 and shape[0] == B else 0, st[-2], st[-1])


def _like(t):
    """A new contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _turn(x, p, axes, dt, back):
    """x (dense heads) turned by the positions that p describes, or back."""
    y = _like(x)
    if y.numel():
        B, L, H, D = x.shape
        sb, sl, sh, _ = x.stride()
        _launch(x, "splat_rotary", axes._c, p, x.data_ptr(), sb, sl, sh, dt, B, L, H, D, back, y.data_ptr())
    return y


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, axes, p, dt):
        x = _dense(x)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, positions)
        ctx.args = (axes, dt)
        return _turn(x, p, axes, dt, 0)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, positions = ctx.saved_tensors
        axes, dt = ctx.args
        g = _dense(g)
        B, L, H, D = g.shape
        p = _positions(positions, axes, B, L, D, g)
        if not ctx.needs_input_grad[1]:
            return _turn(g, p, axes, dt, 1), None, None, None, None
        x = _dense(x)
        dx = _like(x)
        shared = positions.dim() == 2 or positions.shape[0] != B
        new = torch.empty if dx.numel() else torch.zeros
        dp = new(positions.shape, dtype=torch.float32, device=x.device)
        if dx.numel():
            n = _lib.load().splat_rotary_bwd_workspace_bytes(B, L, len(axes.dims), shared)
            keep, ws = _scratch(n, x)
            _launch(x, "splat_rotary_bwd", axes._c, p, x.data_ptr(), *x.stride()[:3], g.data_ptr(), *g.stride()[:3], dt, B,
                    L, H, D, dx.data_ptr(), dp.data_ptr(), shared, ws, n)
        return dx if ctx.needs_input_grad[0] else None, dp, None, None, None


def rotary(x, positions, axes):
    """Turns the pairs of x's heads by their tokens' positions: x [B, L, H, D] (heads may be views) -> the same shape and type.

    positions [B, L, axes], or [L, axes] and [1, L, axes] for all images: float32 (splat centres; they have a gradient, summed
    over the images that share them), int32 or int64. axes: RotaryAxes. Angles are taken in 64 bits: up to 2^31
    radians they are right to 1e-6; far past that they mean nothing, but pairs still keep their length."""
    dt, _ = _args("none", x)
    shape = x.shape
    if len(shape) != 4 or not 1 <= shape[3] <= MAX_HEAD or shape[2] < 1:
        raise ValueError(f"x must be [B, L, H, D] with heads of 1 to {MAX_HEAD} values, got {list(shape)}")
    p = _positions(positions, axes, shape[0], shape[1], shape[3], x)
    if _wants_grad(x, positions):
        return _Rotary.apply(x, positions, axes, p, dt)
    return _turn(_dense(x), p, axes, dt, 0)


# ------------------------------------------------------------------------------------------------ the paged cache
class PagedCache:
    """Pages of keys and values: k and v [pages, page, Hk, D] (any strides with dense heads), and live [pages, page] (bool) or
    None: tokens that are False do not count. Which pages a sequence's tokens lie on is in its table (cache_append)."""

    def __init__(self, k, v, live=None):
        self.dt, _ = _args("none", k, v)
        if k.dim() != 4 or v.shape != k.shape or k.shape[1] < 1 or k.shape[2] < 1 or not 1 <= k.shape[3] <= MAX_HEAD:
            raise ValueError(f"k and v must be [pages, page, Hk, D] with heads of 1 to {MAX_HEAD} values, got "
                             f"{list(k.shape)} and {list(v.shape)}")
        if any(t.shape[3] != 1 and t.stride(3) != 1 for t in (k, v)):
            raise ValueError("a cache's heads must be dense")
        if live is not None and (live.shape != k.shape[:2] or live.dtype is not torch.bool
                                 or live.get_device() != k.get_device()):
            raise ValueError(f"live must be {list(k.shape[:2])} bool on {k.device}, got {list(live.shape)} {live.dtype} on "
                             f"{live.device}")
        if k.requires_grad or v.requires_grad:
            raise ValueError("a cache's pages must not require a gradient")
        self.k, self.v, self.live = k, v, live
        self._shared = any(n > 1 and st == 0 for t in (k, v, live) if t is not None for n, st in zip(t.shape, t.stride()))
        self.pages, self.page, self.heads, self.head_dim = k.shape

    @classmethod
    def empty(cls, pages, page, heads, head_dim, dtype=torch.bfloat16, device="cuda", masked=False):
        """A cache of zeros whose pages hold their tokens head by head (what the attention reads lies together)."""
        k, v = (torch.zeros(pages, heads, page, head_dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
        return cls(k, v, torch.zeros(pages, page, dtype=torch.bool, device=device) if masked else None)

    def tables(self, sequences, first=0):
        """Tables [sequences, pages / sequences] (int32) that share the pages from `first` on out evenly, in order."""
        width = (self.pages - first) // max(1, sequences)
        t = torch.arange(first, first + sequences * width, dtype=torch.int32, device=self.k.device)
        return t.view(sequences, width)

    def _describe(self, tables, lengths, counts, B, T):
        dev = self.k.get_device()
        if tables.dim() != 2 or tables.shape[0] != B or tables.dtype is not torch.int32 or tables.get_device() != dev:
            raise ValueError(f"tables must be [{B}, pages of a sequence] int32 on {self.k.device}, got {list(tables.shape)} "
                             f"{tables.dtype} on {tables.device}")
        if tables.shape[1] > 1 and tables.stride(1) != 1:
            tables = tables.contiguous()
        lengths = self._numbers("lengths", lengths, B, 2 ** 31 - 1)
        counts = None if counts is None else self._numbers("counts", counts, B, T)
        k, v, live = self.k, self.v, self.live
        c = SplatCache(self.dt, B, self.heads, self.head_dim, self.page, tables.shape[1], self.pages, k.data_ptr(),
                       v.data_ptr(), _ptr(live), *k.stride()[:3], *v.stride()[:3], *((0, 0) if live is None else live.stride()),
                       tables.data_ptr(), tables.stride(0), lengths.data_ptr(), _ptr(counts))
        return c, (tables, lengths, counts)

    def _numbers(self, name, t, B, most):
        if t.shape != (B,) or t.dtype not in (torch.int32, torch.int64) or t.get_device() != self.k.get_device():
            raise ValueError(f"{name} must be [{B}] int32 or int64 on {self.k.device}, got {list(t.shape)} {t.dtype} on "
                             f"{t.device}")
        if t.dtype is torch.int64:
            t = t.clamp(0, most).to(torch.int32)
        return t if t.is_contiguous() else t.contiguous()


def _of_cache(cache, positions, axes, *ts):
    """The checks that both operators of a cache share."""
    if not isinstance(cache, PagedCache):
        raise ValueError(f"cache must be a PagedCache, got {type(cache).__name__}")
    _args("none", cache.k, *ts)
    if _wants_grad(cache.k, cache.v, None if axes is None else positions, *ts):
        raise NotImplementedError("the paged cache is for inference: its operators have no gradients")


def cache_append(cache, tables, lengths, k, v, counts=None, positions=None, axes=None, key_mask=None):
    """Writes new tokens' keys and values k, v [B, T, Hk, D] into the cache's pages, the keys turned by positions and axes as by
    rotary where axes is given.

    tables [B, pages of a sequence] (int32): token j of sequence b lies on page tables[b, j // page], place j % page.
    lengths [B] (int32 or int64) counts each sequence's tokens with the new ones; counts [B]: new tokens of each sequence, the
    first ones of its T (all by default): token t goes to place lengths[b] - counts[b] + t. Tokens past their count, before
    the sequence's start, behind its table or on an entry that is no page of the cache are left out, and all other places stay
    as they were. Two tokens of a call must not go to one place. key_mask [B, T] (bool, for a cache with `live`): tokens
    that are False do not count (all do by default). Every tensor is on the device: a captured call follows them. For autograd
    a call is a write in place of the cache's tensors."""
    _of_cache(cache, positions, axes, k, v)
    if cache._shared:
        raise ValueError("a cache of expanded tensors, whose tokens share memory, is only read")
    B, T = k.shape[:2] if k.dim() == 4 else (0, 0)
    if k.dim() != 4 or k.shape != v.shape or k.shape[2:] != cache.k.shape[2:]:
        raise ValueError(f"k and v must be [B, T, {cache.heads}, {cache.head_dim}], got {list(k.shape)} and {list(v.shape)}")
    if key_mask is not None:
        if cache.live is None:
            raise ValueError("key_mask needs a cache with `live`")
        if key_mask.shape != (B, T) or key_mask.dtype is not torch.bool or key_mask.get_device() != k.get_device():
            raise ValueError(f"key_mask must be [{B}, {T}] bool on {k.device}, got {list(key_mask.shape)} {key_mask.dtype} on "
                             f"{key_mask.device}")
    c, keep = cache._describe(tables, lengths, counts, B, T)
    p = r = None
    if axes is not None:
        p, r = _positions(positions, axes, B, T, cache.head_dim, k), axes._c
    if B and T and cache.pages and c.width:
        k, v = _dense(k), _dense(v)
        _launch(k, "splat_cache_append", c, r, p, k.data_ptr(), *k.stride()[:3], v.data_ptr(),
                *v.stride()[:3], _ptr(key_mask), *((0, 0) if key_mask is None else key_mask.stride()), T)
        # the kernel wrote through pointers: what saved a page for its backward has to notice
        increment_version((cache.k, cache.v) if cache.live is None else (cache.k, cache.v, cache.live))


def cached_attention(q, cache, tables, lengths, counts=None, positions=None, axes=None, causal=True, scale=None):
    """Attention of new tokens' queries q [B, T, H, D] over their sequences' cached tokens -> [B, T, H, D]. H is a multiple of the
    cache's heads (each serves H / Hk neighbouring query heads). Meant for one to some tens of new tokens: any number is right, but
    hundreds run at a fraction of cross_attention's rate.

    tables, lengths, counts as in cache_append: the queries are the last counts[b] tokens that lengths[b] counts. causal: query t
    sees the tokens up to its own place, lengths[b] - counts[b] + t; otherwise all. Tokens that the cache's `live` marks
    False, or whose table entry is no page, do not count, whatever they hold. A query without any token, and those past their
    sequence's count, give zeros; an infinite value that counts may give NaN for bfloat16, and for float32 where its probability
    is less than 2^-126. positions, axes: turns q as by rotary. scale defaults to D ** -0.5."""
    _of_cache(cache, positions, axes, q)
    if q.dim() != 4 or q.shape[3] != cache.head_dim or q.shape[2] < 1 or q.shape[2] % cache.heads:
        raise ValueError(f"q must be [B, T, a multiple of {cache.heads}, {cache.head_dim}], got {list(q.shape)}")
    B, T, H, D = q.shape
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _MAX_FLOAT:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    c, keep = cache._describe(tables, lengths, counts, B, T)
    p = r = None
    if axes is not None:
        p, r = _positions(positions, axes, B, T, D, q), axes._c
    o = _like(q)
    if o.numel():
        q = _dense(q)
        n = _lib.load().splat_cached_attention_workspace_bytes(c, H, T)
        held, ws = _scratch(n, q)
        _launch(q, "splat_cached_attention", c, r, p, q.data_ptr(), *q.stride()[:3], H, T, scale, int(bool(causal)),
                o.data_ptr(), ws, n)
    return o


# ------------------------------------------------------------------------------------------------ norms per token
def _lay(t, C):
    """t [..., C] as rows (itself where it is contiguous, whatever its shape) and the elements from row to row."""
    if t.is_contiguous():
        return t, C
    t = _rows(t)
    return t, t.stride(0)


def _norm_args(x, h, gate, kind, eps, scale, act, post, nxt, dt):
    """C description; x, h and the gate as rows."""
    C = x.shape[-1]
    x, xl = _lay(x, C)
    hl = gl = segs = code = 0
    if h is not None:
        h, hl = _lay(h, C)
    if gate is not None:
        n = gate.numel()
        if n == C or n != x.numel() or gate.dtype is not x.dtype:
            gate, code, segs = gate.contiguous(), 1, n // C
        else:
            code = 2
            gate, gl = _lay(gate, C)
    a = SplatTokenNorm(dt, C, x.numel() // C, kind, post, nxt, code, act, segs, eps, scale, xl, hl, gl)
    return a, x, h, gate


def _norm_fwd(x, h, w1, b1, gate, w2, b2, cfg, save):
    """(y or None, n or None, statistics or None)"""
    a, x2, h2, g2 = _norm_args(x, h, gate, *cfg)
    y = None if h is None else _like(x)
    n = _like(x) if a.next else None
    stat = x.new_empty((a.M, 4), dtype=torch.float32) if save else None
    if a.M:
        _launch(x, "splat_token_norm_fwd", a, x2.data_ptr(), _ptr(h2), _ptr(g2), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2),
                _ptr(y), _ptr(n), _ptr(stat))
    return y, n, stat


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, w1, b1, gate, w2, b2, cfg):
        y, n, stat = _norm_fwd(x, h, w1, b1, gate, w2, b2, cfg, True)
        ctx.save_for_backward(x, h, w1, b1, gate, w2, stat)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        return (y, n) if y is not None and n is not None else n if y is None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *up):
        x, h, w1, b1, gate, w2, stat = ctx.saved_tensors
        a, x2, h2, g2 = _norm_args(x, h, gate, *ctx.cfg)
        dy, dn = up if len(up) == 2 else (None, up[0]) if a.next else (up[0], None)
        need = ctx.needs_input_grad
        if dy is None and dn is None:
            return (None,) * 8
        dx = _like(x) if need[0] else None
        dh = _like(h) if need[1] else None
        dgate = None
        if need[4]:
            dgate = _like(gate) if a.M else torch.zeros_like(gate)
        # the parameters' gradients are rows of one tensor; nothing reaches those of the second norm without dn
        rows = (2, 3, 5, 6) if a.M and dn is not None else (2, 3) if a.M else ()
        rows = [i for i in rows if need[i]]
        grads, ptrs, C = {}, [None] * 7, a.C
        if rows:
            par = x.new_empty((len(rows), C), dtype=torch.float32)
            at = par.data_ptr()
            for k, (i, t) in enumerate(zip(rows, par.unbind())):
                grads[i], ptrs[i] = t, at + 4 * C * k
        for i in (2, 3, 5, 6):
            if need[i] and i not in grads:
                grads[i] = x.new_zeros(C, dtype=torch.float32)
        if a.M:
            if dy is not None:
                dy, a.dyl = _lay(dy, C)
            if dn is not None:
                dn, a.dnl = _lay(dn, C)
            n = _lib.load().splat_token_norm_bwd_workspace_bytes(a) if rows or a.gate == 1 else 0
            keep, ws = _scratch(n, x)
            _launch(x, "splat_token_norm_bwd", a, x2.data_ptr(), _ptr(h2), _ptr(g2), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(dy),
                    _ptr(dn), stat.data_ptr(), _ptr(dx), _ptr(dh), _ptr(dgate), ptrs[2], ptrs[3], ptrs[5], ptrs[6], ws, n)
        return dx, dh, grads.get(2), grads.get(3), dgate, grads.get(5), grads.get(6), None


def _check_norm(x, kind, eps):
    if not x.dim() or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"x must be [..., C] of 1 to {MAX_CHANNELS} channels, got {list(x.shape)}")
    if kind not in _KINDS:
        raise ValueError(f"unknown norm {kind!r}: one of {sorted(_KINDS)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")


def token_norm(x, weight=None, bias=None, kind="rms", eps=1e-6):
    """A norm of each token's channels: x [..., C] -> weight * norm(x) + bias, of x's shape and type. kind "rms":
    x / sqrt(mean(x^2) + eps); "layer": of x less its mean. weight and bias [C] may be None; they are used, and their gradients
    returned, in float32. C at most 8,192. (group_norm_act normalises over an image's positions.)"""
    dt, _ = _args("none", x)
    _check_norm(x, kind, eps)
    C = x.shape[-1]
    weight, bias = _norm_param("weight", weight, C, x), _norm_param("bias", bias, C, x)
    cfg = (_KINDS[kind], float(eps), 1.0, 0, 0, 1, dt)
    if _wants_grad(x, weight, bias):
        return _ResidualNorm.apply(x, None, None, None, None, weight, bias, cfg)
    return _norm_fwd(x, None, None, None, None, weight, bias, cfg, False)[1]


def residual_norm(x, h, weight=None, bias=None, gate=None, gate_act="none", next_weight=None, next_bias=None, kind="rms",
                  eps=1e-6, scale=1.0, norm_block=True, norm_next=True):
    """What lies between one block of a model and the next, in one kernel: x [..., C] the residual stream, h (like x) the block's
    output ->

        y = x + scale * gate_act(gate) * (weight * norm(h) + bias)        the new residual stream
        n = next_weight * norm(y) + next_bias                             the next block's input, of y before its rounding

    as (y, n). norm_block=False takes h as it is, norm_next=False returns y alone. kind, parameters and their gradients as in
    token_norm. gate: None; [C] (a learned one), or [B, C] or [B, 1, .., C] (a row for each image of x [B, ..., C]), used in
    float32; or x's shape and type (a row for each token). gate_act: "none", "sigmoid", "silu" or "tanh"."""
    dt, _ = _args("none", x, h)
    _check_norm(x, kind, eps)
    if h.shape != x.shape:
        raise ValueError(f"h must be {list(x.shape)}, got {list(h.shape)}")
    if gate_act not in _GATE_CODES:
        raise ValueError(f"unknown activation {gate_act!r} of a gate: one of {sorted(_GATE_CODES)}")
    scale = float(scale)
    if not abs(scale) <= _MAX_FLOAT:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    C = x.shape[-1]
    if not norm_block and (weight is not None or bias is not None):
        raise ValueError("weight and bias belong to the block's norm, which norm_block=False leaves out")
    if not norm_next and (next_weight is not None or next_bias is not None):
        raise ValueError("next_weight and next_bias belong to the next norm, which norm_next=False leaves out")
    weight, bias = _norm_param("weight", weight, C, x), _norm_param("bias", bias, C, x)
    next_weight, next_bias = _norm_param("next_weight", next_weight, C, x), _norm_param("next_bias", next_bias, C, x)
    if gate is not None:
        gate = _gate(gate, x)
    cfg = (_KINDS[kind], float(eps), scale, _GATE_CODES[gate_act], int(bool(norm_block)), int(bool(norm_next)), dt)
    if _wants_grad(x, h, weight, bias, gate, next_weight, next_bias):
        return _ResidualNorm.apply(x, h, weight, bias, gate, next_weight, next_bias, cfg)
    y, n, _ = _norm_fwd(x, h, weight, bias, gate, next_weight, next_bias, cfg, False)
    return (y, n) if norm_next else y


def _gate(gate, x):
    """The gate as it is (a row for each token), or in float32 (one row, or one for each image)."""
    shape, B, C = gate.shape, x.shape[0] if x.dim() > 1 else 1, x.shape[-1]
    if gate.get_device() != x.get_device():
        raise ValueError(f"gate is on {gate.device}, x on {x.device}")
    if shape == x.shape and gate.dtype is x.dtype and gate.numel() != C:
        return gate
    one = (1,) * (x.dim() - 1) + (C,)
    image = (B,) + (1,) * (x.dim() - 2) + (C,)
    if shape != (C,) and shape != one and (x.dim() < 3 or shape not in (image, (B, C))):
        if shape == x.shape:
            raise ValueError(f"a gate for each token must be {x.dtype}, got {gate.dtype}")
        raise ValueError(f"gate must be [{C}], {list(image)} or {list(x.shape)}, got {list(shape)}")
    return gate if gate.dtype is torch.float32 else gate.float()
