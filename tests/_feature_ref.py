"""Plain float64 implementations of the feature operators (group norm with an activation, products with an epilogue, cross
attention) and the bounds that tests hold the kernels to.

Bounds, on the 2-norm of the error over the 2-norm of the result: float32 kernels sum up to some tens of thousands of terms
in 32-bit floats, in blocks, 64 units of 2^-24 cover that with the activations' own few units; bfloat16 kernels round their
result once (2^-9 at most) and the factor of a second matrix product once (2^-9 at most), so 2^-8 holds both."""

import math

import torch

BOUND = {torch.float32: 64 * 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def act(x, name):
    if name == "gelu":
        return 0.5 * x * torch.erfc(-x * math.sqrt(0.5))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if name == "tanh":
        return torch.tanh(x)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    return x


def group_norm_act(x, G, w, b, eps, name, first):
    B, C = x.shape[0], x.shape[-1]
    u = (act(x, name) if first else x).reshape(B, -1, G, C // G)
    d = u - u.mean((1, 3), keepdim=True)
    y = (d / (d.square().mean((1, 3), keepdim=True) + eps).sqrt()).reshape(x.shape)
    y = y if w is None else y * w
    y = y if b is None else y + b
    return y if first else act(y, name)


def linear_act(x, w, b, name, r):
    z = x @ w.t()
    y = act(z if b is None else z + b, name)
    return y if r is None else y + r


def valid(q, k, lengths, mask):
    """[B, Lk] truth values of the keys that count."""
    B, Lk = k.shape[:2]
    ok = torch.ones(B, Lk, dtype=torch.bool, device=q.device)
    if lengths is not None:
        ok &= torch.arange(Lk, device=q.device)[None] < lengths[:, None]
    return ok if mask is None else ok & mask


def cross_attention(q, k, v, lengths, mask, scale):
    rep = q.shape[2] // k.shape[2]
    ok = valid(q, k, lengths, mask)
    zero = torch.zeros((), dtype=k.dtype, device=k.device)
    k = torch.where(ok[:, :, None, None], k, zero).repeat_interleave(rep, 2).permute(0, 2, 3, 1)
    v = torch.where(ok[:, :, None, None], v, zero).repeat_interleave(rep, 2).permute(0, 2, 1, 3)
    s = q.permute(0, 2, 1, 3) @ k * scale
    ok = ok[:, None, None, :]
    s = torch.where(ok, s, torch.full((), -math.inf, dtype=s.dtype, device=s.device))
    m = s.detach().amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:3] + (1,))
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    t = e.sum(-1, keepdim=True)
    return ((e @ v) / torch.where(t == 0, torch.ones_like(t), t)).permute(0, 2, 1, 3)


def rel(a, b):
    """2-norm of the difference over the 2-norm of b (0 where both are empty or zero)."""
    a, b = a.double(), b.double()
    assert a.shape == b.shape
    if not b.numel():
        return 0.0
    d, n = (a - b).norm().item(), b.norm().item()
    return d / n if n else (0.0 if d == 0 else math.inf)
