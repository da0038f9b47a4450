"""Plain float64 implementations of the token operators (rotary positions, paged cache, norms per token with gate and residual).

Bounds as in _feature_ref: a float32 result is a sum of some thousands of terms in blocks (64 units of 2^-24 of the 2-norm), a
bfloat16 one is rounded once more, by 2^-8 of itself at most."""

import math

import torch


def rotary(x, positions, axes):
    """x [B, L, H, D], positions [B or 1, L, A] or [L, A], all float64."""
    out, at = [], 0
    for a, d in enumerate(axes.dims):
        i = torch.arange(d // 2, dtype=torch.float64, device=x.device)
        w = positions[..., a, None, None] * (axes.scale[a] * axes.base[a] ** (-2 * i / d))
        c, s = torch.cos(w), torch.sin(w)
        v = x[..., at:at + d]
        x0, x1 = (v[..., 0::2], v[..., 1::2]) if axes.interleaved else (v[..., :d // 2], v[..., d // 2:])
        y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
        out.append(torch.stack([y0, y1], -1).flatten(-2) if axes.interleaved else torch.cat([y0, y1], -1))
        at += d
    return torch.cat(out + [x[..., at:]], -1)


def places(tables, length, count, page):
    """(token, page, place) of a sequence's new tokens that have one; `tables` is its row (a list)."""
    out = []
    for t in range(count):
        j = length - count + t
        if 0 <= j < len(tables) * page:
            out.append((t, tables[j // page], j % page))
    return out


def append(kc, vc, live, tables, lengths, k, v, counts, mask):
    """Writes into clones of the cache's tensors; k as it is stored."""
    kc, vc, live = kc.clone(), vc.clone(), None if live is None else live.clone()
    pages, page = kc.shape[:2]
    B, T = k.shape[:2]
    for b in range(B):
        n = T if counts is None else max(0, min(T, int(counts[b])))
        for t, p, o in places(tables[b].tolist(), int(lengths[b]), n, page):
            if 0 <= p < pages:
                kc[p, o], vc[p, o] = k[b, t], v[b, t]
                if live is not None:
                    live[p, o] = True if mask is None else mask[b, t]
    return kc, vc, live


def attention(q, kc, vc, live, tables, lengths, counts, causal, scale):
    """q [B, T, H, D] float64 as turned; the cache in its own type."""
    B, T, H, D = q.shape
    pages, page, Hk, _ = kc.shape
    o = torch.zeros_like(q)
    rep = H // Hk
    for b in range(B):
        n = max(0, min(int(lengths[b]), tables.shape[1] * page))
        c = T if counts is None else max(0, min(T, int(counts[b])))
        j = torch.arange(n, device=q.device)
        p, at = tables[b].long()[j // page], j % page
        ok = (p >= 0) & (p < pages)
        if live is not None:
            ok = ok & live[p.clamp(0, pages - 1), at]
        j, p, at = j[ok], p[ok], at[ok]
        k, v = kc[p, at].double(), vc[p, at].double()            # [keys, Hk, D]
        for t in range(c):
            see = j < max(0, int(lengths[b])) - (c - 1 - t) if causal else j >= 0
            if not bool(see.any()):
                continue
            kt, vt = k[see].repeat_interleave(rep, 1), v[see].repeat_interleave(rep, 1)
            s = (q[b, t][None] * kt).sum(-1) * scale             # [keys, H]
            w = torch.exp(s - s.amax(0))
            o[b, t] = (w[..., None] * vt).sum(0) / w.sum(0)[:, None]
    return o


def norm(x, w, b, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if w is None else y * w
    return y if b is None else y + b


def act(g, name):
    return {"none": lambda t: t, "sigmoid": lambda t: 1 / (1 + torch.exp(-t)), "tanh": torch.tanh,
            "silu": lambda t: t / (1 + torch.exp(-t))}[name](g)


def residual_norm(x, h, w, b, gate, name, w2, b2, kind, eps, scale, block, nxt):
    z = norm(h, w, b, kind, eps) if block else h
    if gate is not None:
        if gate.dim() == 2 and x.dim() > 2:
            gate = gate.reshape(gate.shape[:1] + (1,) * (x.dim() - 2) + gate.shape[1:])
        z = z * act(gate, name)
    y = x + scale * z
    return (y, norm(y, w2, b2, kind, eps)) if nxt else (y,)


def bound_of(t):
    """Bound on the 2-norm of the error of a result of type t that float32 arithmetic made."""
    return 64 * 2.0 ** -24 + (2.0 ** -8 if t is torch.bfloat16 else 0.0)
