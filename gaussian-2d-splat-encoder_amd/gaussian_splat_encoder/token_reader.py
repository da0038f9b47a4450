"""TokenReader: a layer of tokens that read states with positions (the splats of a stream of frames, a map's cells, earlier
tokens), dense in training and over a paged cache in serving (there also in order, which the dense attention has no mode for):

    a = attention(turn(q(norm(x))), turn(k(states)), v(states))     y = x + gate norm(out(a))     y + gate norm(fc2(gelu(fc1(norm(y)))))

on token_ops (norms per token before and after each half, its gate and residual in one kernel; rotary positions of several
axes; the cache) and feature_ops (products, dense attention). Gates start at zero, so a new layer is the identity. The
norms run over a token's channels, not over an image as CellReader's do, so that tokens that come one by one give what they
give together. The reference has no counterpart."""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .cell_reader import CellReader
from .feature_ops import cross_attention
from .token_ops import PagedCache, RotaryAxes, cache_append, cached_attention, residual_norm, rotary, token_norm


class TokenReader(nn.Module):
    """channels: of x; state_channels: of the states; axes: RotaryAxes of the positions; heads, kv_heads: query heads and the key
    heads that they share (all their own by default); hidden: the perceptron's width (twice the channels by default); kind, eps:
    of the norms."""

    def __init__(self, channels, state_channels, axes, heads=4, kv_heads=None, head_dim=None, hidden=None, kind="rms",
                 eps=1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads do not divide over {kv_heads} key heads")
        if head_dim is None:
            if channels % heads:
                raise ValueError(f"{channels} channels do not divide into {heads} heads: give head_dim")
            head_dim = channels // heads
        if not isinstance(axes, RotaryAxes) or sum(axes.dims) > head_dim:
            raise ValueError(f"axes must be RotaryAxes of {head_dim} values at most, got {axes}")
        hidden = 2 * channels if hidden is None else hidden
        self.axes, self.heads, self.kv_heads, self.head_dim, self.kind, self.eps = axes, heads, kv_heads, head_dim, kind, eps
        self.to_q = nn.Linear(channels, heads * head_dim)
        self.to_kv = nn.Linear(state_channels, 2 * kv_heads * head_dim)
        self.to_out = nn.Linear(heads * head_dim, channels)
        self.fc1 = nn.Linear(channels, hidden)
        self.fc2 = nn.Linear(hidden, channels)
        for name in ("norm1", "post1", "norm2", "post2"):      # before and after the attention and the perceptron
            self.register_parameter(name, nn.Parameter(torch.ones(channels)))
        self.gate1, self.gate2 = nn.Parameter(torch.zeros(channels)), nn.Parameter(torch.zeros(channels))

    _product = staticmethod(CellReader._product)

    def _queries(self, x):
        """[B, L, heads, head_dim] of x [B, L, channels], before their turn."""
        n = token_norm(x, self.norm1, kind=self.kind, eps=self.eps)
        return self._product(n, self.to_q).reshape(x.shape[0], x.shape[1], self.heads, self.head_dim)

    def keys_values(self, states):
        """Keys (before their turn) and values, each [B, Lk, kv_heads, head_dim], of states [B, Lk, state_channels]."""
        kv = self._product(states, self.to_kv)
        kv = kv.reshape(states.shape[0], math.prod(states.shape[1:-1]), 2, self.kv_heads, self.head_dim)
        return kv[:, :, 0], kv[:, :, 1]

    def _rest(self, x, a):
        """What follows the attention a [B, L, heads, head_dim]."""
        h = self._product(a.reshape(x.shape[:-1] + (self.heads * self.head_dim,)), self.to_out)
        y, n = residual_norm(x, h, self.post1, gate=self.gate1, next_weight=self.norm2, kind=self.kind, eps=self.eps)
        h = self._product(self._product(n, self.fc1, act="gelu"), self.fc2)
        return residual_norm(y, h, self.post2, gate=self.gate2, norm_next=False, kind=self.kind, eps=self.eps)

    def forward(self, x, positions, states, state_positions, kv_lengths=None, key_mask=None):
        """x [B, L, channels] at positions [B, L, axes] or [L, axes] reads states [B, Lk, state_channels] at state_positions
        -> like x, with gradients. kv_lengths [B] and key_mask [B, Lk] leave states out."""
        k, v = self.keys_values(states)
        q = rotary(self._queries(x), positions, self.axes)
        return self._rest(x, cross_attention(q, rotary(k, state_positions, self.axes), v, kv_lengths=kv_lengths,
                                             key_mask=key_mask))

    def new_cache(self, sequences, tokens, page=64, dtype=torch.bfloat16, device="cuda", masked=False):
        """A cache with room for `tokens` states of each sequence, and its tables. dtype: the states', which keys and values
        have too."""
        cache = PagedCache.empty(sequences * -(-tokens // page), page, self.kv_heads, self.head_dim, dtype, device, masked)
        return cache, cache.tables(sequences)

    @torch.no_grad()
    def append(self, cache, tables, lengths, states, state_positions, counts=None, key_mask=None):
        """Puts states [B, T, state_channels] behind those in the cache; lengths [B] count them already (cache_append)."""
        k, v = self.keys_values(states)
        cache_append(cache, tables, lengths, k, v, counts=counts, positions=state_positions, axes=self.axes, key_mask=key_mask)

    @torch.no_grad()
    def read(self, x, positions, cache, tables, lengths, counts=None, causal=False):
        """forward's result for x [B, T, channels] over the cached states, without gradients; causal: x are the last tokens that
        the cache holds, and each sees those up to itself (cached_attention)."""
        a = cached_attention(self._queries(x), cache, tables, lengths, counts=counts, positions=positions, axes=self.axes,
                             causal=causal)
        return self._rest(x, a)
