"""CellReader: positions of one channels-last map, or tokens of a model, read another map's states by cross attention,
then go through a two-layer perceptron, both with residuals:

    x + out(attention(q(norm(x)), k(states), v(states)))     then     x + fc2(gelu(fc1(norm(x))))

on the operators of feature_ops (group norm, products with their bias, activation and residual in the epilogue, attention
over states of another length). The output projections start at zero, so a new reader is the identity. The encoder uses it
for its fine cells (efficient_encoder.py, `fine_reader_heads`); on its own it lets a few query tokens read the latents of
all splats of an image (EfficientGaussianEncoder.gather_splat_latents). The reference has no counterpart."""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .feature_ops import cross_attention, group_norm_act, linear_act


class CellReader(nn.Module):
    """channels: of x; state_channels: of the states; heads, kv_heads: query heads and the key heads that they share (all
    their own by default); groups: of the norms, whose statistics run over all positions of an image; hidden: the
    perceptron's width (twice the channels by default)."""

    def __init__(self, channels, state_channels, heads=4, kv_heads=None, head_dim=None, groups=8, hidden=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads do not divide over {kv_heads} key heads")
        if head_dim is None:
            if channels % heads:
                raise ValueError(f"{channels} channels do not divide into {heads} heads: give head_dim")
            head_dim = channels // heads
        hidden = 2 * channels if hidden is None else hidden
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm1 = nn.GroupNorm(groups, channels)
        self.to_q = nn.Linear(channels, heads * head_dim)
        self.to_kv = nn.Linear(state_channels, 2 * kv_heads * head_dim)
        self.to_out = nn.Linear(heads * head_dim, channels)
        self.norm2 = nn.GroupNorm(groups, channels)
        self.fc1 = nn.Linear(channels, hidden)
        self.fc2 = nn.Linear(hidden, channels)
        for m in (self.to_out, self.fc2):
            nn.init.zeros_(m.weight)
            nn.init.zeros_(m.bias)

    @staticmethod
    def _norm(x, norm):
        return group_norm_act(x, norm.num_groups, norm.weight, norm.bias, norm.eps, act="none")

    @staticmethod
    def _product(x, layer, act="none", residual=None):
        """The layer's product in x's type (float32 weights are rounded for bfloat16 features)."""
        return linear_act(x, layer.weight.to(x.dtype), layer.bias.to(x.dtype), act=act, residual=residual)

    @staticmethod
    def _tokens(t):
        """Images and tokens of an image of t [B, ..., C]."""
        return t.shape[0], math.prod(t.shape[1:-1])

    def keys_values(self, states):
        """[B, Lk, 2, kv_heads, head_dim] of states [B, ..., state_channels]: what a program keeps where many calls read
        the same states (forward's `kv`)."""
        kv = self._product(states, self.to_kv)
        return kv.reshape(self._tokens(states) + (2, self.kv_heads, self.head_dim))

    def forward(self, x, states=None, kv_lengths=None, key_mask=None, kv=None):
        """x [B, ..., channels], states [B, ..., state_channels] (or kv from keys_values) -> like x. kv_lengths [B] and
        key_mask [B, Lk] leave states out; where none is left the attention adds its projection's bias alone."""
        if (states is None) == (kv is None):
            raise ValueError("either states or kv is needed")
        if kv is None:
            kv = self.keys_values(states)
        q = self._product(self._norm(x, self.norm1), self.to_q)
        q = q.reshape(self._tokens(x) + (self.heads, self.head_dim))
        a = cross_attention(q, kv[:, :, 0], kv[:, :, 1], kv_lengths=kv_lengths, key_mask=key_mask)
        x = self._product(a.reshape(x.shape[:-1] + (self.heads * self.head_dim,)), self.to_out, residual=x)
        return self._product(self._product(self._norm(x, self.norm2), self.fc1, act="gelu"), self.fc2, residual=x)
