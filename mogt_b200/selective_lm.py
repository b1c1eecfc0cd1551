"""A small language model of selective state space blocks, in the three forms
that a program uses it in: over training batches, over prompts, token by token.

``SelectiveBlock`` has the calling convention of ``backbone.MOGTBlock``
(``block(x, prefix_condition=None)``), so both kinds can be stacked in one
``MOGTModel.blocks``.  A block is

    x, z = in_proj(norm(h));  u = silu(causal_conv(x))
    delta, B, C = x_proj(u);  y = selective_scan(u, dt_proj(delta), A, B, C, D, z)
    h + out_proj(y)

and keeps, per sequence, the last K-1 convolution inputs and the scan's
[channels, N] state: a generation's memory does not grow with its length.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .backbone import RMSNorm
from .selective import causal_conv, causal_conv_step, selective_scan, selective_scan_step

__all__ = ["SelectiveBlock", "SelectiveLM"]


class SelectiveBlock(nn.Module):
    def __init__(self, d_model: int, *, d_state: int = 16, conv_taps: int = 4, expand: int = 2, rank: int | None = None):
        super().__init__()
        self.d_inner, self.d_state, self.taps = expand * d_model, d_state, conv_taps
        self.rank = rank or math.ceil(d_model / 16)
        di = self.d_inner
        self.norm = RMSNorm(d_model)
        self.in_proj = nn.Linear(d_model, 2 * di, bias=False)
        self.conv_weight = nn.Parameter(torch.randn(di, conv_taps) / math.sqrt(conv_taps))
        self.conv_bias = nn.Parameter(torch.zeros(di))
        self.x_proj = nn.Linear(di, self.rank + 2 * d_state, bias=False)
        self.dt_proj = nn.Linear(self.rank, di, bias=False)
        # steps spread over [1e-3, 1e-1], decays -1 .. -d_state
        step = torch.exp(torch.rand(di) * math.log(100.0) + math.log(1e-3))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1).float()).repeat(di, 1))
        self.D = nn.Parameter(torch.ones(di))
        self.out_proj = nn.Linear(di, d_model, bias=False)

    def _split(self, u):
        dbc = self.x_proj(u)
        delta, B, C = dbc.split([self.rank, self.d_state, self.d_state], -1)
        return self.dt_proj(delta), -torch.exp(self.A_log.float()), B, C

    def _mix(self, x, lengths=None, cache=None, return_cache=False):
        xz = self.in_proj(self.norm(x))
        conv_state, state = cache if cache is not None else (None, None)
        u = causal_conv(xz[..., :self.d_inner], self.conv_weight, self.conv_bias, initial_state=conv_state,
                        lengths=lengths, return_state=return_cache)
        if return_cache:
            u, conv_state = u
        delta, A, B, C = self._split(u)
        y = selective_scan(u, delta, A, B, C, D=self.D, z=xz[..., self.d_inner:], delta_bias=self.dt_bias,
                           delta_softplus=True, initial_state=state, lengths=lengths, return_state=return_cache)
        if return_cache:
            y, state = y
        return x + self.out_proj(y), (conv_state, state)

    def forward(self, x, prefix_condition=None):
        """x: [B, L, d_model].  prefix_condition is MOGTBlock's, not used here."""
        return self._mix(x)[0]

    def prefill(self, x, lengths=None, cache=None):
        """As forward, from `cache` (default: nothing before x); returns (out,
        cache after each sequence's last token)."""
        return self._mix(x, lengths, cache, True)

    def step(self, x, cache):
        """One token per sequence, x: [B, d_model]; updates the cache in place."""
        conv_state, state = cache
        xz = self.in_proj(self.norm(x))
        u = causal_conv_step(xz[..., :self.d_inner], conv_state, self.conv_weight, self.conv_bias)
        delta, A, B, C = self._split(u)
        y = selective_scan_step(state, u, delta, A, B, C, D=self.D, z=xz[..., self.d_inner:],
                                delta_bias=self.dt_bias, delta_softplus=True)
        return x + self.out_proj(y)


class SelectiveLM(nn.Module):
    """Embedding, blocks, final norm, head tied to the embedding."""

    def __init__(self, vocab_size: int, d_model: int = 768, num_layers: int = 12, **block):
        super().__init__()
        self.embedding = nn.Embedding(vocab_size, d_model)
        nn.init.normal_(self.embedding.weight, std=0.02)
        self.blocks = nn.ModuleList([SelectiveBlock(d_model, **block) for _ in range(num_layers)])
        self.norm_f = RMSNorm(d_model)

    def _head(self, x):
        return F.linear(self.norm_f(x), self.embedding.weight)

    def forward(self, input_ids):
        """Logits [B, L, vocab] of the token after each position."""
        x = self.embedding(input_ids)
        for blk in self.blocks:
            x = blk(x)
        return self._head(x)

    @torch.no_grad()
    def prefill(self, input_ids, lengths=None):
        """Logits after each prompt's last token [B, vocab], and the caches.
        lengths are clamped to [0, L] as in the operators; a prompt without
        tokens has all logits 0."""
        B, L = input_ids.shape
        x = self.embedding(input_ids)
        caches = []
        for blk in self.blocks:
            x, cache = blk.prefill(x, lengths)
            caches.append(cache)
        if L == 0:
            x = x.new_zeros(B, x.shape[-1])
        elif lengths is None:
            x = x[:, -1]
        else:
            n = lengths.long().clamp(0, L)
            x = x[torch.arange(B, device=x.device), (n - 1).clamp(min=0)]
            x = torch.where((n > 0)[:, None], x, 0.0)
        return self._head(x), caches

    @torch.no_grad()
    def step(self, tokens, caches):
        """Logits after one more token per sequence, tokens: [B]."""
        x = self.embedding(tokens)
        for blk, cache in zip(self.blocks, caches):
            x = blk.step(x, cache)
        return self._head(x)
