"""A self-attention layer of a streamed video (or causal text) model on the layer operators:
projection, head norms with the rotation (``qk_norm_rope``), attention in a sliding window with
the first tokens kept visible (``window_attn``), projection.

    layer = StreamingSelfAttention(dim=5120, heads=40, left=3 * 1560, sinks=1560).cuda().bfloat16()
    y = layer(x, cos, sin)                      # a whole sequence (training, or a prompt)
    cache = layer.new_cache(batch, capacity)
    y = layer(chunk, cos, sin, cache=cache)     # the next tokens: a frame, or a single token

A chunk's tokens see the chunk, the window before it and the sinks. With ``cache`` the new keys
and values are written behind each sequence's length, which stays on the device: a step makes no
host copy. ``lengths`` of ragged sequences (right-padded) may be set on the cache.
"""

from __future__ import annotations

import torch

from .layer_ops import qk_norm_rope, window_attn


class KVCache:
    """Keys and values of ``capacity`` tokens per sequence, and how many of them are filled
    (``lengths``, int32 [B] on the device)."""

    def __init__(self, batch, capacity, heads, head_dim, device):
        self.k = torch.empty((batch, capacity, heads, head_dim), dtype=torch.bfloat16, device=device)
        self.v = torch.empty_like(self.k)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._rows = torch.arange(batch, device=device)[:, None]

    def append(self, k, v):
        """Write k / v [B, T, heads, head_dim] behind each sequence's length. The caller keeps the
        length within the capacity (an index past it is an error of the index operation)."""
        at = self.lengths[:, None].long() + torch.arange(k.shape[1], device=k.device)
        self.k[self._rows, at] = k
        self.v[self._rows, at] = v
        self.lengths += k.shape[1]


class StreamingSelfAttention(torch.nn.Module):
    """``left`` / ``right`` / ``sinks`` as in ``window_attn``; ``kv_heads`` fewer key heads than
    query heads; ``interleaved`` as in ``qk_norm_rope``."""

    def __init__(self, dim, heads, *, kv_heads=None, head_dim=128, left=None, right=0, sinks=0, eps=1e-6,
                 interleaved=True):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, heads if kv_heads is None else kv_heads, head_dim
        self.window = dict(left=left, right=right, sinks=sinks)
        self.eps, self.interleaved = eps, interleaved
        self.qkv = torch.nn.Linear(dim, (heads + 2 * self.kv_heads) * head_dim, bias=False)
        self.out = torch.nn.Linear(heads * head_dim, dim, bias=False)
        self.q_norm = torch.nn.Parameter(torch.ones(head_dim))
        self.k_norm = torch.nn.Parameter(torch.ones(head_dim))

    def new_cache(self, batch, capacity):
        return KVCache(batch, capacity, self.kv_heads, self.head_dim, self.qkv.weight.device)

    def forward(self, x, cos, sin, cache=None):
        B, T, _ = x.shape
        qkv = self.qkv(x).view(B, T, -1, self.head_dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        q, k = qk_norm_rope(q, k, self.q_norm, self.k_norm, cos, sin, eps=self.eps, interleaved=self.interleaved)
        if cache is None:
            a = window_attn(q, k, v, **self.window)
        else:
            cache.append(k, v)
            a = window_attn(q, cache.k, cache.v, lengths=cache.lengths, **self.window)
        return self.out(a.reshape(B, T, -1))
