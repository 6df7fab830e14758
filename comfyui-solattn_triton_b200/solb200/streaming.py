"""A self-attention layer of a streamed video (or causal text) model on the layer operators:
projection, head norms with the rotation (``qk_norm_rope``), attention in a sliding window with
the first tokens kept visible (``window_attn``), projection.

    layer = StreamingSelfAttention(dim=5120, heads=40, left=3 * 1560, sinks=1560).cuda().bfloat16()
    y = layer(x, cos, sin)                      # a whole sequence (training, or a prompt)
    cache = layer.new_cache(batch, capacity)
    y = layer(chunk, cos, sin, cache=cache)     # the next tokens: a frame, or a single token

A chunk's tokens see the chunk, the window before it and the sinks. With ``cache`` the new keys
and values are written behind each sequence's length, which stays on the device: a step makes no
host copy. ``lengths`` of ragged sequences (right-padded) may be set on the cache. A call with a
cache is inference: it records nothing for a gradient, and refuses an input that requires one.
"""

from __future__ import annotations

import torch

from .layer_ops import qk_norm_rope, window_attn


class KVCache:
    """Keys and values of ``capacity`` tokens per sequence, and how many of them are filled
    (``lengths``, int32 [B] on the device; they may be set, or changed in place)."""

    def __init__(self, batch, capacity, heads, head_dim, device):
        self.k = torch.empty((batch, capacity, heads, head_dim), dtype=torch.bfloat16, device=device)
        self.v = torch.empty_like(self.k)
        with torch.inference_mode(False):      # (a tensor whose changes are counted in every mode)
            self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self._rows = torch.arange(batch, device=device)[:, None]
        self._captured = False                 # replays of a captured call change the lengths uncounted
        self._at_most(0)

    def _at_most(self, n):
        """No sequence is longer than n as long as the lengths are this tensor, unchanged."""
        self._most, self._of = n, self.lengths
        self._version = None if self.lengths.is_inference() else self.lengths._version

    def _counted(self):
        return (not self._captured and self._of is self.lengths and self._version is not None
                and self._version == self.lengths._version)

    def append(self, k, v):
        """Write k / v [B, T, heads, head_dim] behind each sequence's length; what does not fit the
        capacity is refused. The lengths are read back for that only where the tokens appended so
        far could exceed it, or the lengths were changed by someone else. A captured call reads
        nothing: its tokens past the capacity land on the last place. The cache takes the values
        alone: no gradient goes through it."""
        T, capacity = k.shape[1], self.k.shape[1]
        capturing = self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()
        self._captured = self._captured or capturing
        if self.lengths.numel() and T and not capturing:
            if not self._counted() or self._most + T > capacity:
                self._at_most(int(self.lengths.max()))
            if self._most + T > capacity:
                raise RuntimeError(f"solb200: {T} tokens behind {self._most} do not fit a cache of {capacity}")
        elif T > capacity:
            raise RuntimeError(f"solb200: {T} tokens do not fit a cache of {capacity}")
        # (an index outside the cache would be a device assertion)
        at = (self.lengths[:, None] + torch.arange(T, device=k.device)).clamp_(0, capacity - 1)
        self.k[self._rows, at] = k.detach()
        self.v[self._rows, at] = v.detach()
        self.lengths += T
        self._at_most(self._most + T)


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
        if cache is not None and torch.is_grad_enabled():
            if x.requires_grad:
                raise RuntimeError("solb200: a call with a cache takes no gradient, and its input requires one; "
                                   "make it under torch.no_grad()")
            with torch.no_grad():
                return self.forward(x, cos, sin, cache)
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
