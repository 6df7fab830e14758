"""Operators of the attention layer around the kernels: head norms with the position rotation,
and sliding-window attention with sinks.

    qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, eps=1e-6, interleaved=True) -> (q, k)
    window_attn(q, k, v, *, left=None, right=0, sinks=0, scale=None, lengths=None, offsets=None,
                return_lse=False) -> out or (out, lse)

and their gradients (``qk_norm_rope_backward``, ``window_attn_backward``). The forward calls
take part in autograd: an input that requires a gradient gets one. Tensors are BTHD as in
``solb200.ops``; everything runs through libsolb200.so on the current CUDA stream, and there is
no CPU path. The reference starts at q, k and v that its host has normed and turned, and has
no gradient and no windowed attention: these have no counterpart there.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from ctypes import c_int32, c_int64
from functools import lru_cache

import torch

from ._lib import I64x2, I64x3, check, lib
from .ops import _SYNC_CHECK, _stream_ptr

# element types as the C ABI numbers them (SOLB200_BF16, _F16, _F32)
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _refuse(what):
    raise RuntimeError(f"solb200: {what}")


def _on(device):
    """A context in which `device` is current."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows16(t, broadcast):
    """`t` itself when its rows can be read with 16-byte accesses in place (a contiguous last
    dimension, base and strides multiples of 16 bytes; with `broadcast`, stride 0 too), else a
    packed copy."""
    step = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0:
        for n, s in zip(t.shape[:-1], t.stride()):
            if n > 1 and (s % step or (s == 0 and not broadcast)):
                break
        else:
            return t
    return t.contiguous(memory_format=torch.contiguous_format) if not t.is_contiguous() else t.clone()


def _bthd(t, name, dtype, device, shape=None):
    if not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor")
    if t.device != device:
        _refuse(f"{name} is on {t.device}, not on {device}")
    if t.dtype != dtype:
        _refuse(f"{name} must be {dtype} (got {t.dtype})")
    if t.dim() != 4:
        _refuse(f"{name} must be BTHD (4-D), got shape {tuple(t.shape)}")
    if shape is not None and t.shape != shape:
        _refuse(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


def _strides(t):
    s = t.stride()
    return I64x3(s[0], s[1], s[2])


# ------------------------------------------------------- head norms and rotation


def _rope_check(q, k, q_weight, k_weight, cos, sin, interleaved):
    """Checked and packed arguments: (q, k, weights, tables, table strides)."""
    if q.dtype not in DTYPES:
        _refuse(f"q must be bfloat16, float16 or float32 (got {q.dtype})")
    _bthd(q, "q", q.dtype, q.device)
    _bthd(k, "k", q.dtype, q.device)
    B, T, H, D = q.shape
    if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
        _refuse(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, tokens or head_dim")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w.shape != (D,) or w.device != q.device:
            _refuse(f"{name} must be one element per channel of a head, [{D}] on {q.device}")
        if w.dtype != q_weight.dtype or w.dtype not in (q.dtype, torch.float32):
            _refuse(f"{name} must be {q.dtype} or float32, both weights alike (got {w.dtype})")
    if cos.shape != sin.shape or cos.dim() not in (2, 3) or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
            or cos.device != q.device or sin.device != q.device:
        _refuse("cos and sin must be float32 [tokens, rotated / 2] or [batch, tokens, rotated / 2], alike, "
                "on the tensors' device")
    if cos.shape[-2] != T or (cos.dim() == 3 and cos.shape[0] != B):
        _refuse(f"cos and sin of shape {tuple(cos.shape)} do not match {B} sequences of {T} tokens")
    R = 2 * cos.shape[-1]
    step = 8 if interleaved else 16
    if D % 8 or not 8 <= D <= 256 or R % step or not step <= R <= D:
        _refuse(f"head_dim {D} must be a multiple of 8 up to 256, and {R} rotated elements a multiple of {step} in it")
    cos, sin = _rows16(cos, True), _rows16(sin, True)
    if cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    ts = I64x2(0, cos.stride(0)) if cos.dim() == 2 else I64x2(cos.stride(0), cos.stride(1))
    return (_rows16(q, True), _rows16(k, True), q_weight.contiguous(), k_weight.contiguous(), cos, sin, ts, R)


def _rope_forward(q, k, q_weight, k_weight, cos, sin, eps, interleaved):
    q, k, wq, wk, cos, sin, ts, R = _rope_check(q, k, q_weight, k_weight, cos, sin, interleaved)
    B, T, H, D = q.shape
    q_out = torch.empty((B, T, H, D), dtype=q.dtype, device=q.device)
    k_out = torch.empty((B, T, k.shape[2], D), dtype=q.dtype, device=q.device)
    if q.numel() and k.numel():
        with _on(q.device):
            check(lib().solb200_qk_norm_rope(
                q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), wq.data_ptr(), wk.data_ptr(), DTYPES[wq.dtype],
                cos.data_ptr(), sin.data_ptr(), ts, q_out.data_ptr(), k_out.data_ptr(), B, T, H, k.shape[2], D, R,
                DTYPES[q.dtype], eps, int(interleaved), _stream_ptr(q.device)), "qk_norm_rope")
    elif q.numel() or k.numel():
        _refuse("q and k must both have heads")
    return q_out, k_out


@lru_cache(maxsize=256)
def _rope_workspace(B, T, H, Hk, D):
    n = c_int64(0)
    check(lib().solb200_qk_norm_rope_backward_workspace(B, T, H, Hk, D, ctypes.byref(n)), "workspace")
    return n.value


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, *, eps=1e-6, interleaved=True):
    """(dq, dk, dq_weight, dk_weight) from the gradients of ``qk_norm_rope``'s outputs and its
    inputs. The weights' gradients are summed in fp32 in a fixed order."""
    q, k, wq, wk, cos, sin, ts, R = _rope_check(q, k, q_weight, k_weight, cos, sin, interleaved)
    _bthd(dq_out, "dq_out", q.dtype, q.device, q.shape)
    _bthd(dk_out, "dk_out", q.dtype, q.device, k.shape)
    dq_out, dk_out = _rows16(dq_out, True), _rows16(dk_out, True)
    B, T, H, D = q.shape
    Hk = k.shape[2]
    dq = torch.empty((B, T, H, D), dtype=q.dtype, device=q.device)
    dk = torch.empty((B, T, Hk, D), dtype=q.dtype, device=q.device)
    if not (q.numel() and k.numel()):
        if q.numel() or k.numel():
            _refuse("q and k must both have heads")
        return dq, dk, torch.zeros_like(wq), torch.zeros_like(wk)
    dw = torch.empty((2, D), dtype=wq.dtype, device=q.device)
    with _on(q.device):
        n = _rope_workspace(B, T, H, Hk, D)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        check(lib().solb200_qk_norm_rope_backward(
            dq_out.data_ptr(), _strides(dq_out), dk_out.data_ptr(), _strides(dk_out), q.data_ptr(), _strides(q),
            k.data_ptr(), _strides(k), wq.data_ptr(), wk.data_ptr(), DTYPES[wq.dtype], cos.data_ptr(), sin.data_ptr(),
            ts, dq.data_ptr(), dk.data_ptr(), dw.data_ptr(), dw.data_ptr() + D * dw.element_size(), B, T, H, Hk, D, R,
            DTYPES[q.dtype], eps, int(interleaved), ws.data_ptr(), n, _stream_ptr(q.device)), "qk_norm_rope_backward")
    return dq, dk, dw[0], dw[1]


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin)
        ctx.how = dict(eps=eps, interleaved=interleaved)
        return _rope_forward(q, k, q_weight, k_weight, cos, sin, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        return (*qk_norm_rope_backward(dq_out, dk_out, *ctx.saved_tensors, **ctx.how), None, None, None, None)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, eps=1e-6, interleaved=True):
    """Root-mean-square norm of every head of q [B, T, H, D] and k [B, T, Hk, D] times its
    weight [D], with the position rotation of the result, in one pass: fresh (q, k) of the same
    dtype (bfloat16, float16 or float32; arithmetic in fp32). ``cos`` / ``sin`` float32 [T, R / 2]
    or [B, T, R / 2] turn the first R elements of each head, (a, b) -> (a cos - b sin, a sin +
    b cos), on the pairs (2i, 2i + 1) if ``interleaved``, else (i, i + R / 2). D: a multiple of 8
    up to 256, R: of 8 (interleaved) or 16. Weights: the tensors' dtype or float32."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad
                                    or k_weight.requires_grad or cos.requires_grad or sin.requires_grad):
        if cos.requires_grad or sin.requires_grad:
            _refuse("cos and sin take no gradient")
        return _NormRope.apply(q, k, q_weight, k_weight, cos, sin, float(eps), bool(interleaved))
    return _rope_forward(q, k, q_weight, k_weight, cos, sin, float(eps), bool(interleaved))


# ------------------------------------------------------------- windowed attention


@lru_cache(maxsize=1024)
def _window_workspace(B, Tq, Tk, H, Hk, D, left, right, sinks, backward):
    n = c_int64(0)
    check(lib().solb200_window_attn_workspace(B, Tq, Tk, H, Hk, D, left, right, sinks, backward, ctypes.byref(n)),
          "window_attn workspace")
    return n.value


def _bound(x, name):
    if x is None:
        return -1
    if x < 0:
        _refuse(f"{name} must be None (no bound) or >= 0, got {x}")
    return int(x)


def _per_sequence(t, name, B, device):
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype != torch.int32 or t.shape != (B,) or t.device != device:
        _refuse(f"{name} must be an int32 tensor of one number per sequence, [{B}] on {device}")
    return t.contiguous()


def _window_check(q, k, v, left, right, sinks, scale, lengths, offsets):
    _bthd(q, "q", torch.bfloat16, q.device)
    _bthd(k, "k", torch.bfloat16, q.device)
    _bthd(v, "v", torch.bfloat16, q.device, k.shape)
    B, Tq, H, D = q.shape
    Bk, Tk, Hk, Dk = k.shape
    if Bk != B or Dk != D:
        _refuse(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch or head_dim")
    if D not in (64, 128):
        _refuse(f"head_dim must be 64 or 128 (got {D})")
    if (H == 0) != (Hk == 0) or (Hk and (H % Hk or H // Hk > 128)):
        _refuse(f"{H} heads are not a multiple of {Hk} key heads (at most 128 times as many)")
    if sinks < 0:
        _refuse(f"sinks must be >= 0, got {sinks}")
    scale = D ** -0.5 if scale is None else float(scale)
    if not scale > 0:
        _refuse(f"scale must be > 0, got {scale}")
    bounds = (_bound(left, "left"), _bound(right, "right"), int(sinks))
    return bounds, scale, _per_sequence(lengths, "lengths", B, q.device), _per_sequence(offsets, "offsets", B, q.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _device_error(ws, what):
    code = c_int32(0)
    check(lib().solb200_read_device_error(ws.data_ptr(), ctypes.byref(code), _stream_ptr(ws.device)), what)


def _window_forward(q, k, v, left, right, sinks, scale, lengths, offsets, want_lse):
    bounds, scale, lengths, offsets = _window_check(q, k, v, left, right, sinks, scale, lengths, offsets)
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    if not (q.numel() and k.numel()):      # no queries, or no keys for them to see
        out = torch.zeros((B, Tq, H, D), dtype=q.dtype, device=q.device)
        return out, torch.full((B, H, Tq), -torch.inf, device=q.device) if want_lse else None
    q, k, v = _rows16(q, False), _rows16(k, False), _rows16(v, False)
    with _on(q.device):
        out = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device)
        lse = torch.empty((B, H, Tq), dtype=torch.float32, device=q.device) if want_lse else None
        n = _window_workspace(B, Tq, Tk, H, Hk, D, *bounds, 0)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        check(lib().solb200_window_attn(
            q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), out.data_ptr(),
            _ptr(lse), _ptr(lengths), _ptr(offsets), B, Tq, Tk, H, Hk, D, *bounds, scale, ws.data_ptr(), n,
            _stream_ptr(q.device)), "window_attn")
        if _SYNC_CHECK:
            _device_error(ws, "window_attn device error check")
    return out, lse


def window_attn_backward(dout, q, k, v, out, lse, *, left=None, right=0, sinks=0, scale=None, lengths=None,
                         offsets=None):
    """(dq, dk, dv) from the gradient of ``window_attn``'s output, its inputs, its output and
    its log-sum-exp (``return_lse``), with the same bounds. Sums are in a fixed order. ``q`` and
    ``dout`` have to be finite in every row, the rows of queries that see nothing included."""
    bounds, scale, lengths, offsets = _window_check(q, k, v, left, right, sinks, scale, lengths, offsets)
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    _bthd(dout, "dout", q.dtype, q.device, q.shape)
    _bthd(out, "out", q.dtype, q.device, q.shape)
    if lse.shape != (B, H, Tq) or lse.dtype != torch.float32 or lse.device != q.device:
        _refuse(f"lse must be float32 [{B}, {H}, {Tq}] on {q.device}")
    if not (q.numel() and k.numel()):
        return tuple(torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    q, k, v, dout, out = (_rows16(t, False) for t in (q, k, v, dout, out))
    lse = lse.contiguous()
    with _on(q.device):
        dq = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device)
        dk = torch.empty((B, Tk, Hk, D), dtype=q.dtype, device=q.device)
        dv = torch.empty((B, Tk, Hk, D), dtype=q.dtype, device=q.device)
        n = _window_workspace(B, Tq, Tk, H, Hk, D, *bounds, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        check(lib().solb200_window_attn_backward(
            dout.data_ptr(), _strides(dout), q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(),
            _strides(v), out.data_ptr(), _strides(out), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            _ptr(lengths), _ptr(offsets), B, Tq, Tk, H, Hk, D, *bounds, scale, ws.data_ptr(), n,
            _stream_ptr(q.device)), "window_attn_backward")
        if _SYNC_CHECK:
            _device_error(ws, "window_attn_backward device error check")
    return dq, dk, dv


class _WindowAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, left, right, sinks, scale, lengths, offsets):
        out, lse = _window_forward(q, k, v, left, right, sinks, scale, lengths, offsets, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths, offsets)
        ctx.how = dict(left=left, right=right, sinks=sinks, scale=scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, out, lse, lengths, offsets = ctx.saved_tensors
        grads = window_attn_backward(dout, q, k, v, out, lse, lengths=lengths, offsets=offsets, **ctx.how)
        return (*grads, None, None, None, None, None, None)


def window_attn(q, k, v, *, left=None, right=0, sinks=0, scale=None, lengths=None, offsets=None, return_lse=False):
    """Attention in a sliding window with a few first keys that stay visible: query i of
    sequence b sits at p = offsets[b] + i and sees key j when j < lengths[b], j <= p + right and
    (j >= p - left or j < sinks). ``left`` / ``right`` None: no bound; right 0 is causal, and
    holds for the sinks too. q bf16 [B, Tq, H, D], k / v bf16 [B, Tk, Hk, D], D 64 or 128, H a
    multiple of Hk; ``lengths`` / ``offsets`` int32 [B] on the device (defaults: Tk, and the last
    query at the last key), so a cache's lengths need no host copy. Keys past a length may hold
    anything. Returns a fresh bf16 tensor like q (zeros for a query that sees nothing), and with
    ``return_lse`` also float32 [B, H, Tq], the logarithm of each row's sum (-inf there; it takes
    no gradient)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttn.apply(q, k, v, left, right, sinks, scale, lengths, offsets)
    else:
        out, lse = _window_forward(q, k, v, left, right, sinks, scale, lengths, offsets, return_lse)
    return (out, lse) if return_lse else out
