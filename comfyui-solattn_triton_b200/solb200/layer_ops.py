"""Operators of the attention layer around the kernels: head norms with the position rotation,
and sliding-window attention with sinks.

    qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, eps=1e-6, interleaved=True) -> (q, k)
    window_attn(q, k, v, *, left=None, right=0, sinks=0, scale=None, lengths=None, offsets=None,
                return_lse=False) -> out or (out, lse)

and their gradients (``qk_norm_rope_backward``, ``window_attn_backward``). The forward calls
take part in autograd: an input that requires a gradient gets one (reverse mode; a tangent is
refused). Tensors are BTHD as in ``solb200.ops``; everything runs through libsolb200.so on the
current CUDA stream, and there is no CPU path. The reference starts at q, k and v that its host has normed and turned, and has
no gradient and no windowed attention: these have no counterpart there.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from ctypes import c_float, c_int32, c_int64
from types import SimpleNamespace

import torch
from torch.autograd import forward_ad

from ._lib import I64x2, I64x3, check, lib
from .ops import _SYNC_CHECK

# element types as the C ABI numbers them (SOLB200_BF16, _F16, _F32)
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _refuse(what):
    raise RuntimeError(f"solb200: {what}")


_HERE = nullcontext()
_device_now = torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream     # the current stream's handle, by device index


def _on(index):
    """A context in which device `index` is current."""
    return _HERE if index == _device_now() else torch.cuda.device(index)


# What a call's shapes, strides, types and options determine (the checks passed, output shapes,
# stride arrays, workspace sizes), by those alone: a repeated geometry skips the checks.
_PLANS = {}


def _plan(key, make, *args):
    plan = _PLANS.get(key)
    if plan is None:
        plan = make(*args)
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        _PLANS[key] = plan
    return plan


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


def _numbers(**named):
    # (a tensor's value could change under a plan kept for it)
    for name, x in named.items():
        if torch.is_tensor(x):
            _refuse(f"{name} must be a number, not a tensor")


def _no_tangents(*tensors):
    """Refuse forward-mode derivatives: the kernels read values only, a tangent would be dropped."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if torch.is_tensor(t) and forward_ad.unpack_dual(t).tangent is not None:
                _refuse("a tensor has a tangent: forward-mode derivatives are not supported")


def _fresh(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _strides(t):
    s = t.stride()
    return I64x3(s[0], s[1], s[2])


def _dense(B, T, H, D):
    return I64x3(T * H * D, H * D, D)


def _readable(t, dense, broadcast):
    """(tensor, strides) of `t` as the kernels can read it; `dense`: the strides of a packed one
    (head_dim is a multiple of 16 bytes)."""
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t, dense
    t = _rows16(t, broadcast)
    return t, _strides(t)


def _in_place(t, broadcast):
    """Whether `t`'s rows can be read with 16-byte accesses where they lie, its base aside."""
    step = 16 // t.element_size()
    return t.stride(-1) == 1 and not any(n > 1 and (s % step or (s == 0 and not broadcast))
                                         for n, s in zip(t.shape[:-1], t.stride()))


# ------------------------------------------------------- head norms and rotation


def _rope_plan(q, k, q_weight, k_weight, cos, sin, eps, interleaved):
    _numbers(eps=eps, interleaved=interleaved)
    if q.dtype not in DTYPES:
        _refuse(f"q must be bfloat16, float16 or float32 (got {q.dtype})")
    _bthd(q, "q", q.dtype, q.device)
    _bthd(k, "k", q.dtype, q.device)
    B, T, H, D = q.shape
    Hk = k.shape[2]
    if k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
        _refuse(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, tokens or head_dim")
    if (H == 0) != (Hk == 0):
        _refuse("q and k must both have heads")
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
    if not eps >= 0:
        _refuse(f"eps must be >= 0, got {eps}")
    n = c_int64(0)
    if B and T and H:
        check(lib().solb200_qk_norm_rope_backward_workspace(B, T, H, Hk, D, ctypes.byref(n)), "workspace")
    return SimpleNamespace(
        place=(c_int64(B), c_int64(T), c_int64(H), c_int64(Hk), c_int64(D), c_int64(R), c_int32(DTYPES[q.dtype]),
               c_float(eps), c_int32(bool(interleaved))), empty=not (B and T and H),
        wtype=DTYPES[q_weight.dtype], qs=_strides(q), ks=_strides(k), backward_bytes=n.value,
        dense_q=_dense(B, T, H, D), dense_k=_dense(B, T, Hk, D),
        ts=I64x2(0, cos.stride(0)) if cos.dim() == 2 else I64x2(cos.stride(0), cos.stride(1)),
        in_place=(_in_place(q, True) and _in_place(k, True) and _in_place(cos, True) and cos.stride() == sin.stride()
                  and q_weight.is_contiguous() and k_weight.is_contiguous()))


def _rope_inputs(q, k, q_weight, k_weight, cos, sin, eps, interleaved):
    """(plan, tensors): the tensors as the kernels can read them, packed where they have to be."""
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(),
           q_weight.shape, q_weight.stride(), q_weight.dtype, q_weight.get_device(), k_weight.shape,
           k_weight.stride(), k_weight.dtype, k_weight.get_device(), cos.shape, cos.stride(), cos.dtype,
           cos.get_device(), sin.shape, sin.stride(), sin.dtype, sin.get_device(), eps, interleaved)
    plan = _PLANS.get(key) or _plan(key, _rope_plan, q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    if plan.in_place and not (q.data_ptr() | k.data_ptr() | cos.data_ptr() | sin.data_ptr()) & 15:
        return plan, q, k, q_weight, k_weight, cos, sin
    q, k, q_weight, k_weight = _rows16(q, True), _rows16(k, True), q_weight.contiguous(), k_weight.contiguous()
    cos, sin = _rows16(cos, True), _rows16(sin, True)
    if cos.stride() != sin.stride():
        cos, sin = _rows16(cos.contiguous(), True), _rows16(sin.contiguous(), True)
    return _rope_plan(q, k, q_weight, k_weight, cos, sin, eps, interleaved), q, k, q_weight, k_weight, cos, sin


def _rope_forward(q, k, q_weight, k_weight, cos, sin, eps, interleaved):
    plan, q, k, wq, wk, cos, sin = _rope_inputs(q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    q_out, k_out = _fresh(q), _fresh(k)
    if not plan.empty:
        index = q.get_device()
        with _on(index):
            rc = lib().solb200_qk_norm_rope(
                q.data_ptr(), plan.qs, k.data_ptr(), plan.ks, wq.data_ptr(), wk.data_ptr(), plan.wtype, cos.data_ptr(),
                sin.data_ptr(), plan.ts, q_out.data_ptr(), k_out.data_ptr(), *plan.place, _raw_stream(index))
        if rc:
            check(rc, "qk_norm_rope")
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin, *, eps=1e-6, interleaved=True):
    """(dq, dk, dq_weight, dk_weight) from the gradients of ``qk_norm_rope``'s outputs and its
    inputs. The weights' gradients are summed in fp32 in a fixed order."""
    _no_tangents(dq_out, dk_out, q, k, q_weight, k_weight, cos, sin)
    plan, q, k, wq, wk, cos, sin = _rope_inputs(q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    for g, x, name in ((dq_out, q, "dq_out"), (dk_out, k, "dk_out")):
        if g.shape != x.shape or g.dtype != x.dtype or g.get_device() != x.get_device():
            _bthd(g, name, x.dtype, x.device, x.shape)
    dq_out, dqs = _readable(dq_out, plan.dense_q, True)
    dk_out, dks = _readable(dk_out, plan.dense_k, True)
    dq, dk = _fresh(q), _fresh(k)
    if plan.empty:
        return dq, dk, torch.zeros_like(wq), torch.zeros_like(wk)
    dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
    index = q.get_device()
    with _on(index):
        ws = torch.empty(plan.backward_bytes, dtype=torch.uint8, device=q.device)
        rc = lib().solb200_qk_norm_rope_backward(
            dq_out.data_ptr(), dqs, dk_out.data_ptr(), dks, q.data_ptr(), plan.qs,
            k.data_ptr(), plan.ks, wq.data_ptr(), wk.data_ptr(), plan.wtype, cos.data_ptr(), sin.data_ptr(), plan.ts,
            dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(), *plan.place, ws.data_ptr(),
            plan.backward_bytes, _raw_stream(index))
    if rc:
        check(rc, "qk_norm_rope_backward")
    return dq, dk, dwq, dwk


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
    _no_tangents(q, k, q_weight, k_weight, cos, sin)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad
                                    or k_weight.requires_grad or cos.requires_grad or sin.requires_grad):
        if cos.requires_grad or sin.requires_grad:
            _refuse("cos and sin take no gradient")
        return _NormRope.apply(q, k, q_weight, k_weight, cos, sin, eps, interleaved)
    return _rope_forward(q, k, q_weight, k_weight, cos, sin, eps, interleaved)


# ------------------------------------------------------------- windowed attention


def _bound(x, name):
    if x is None:
        return -1
    if x < 0:
        _refuse(f"{name} must be None (no bound) or >= 0, got {x}")
    return min(int(x), 1 << 40)                # past every position


def _window_plan(q, k, v, left, right, sinks, scale):
    _numbers(left=left, right=right, sinks=sinks, scale=scale)
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
    bounds = (_bound(left, "left"), _bound(right, "right"), min(int(sinks), 1 << 40))
    empty = not (B and Tq and Tk and H)
    n = [c_int64(0), c_int64(0)]
    if not empty:
        for backward in (0, 1):
            check(lib().solb200_window_attn_workspace(B, Tq, Tk, H, Hk, D, *bounds, backward,
                                                      ctypes.byref(n[backward])), "window_attn workspace")
    return SimpleNamespace(place=(*map(c_int64, (B, Tq, Tk, H, Hk, D, *bounds)), c_float(scale)), empty=empty, bytes=n[0].value,
                           backward_bytes=n[1].value, qs=_strides(q), ks=_strides(k), vs=_strides(v),
                           dense_q=_dense(B, Tq, H, D),
                           in_place=_in_place(q, False) and _in_place(k, False) and _in_place(v, False))


def _window_inputs(q, k, v, left, right, sinks, scale, lengths, offsets):
    """(plan, tensors, pointers of lengths and offsets): the tensors as the kernels can read them."""
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), v.shape,
           v.stride(), v.dtype, v.get_device(), left, right, sinks, scale)
    plan = _PLANS.get(key) or _plan(key, _window_plan, q, k, v, left, right, sinks, scale)
    per_sequence = []
    for t, name in ((lengths, "lengths"), (offsets, "offsets")):
        if t is None:
            per_sequence.append(None)
            continue
        if not torch.is_tensor(t) or t.dtype != torch.int32 or t.shape != q.shape[:1] or t.device != q.device:
            _refuse(f"{name} must be an int32 tensor of one number per sequence, [{q.shape[0]}] on {q.device}")
        per_sequence.append(t.contiguous())
    if not plan.in_place or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v = _rows16(q, False), _rows16(k, False), _rows16(v, False)
        plan = _window_plan(q, k, v, left, right, sinks, scale)
    return plan, q, k, v, *per_sequence


def _ptr(t):
    return None if t is None else t.data_ptr()


def _device_error(ws, stream, what):
    code = c_int32(0)
    check(lib().solb200_read_device_error(ws.data_ptr(), ctypes.byref(code), stream), what)


# The device error word of calls that need no other workspace, by device and stream: calls of one
# stream run one after the other, and each clears it first. A captured call takes a word of its
# own (the graph's memory): its replays may run on another stream beside plain calls.
_ERROR_WORDS = {}


def _workspace(nbytes, q, index, stream):
    if nbytes > 256 or torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    ws = _ERROR_WORDS.get((index, stream))
    if ws is None:
        ws = _ERROR_WORDS[(index, stream)] = torch.empty(256, dtype=torch.uint8, device=q.device)
    return ws


def _window_forward(q, k, v, left, right, sinks, scale, lengths, offsets, want_lse):
    plan, q, k, v, lengths, offsets = _window_inputs(q, k, v, left, right, sinks, scale, lengths, offsets)
    B, Tq, H, _ = q.shape
    if plan.empty:      # no queries, or no keys for them to see
        lse = torch.full((B, H, Tq), -torch.inf, dtype=torch.float32, device=q.device) if want_lse else None
        return q.new_zeros(q.shape), lse
    index = q.get_device()
    with _on(index):
        out = _fresh(q)
        lse = torch.empty((B, H, Tq), dtype=torch.float32, device=q.device) if want_lse else None
        stream = _raw_stream(index)
        ws = _workspace(plan.bytes, q, index, stream)
        rc = lib().solb200_window_attn(
            q.data_ptr(), plan.qs, k.data_ptr(), plan.ks, v.data_ptr(), plan.vs, out.data_ptr(), _ptr(lse),
            _ptr(lengths), _ptr(offsets), *plan.place, ws.data_ptr(), plan.bytes, stream)
        if rc:
            check(rc, "window_attn")
        if _SYNC_CHECK:
            _device_error(ws, stream, "window_attn device error check")
    return out, lse


def window_attn_backward(dout, q, k, v, out, lse, *, left=None, right=0, sinks=0, scale=None, lengths=None,
                         offsets=None):
    """(dq, dk, dv) from the gradient of ``window_attn``'s output, its inputs, its output and
    its log-sum-exp (``return_lse``), with the same bounds. Sums are in a fixed order. ``q`` and
    ``dout`` of queries that see nothing may hold anything (their dq is zero)."""
    _no_tangents(dout, q, k, v, out, lse)
    plan, q, k, v, lengths, offsets = _window_inputs(q, k, v, left, right, sinks, scale, lengths, offsets)
    B, Tq, H, _ = q.shape
    for t, name in ((dout, "dout"), (out, "out")):
        if t.shape != q.shape or t.dtype != q.dtype or t.get_device() != q.get_device():
            _bthd(t, name, q.dtype, q.device, q.shape)
    if lse.shape != (B, H, Tq) or lse.dtype != torch.float32 or lse.device != q.device:
        _refuse(f"lse must be float32 [{B}, {H}, {Tq}] on {q.device}")
    if plan.empty:
        return tuple(t.new_zeros(t.shape) for t in (q, k, v))
    dout, dos = _readable(dout, plan.dense_q, False)
    out, outs = _readable(out, plan.dense_q, False)
    lse = lse.contiguous()
    index = q.get_device()
    with _on(index):
        dq, dk, dv = _fresh(q), _fresh(k), _fresh(v)
        ws = torch.empty(plan.backward_bytes, dtype=torch.uint8, device=q.device)
        stream = _raw_stream(index)
        rc = lib().solb200_window_attn_backward(
            dout.data_ptr(), dos, q.data_ptr(), plan.qs, k.data_ptr(), plan.ks, v.data_ptr(), plan.vs,
            out.data_ptr(), outs, lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            _ptr(lengths), _ptr(offsets), *plan.place, ws.data_ptr(), plan.backward_bytes, stream)
        if rc:
            check(rc, "window_attn_backward")
        if _SYNC_CHECK:
            _device_error(ws, stream, "window_attn_backward device error check")
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
    _no_tangents(q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out, lse = _WindowAttn.apply(q, k, v, left, right, sinks, scale, lengths, offsets)
    else:
        out, lse = _window_forward(q, k, v, left, right, sinks, scale, lengths, offsets, return_lse)
    return (out, lse) if return_lse else out
