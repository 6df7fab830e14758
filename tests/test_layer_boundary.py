"""The layer operators' refusals that need no GPU: status codes of the C ABI's planning calls,
and the Python layer's refusal of host tensors."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import solb200
from solb200 import _lib


def _window_bytes(*args, backward=0):
    n = ctypes.c_int64(-1)
    return _lib.lib().solb200_window_attn_workspace(*args, backward, ctypes.byref(n)), n.value


@pytest.mark.parametrize("args", [
    (0, 4, 4, 2, 2, 64, -1, 0, 0),            # no sequence
    (1, 0, 4, 2, 2, 64, -1, 0, 0),            # no query
    (1, 4, 0, 2, 2, 64, -1, 0, 0),            # no key
    (1, 4, 4, 2, 2, 96, -1, 0, 0),            # head_dim
    (1, 4, 4, 3, 2, 64, -1, 0, 0),            # heads not a multiple
    (1, 4, 4, 258, 2, 64, -1, 0, 0),          # more than 128 heads per key head
    (1, 4, 4, 2, 2, 64, -2, 0, 0),            # bounds
    (1, 4, 4, 2, 2, 64, -1, -2, 0),
    (1, 4, 4, 2, 2, 64, -1, 0, -1),           # sinks
    (1, 1 << 31, 4, 2, 2, 64, -1, 0, 0),      # lengths
    (1, 4, 1 << 31, 2, 2, 64, -1, 0, 0),
])
def test_window_plan_refuses(args):
    rc, n = _window_bytes(*args)
    assert rc == 1 and n == -1 and _lib.last_error()


def test_window_plan_splits_only_where_tiles_are_few():
    rc, whole = _window_bytes(1, 32760, 32760, 40, 40, 128, 2340, 2340, 1560)
    assert rc == 0 and whole == 256                      # fills the GPU: no parts
    rc, token = _window_bytes(1, 1, 262144, 8, 8, 128, -1, 0, 0)
    assert rc == 0 and token > 2 * 8 * (128 + 2) * 4     # several parts of one row per head
    rc, short = _window_bytes(1, 1, 262144, 8, 8, 128, 30, 0, 0)
    assert rc == 0 and short < token                     # a short window has few steps to divide
    rc, huge = _window_bytes(1, 1, 262144, 8, 8, 128, (1 << 62), (1 << 62), 1 << 62)
    assert rc == 0 and huge == token                     # bounds past every position
    rc, grad = _window_bytes(2, 100, 100, 6, 2, 64, -1, 0, 0, backward=1)
    assert rc == 0 and grad == 256 + 2 * 2 * 2 * 3 * 128 * 4   # two numbers per row of 3 tiles
    rc, grad = _window_bytes(1, 1500, 1500, 2, 2, 64, -1, 0, 0, backward=1)
    assert rc == 0 and grad > 256 + 2 * 2 * 12 * 128 * 4 + 2 * 1500 * 2 * 64 * 4   # and parts of the gradients
    rc, grad = _window_bytes(4, 4096, 4096, 24, 24, 128, 1023, 0, 64, backward=1)
    assert rc == 0 and grad == 256 + 2 * 4 * 24 * 32 * 128 * 4


@pytest.mark.parametrize("args", [(0, 4, 2, 2, 64), (1, 0, 2, 2, 64), (1, 4, 0, 2, 64), (1, 4, 2, 0, 64),
                                  (1, 4, 2, 2, 0), (1, 4, 2, 2, 60), (1, 4, 2, 2, 264)])
def test_rope_plan_refuses(args):
    n = ctypes.c_int64(-1)
    assert _lib.lib().solb200_qk_norm_rope_backward_workspace(*args, ctypes.byref(n)) == 1
    assert n.value == -1 and _lib.last_error()


def test_host_tensors_are_refused():
    q = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    w, t = torch.ones(64), torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        solb200.qk_norm_rope(q, q, w, w, t, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        solb200.qk_norm_rope_backward(q, q, q, q, w, w, t, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        solb200.window_attn(q, q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        solb200.window_attn_backward(q, q, q, q, q, torch.zeros(1, 2, 8))


def test_options_are_numbers_not_tensors():
    q = torch.zeros(1, 8, 2, 64, dtype=torch.bfloat16)
    w, t = torch.ones(64), torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="eps must be a number"):
        solb200.qk_norm_rope(q, q, w, w, t, t, eps=torch.tensor(1e-6))
    for name in ("left", "right", "sinks", "scale"):
        with pytest.raises(RuntimeError, match=f"{name} must be a number"):
            solb200.window_attn(q, q, q, **{name: torch.tensor(4)})


def _rope_lines(rows, per, most=148 * 3):
    """CTAs of the rotation's gradient: one run per warp while they last, else a share of `most`."""
    want = [-(-r // per) for r in rows]
    if sum(want) > most:
        want = [min(w, max(1, most * r // sum(rows))) for w, r in zip(want, rows)]
    return sum(want)


@pytest.mark.parametrize("D,lanes", [(64, 8), (128, 16), (256, 32)])
def test_rope_gradient_workspace_holds_every_types_lines(D, lanes):
    """One line of D sums per CTA, whether the element type takes 4 rows a run (16 bits) or 2 (32)."""
    n, short = ctypes.c_int64(-1), []
    for H, Hk in ((32, 8), (16, 4), (8, 2), (32, 4), (28, 4), (64, 8), (40, 40), (24, 24), (15, 5), (1, 1)):
        for T in range(1, 6000):
            assert _lib.lib().solb200_qk_norm_rope_backward_workspace(1, T, H, Hk, D, ctypes.byref(n)) == 0
            need = max(_rope_lines((T * H, T * Hk), 32 // lanes * rows * 8) for rows in (4, 2))
            if n.value < need * D * 4:
                short.append((T, H, Hk))
    assert not short


def _calls():
    """The four calls, as (call, its tensors)."""
    q = torch.randn(1, 8, 2, 64).bfloat16()
    w, t = torch.ones(64), torch.ones(8, 32)
    lse = torch.zeros(1, 2, 8)
    return [(solb200.qk_norm_rope, [q, q, w, w, t, t]), (solb200.qk_norm_rope_backward, [q, q, q, q, w, w, t, t]),
            (solb200.window_attn, [q, q, q]), (solb200.window_attn_backward, [q, q, q, q, q, lse])]


def test_forward_mode_derivatives_are_refused():
    """A tangent would be dropped: the calls refuse it, of every tensor; without one they go on
    to their other checks."""
    for call, args in _calls():
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                with pytest.raises(RuntimeError, match="CUDA"):
                    call(*args)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.func.jvp(lambda x: call(*args[:i], x, *args[i + 1:]), (args[i],), (args[i],))
        with pytest.raises(RuntimeError, match="CUDA"):
            call(*args)


def test_a_captured_call_has_an_error_word_of_its_own(monkeypatch):
    """Plain calls of a stream share one word. A graph may be replayed on another stream, beside
    them: its calls take neither the stream's word nor leave theirs to it."""
    from solb200 import layer_ops
    monkeypatch.setattr(layer_ops, "_ERROR_WORDS", {})
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    q = torch.zeros(1)
    plain = layer_ops._workspace(256, q, 0, 7)
    assert layer_ops._workspace(256, q, 0, 7) is plain and layer_ops._workspace(256, q, 0, 8) is not plain
    capturing = True
    captured = [layer_ops._workspace(256, q, 0, 7) for _ in range(2)] + [layer_ops._workspace(256, q, 0, 9)]
    assert len({t.data_ptr() for t in (plain, *captured)}) == 4
    capturing = False
    assert layer_ops._workspace(256, q, 0, 7) is plain
    assert all(layer_ops._workspace(256, q, 0, 9) is not t for t in captured)
