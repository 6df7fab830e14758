"""Sliding-window attention with sinks (``solb200.window_attn``), its gradient, and the streaming
layer on it, against the definition in 64 bits.

Tolerances (u = 2^-8, the half spacing of bf16 at 1). The forward rounds each weight of a row to
bf16 before the product with V, and the result once: |error| <= u (sum p |v| + |o|), plus the
scores' fp32 error, which moves every weight by a relative 2^-24 * 2 D * (scale sum |q k|) - the
bounds below take 2^-12 of it with room. The gradient rounds P and dS to bf16, takes delta
from the rounded output (off by D_i = u sum_d |dO| (sum p |v| + |o|)), and rounds once: with
e = u |dS| + P D_i, |error of dQ| <= scale e |K| + u |dQ| and alike for dK; of dV
u P^T |dO| + u |dV|."""

import pytest
import torch

import solb200

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
SLACK = 2.0 ** -12      # fp32 scores, exponentials and sums, relative to the magnitudes


def _inputs(B, Tq, Tk, H, Hk, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Tq, H, D, generator=g).bfloat16()
    k, v = (torch.randn(B, Tk, Hk, D, generator=g).bfloat16() for _ in range(2))
    return q, k, v


def _see(Tq, Tk, L, off, left, right, sinks):
    p = off + torch.arange(Tq)[:, None]
    j = torch.arange(Tk)[None]
    see = (j < L).expand(Tq, -1).clone()
    if right is not None:
        see &= j <= p + right
    if left is not None:
        see &= (j >= p - left) | (j < sinks)
    return see


def _definition(q, k, v, *, left=None, right=0, sinks=0, scale=None, lengths=None, offsets=None, dout=None):
    """(out, lse, bounds) in 64 bits, and with ``dout`` (dq, dk, dv) and theirs."""
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out, out_b = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((B, H, Tq), -torch.inf, dtype=torch.float64)
    lse_b = torch.zeros_like(lse)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    bounds = [torch.zeros_like(t) for t in (q, k, v)]
    for b in range(B):
        L = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        off = L - Tq if offsets is None else int(offsets[b])
        see = _see(Tq, Tk, L, off, left, right, sinks)
        rows = see.any(1)
        seen = torch.nan_to_num(k[b]), torch.nan_to_num(v[b])
        for h in range(H):
            kk, vv = (t[:, h // G] * (torch.arange(Tk)[:, None] < L) for t in seen)
            qq = q[b, :, h]
            s = (scale * qq @ kk.T).masked_fill(~see, -torch.inf)
            s[~rows] = 0.0
            p = torch.softmax(s, -1)
            p[~rows] = 0.0
            p = p * see
            o = p @ vv
            mag = p @ vv.abs()
            sm = scale * (qq.abs() @ kk.abs().T * see).amax(-1)
            out[b, :, h] = o
            out_b[b, :, h] = U * (mag + o.abs()) + SLACK * (1 + sm[:, None] / D) * mag
            lse[b, h, rows] = torch.logsumexp(s, -1)[rows]
            lse_b[b, h] = 2.0 ** -17 * (1 + sm)
            if dout is None:
                continue
            do = dout[b, :, h].double()
            dp = do @ vv.T
            ds = p * (dp - (do * o).sum(-1, keepdim=True))
            Di = (do.abs() * out_b[b, :, h]).sum(-1, keepdim=True)
            near = SLACK * (1 + sm[:, None] / D)
            e = (U + near) * ds.abs() + p * Di + near * p * (do.abs() @ vv.abs().T)
            grads[0][b, :, h] = scale * ds @ kk
            bounds[0][b, :, h] = scale * e @ kk.abs()
            grads[1][b, :, h // G] += scale * ds.T @ qq
            bounds[1][b, :, h // G] += scale * e.T @ qq.abs()
            grads[2][b, :, h // G] += p.T @ do
            bounds[2][b, :, h // G] += ((U + near) * p).T @ do.abs()
    bounds = [bd + U * t.abs() for bd, t in zip(bounds, grads)]
    return out, lse, out_b, lse_b, grads, bounds


def _check(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound - 1e-30).max().item()
    assert over <= 0, f"{what}: {over:.3e} past the bound"


def _device(how):
    return {n: torch.tensor(x, dtype=torch.int32).cuda() if isinstance(x, (list, tuple)) else x
            for n, x in how.items()}


def _check_forward(q, k, v, how, **call):
    out, lse = solb200.window_attn(q.cuda(), k.cuda(), v.cuda(), return_lse=True, **_device(how), **call)
    assert out.dtype == torch.bfloat16 and out.is_contiguous() and lse.dtype == torch.float32
    o, l, ob, lb, _, _ = _definition(q, k, v, **how)
    _check(out, o, ob, "out")
    lse = lse.double().cpu()
    assert torch.equal(torch.isinf(lse), torch.isinf(l)) and (lse[torch.isinf(l)] < 0).all()
    fin = torch.isfinite(l)
    assert ((lse - l).abs() <= lb)[fin].all(), ((lse - l).abs() - lb)[fin].max()
    return out


# B, Tq, Tk, H, Hk, D, how
FORWARD = [
    (1, 1, 1, 1, 1, 64, {}),
    (1, 1, 1, 1, 1, 128, dict(left=0)),
    (2, 130, 130, 3, 3, 128, dict(left=None, right=None)),
    (1, 257, 257, 4, 2, 64, dict(left=31, sinks=1)),
    (1, 300, 300, 2, 2, 128, dict(left=64, right=64, sinks=5)),
    (2, 100, 700, 6, 2, 64, dict(left=200, sinks=130)),          # 3 heads a group: a part of the tile unused
    (1, 77, 513, 5, 1, 128, dict(left=100, right=None)),
    (1, 40, 320, 8, 1, 64, dict(left=3, right=2, sinks=70)),
    (1, 2, 129, 128, 1, 64, dict()),                              # 128 heads on one key head
    (1, 3, 129, 100, 1, 64, dict(left=50)),
    (1, 128, 128, 1, 1, 64, dict(left=0, right=0)),               # every query sees itself only
    (1, 65, 192, 2, 1, 128, dict(left=10, sinks=64)),             # sinks end with a step
    (1, 65, 192, 2, 1, 128, dict(left=10, sinks=65)),
    (1, 65, 192, 2, 1, 128, dict(left=10, sinks=1000)),           # all keys are sinks
    (3, 70, 200, 4, 2, 64, dict(left=20, sinks=2, lengths=[200, 0, 1])),
    (4, 333, 333, 4, 4, 64, dict(left=127, sinks=4, lengths=[333, 300, 97, 1], offsets=[0, 0, 0, 0])),
    (3, 150, 150, 2, 2, 128, dict(left=20, lengths=[150, 60, 0], offsets=[0, 0, 0])),    # rows that see nothing
    (2, 50, 100, 2, 2, 64, dict(left=5, offsets=[-30, 90])),      # before the first key, past the last
    (2, 50, 100, 2, 2, 64, dict(left=5, right=None, sinks=3, offsets=[-2 ** 31, 2 ** 31 - 1])),
    (2, 9, 40, 2, 2, 64, dict(lengths=[-5, 1000])),               # lengths are clamped
    (1, 20, 30, 2, 2, 64, dict(left=2 ** 62, right=2 ** 62, sinks=2 ** 40)),
    (1, 33, 90, 2, 1, 64, dict(scale=0.7, left=40)),
    # single tokens and short chunks against long caches: split over the key axis
    (1, 1, 5000, 2, 2, 128, dict()),
    (3, 1, 3000, 6, 2, 64, dict(left=700, sinks=4, lengths=[3000, 1, 0])),
    (2, 1, 4097, 8, 8, 128, dict(left=4000, lengths=[4097, 64])),
    (1, 1, 2000, 10, 2, 128, dict(right=None, lengths=[1999])),
    (1, 7, 3000, 5, 5, 64, dict(sinks=10, left=1000)),
    (1, 5, 3000, 3, 1, 64, dict(offsets=[0])),                    # most parts see nothing
]


@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,how", FORWARD)
def test_forward(cuda_device, B, Tq, Tk, H, Hk, D, how):
    _check_forward(*_inputs(B, Tq, Tk, H, Hk, D, seed=Tq + Tk), how)


# few tiles with long walks: divided over the query tiles and the key steps
LONG_GRADIENT = [
    (1, 1500, 1500, 2, 2, 64, {}),
    (1, 1100, 1100, 3, 1, 128, dict(left=None, right=None)),
    (2, 1300, 1300, 2, 1, 64, dict(left=100, sinks=7, lengths=[1300, 700], offsets=[0, 0])),
    (1, 300, 2500, 2, 2, 128, dict(left=2000, lengths=[2400])),
]


@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,how", [c for c in FORWARD if c[1] <= 333] + LONG_GRADIENT)
def test_gradient(cuda_device, B, Tq, Tk, H, Hk, D, how):
    q, k, v = _inputs(B, Tq, Tk, H, Hk, D, seed=Tq + 3 * Tk)
    dout = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    args = [t.cuda() for t in (q, k, v)]
    dev = _device(how)
    out, lse = solb200.window_attn(*args, return_lse=True, **dev)
    got = solb200.window_attn_backward(dout.cuda(), *args, out, lse, **dev)
    again = solb200.window_attn_backward(dout.cuda(), *args, out, lse, **dev)
    _, _, _, _, want, bounds = _definition(q, k, v, dout=dout, **how)
    for a, b, w, bd, name in zip(got, again, want, bounds, ("dq", "dk", "dv")):
        assert torch.equal(a, b), name                    # the same bits every time
        _check(a, w, bd, name)


def test_one_key_per_row_has_no_score_gradient(cuda_device):
    """Rows that see a single key: P = 1, dS = 0. dq and dk are what fp32 leaves of dP - delta: a
    few units of 2^-24 of the dot product dO . V (sqrt(D) here) times K."""
    q, k, v = (t.cuda() for t in _inputs(2, 70, 70, 2, 2, 64, seed=13))
    for how in (dict(left=0), dict(lengths=torch.tensor([1, 1], dtype=torch.int32).cuda(), right=None)):
        out, lse = solb200.window_attn(q, k, v, return_lse=True, **how)
        dq, dk, dv = solb200.window_attn_backward(torch.randn_like(q), q, k, v, out, lse, **how)
        assert dq.abs().max() <= 2.0 ** -17 and dk.abs().max() <= 70 * 2.0 ** -17 and dv.any()


def test_gradient_against_differences(cuda_device):
    """The definition differenced in 64 bits along random directions: off from the kernels'
    gradient by no more than the gradient's own bounds along that direction (h^2 terms are 1e-8)."""
    how = dict(left=30, sinks=3, lengths=[90, 41])
    q, k, v = _inputs(2, 60, 90, 4, 2, 64, seed=8)
    g = torch.Generator().manual_seed(9)
    dout = torch.randn(q.shape, generator=g).bfloat16()
    xs = [t.cuda() for t in (q, k, v)]
    out, lse = solb200.window_attn(*xs, return_lse=True, **_device(how))
    got = solb200.window_attn_backward(dout.cuda(), *xs, out, lse, **_device(how))
    bounds = _definition(q, k, v, dout=dout, **how)[5]
    h = 1e-4
    for i in range(3):
        d = torch.randn((q, k, v)[i].shape, generator=g).double()
        ends = []
        for sign in (1, -1):
            moved = [t.double() + (sign * h * d if j == i else 0) for j, t in enumerate((q, k, v))]
            ends.append((_definition(*moved, **how)[0] * dout.double()).sum())
        diff = ((ends[0] - ends[1]) / (2 * h)).item()
        mine = (got[i].double().cpu() * d).sum().item()
        assert abs(diff - mine) <= (bounds[i] * d.abs()).sum().item() + 1e-4, (i, diff, mine)


@pytest.mark.parametrize("Tq", [1, 100])
def test_what_lies_behind_a_length_is_not_used(cuda_device, Tq):
    """NaN and infinities in a cache past each sequence's length change nothing, in either direction."""
    q, k, v = (t.cuda() for t in _inputs(3, Tq, 700, 4, 2, 128, seed=2))
    lengths = torch.tensor([650, 300, 129], dtype=torch.int32).cuda()
    how = dict(left=400, sinks=4, lengths=lengths)
    clean = solb200.window_attn(q, k, v, return_lse=True, **how)
    dout = torch.randn_like(q)
    grads = solb200.window_attn_backward(dout, q, k, v, *clean, **how)
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lengths.tolist()):
        k2[b, n:], v2[b, n:] = float("nan"), float("inf")
    dirty = solb200.window_attn(q, k2, v2, return_lse=True, **how)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for a, b in zip(grads, solb200.window_attn_backward(dout, q, k2, v2, *dirty, **how)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Tq", [1, 20])
def test_keys_outside_every_window_are_not_used(cuda_device, Tq):
    """NaN and infinities in keys between the sinks and the window, which no query sees, next to
    keys that are seen, in the same tiles."""
    q, k, v = (t.cuda() for t in _inputs(2, Tq, 700, 4, 2, 64, seed=12))
    how = dict(left=100, sinks=5)
    clean = solb200.window_attn(q, k, v, return_lse=True, **how)
    dout = torch.randn_like(q)
    grads = solb200.window_attn_backward(dout, q, k, v, *clean, **how)
    k2, v2 = k.clone(), v.clone()
    hidden = slice(5, 700 - Tq - 100)
    k2[:, hidden], v2[:, hidden] = float("nan"), float("-inf")
    dirty = solb200.window_attn(q, k2, v2, return_lse=True, **how)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for a, b in zip(grads, solb200.window_attn_backward(dout, q, k2, v2, *dirty, **how)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("Tq,Hk,D", [(1, 2, 64), (100, 4, 64), (300, 2, 128), (300, 4, 64), (700, 1, 128)])
@pytest.mark.parametrize("ends", ["before", "past"])
def test_queries_that_see_nothing_are_not_used(cuda_device, Tq, Hk, D, ends):
    """NaN and infinities in the queries, and in their outputs' gradients, of padding before a
    sequence's first key or past its last window leave the gradients of all keys as they were."""
    q, k, v = (t.cuda() for t in _inputs(4, Tq, 700, 4, Hk, D, seed=31))
    lengths = [0, 1, Tq // 3, Tq]
    offsets = [n - Tq for n in lengths] if ends == "before" else [0] * 4
    left = None if ends == "before" else 20
    how = dict(left=left, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(),
               offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    clean = solb200.window_attn(q, k, v, return_lse=True, **how)
    dout = torch.randn_like(q)
    blind = torch.isneginf(clean[1]).transpose(1, 2)
    assert blind[0].all() and blind[1:].any() and (Tq == 1 or not blind[1:].all())
    grads = solb200.window_attn_backward(dout, q, k, v, *clean, **how)
    q2 = torch.where(blind[..., None], torch.tensor(float("nan"), device="cuda", dtype=q.dtype), q)
    dout2 = torch.where(blind[..., None], torch.tensor(float("inf"), device="cuda", dtype=q.dtype), dout)
    dirty = solb200.window_attn(q2, k, v, return_lse=True, **how)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for a, b in zip(grads, solb200.window_attn_backward(dout2, q2, k, v, *dirty, **how)):
        assert torch.equal(a, b)
    assert not grads[0][blind].any()


def test_agrees_with_the_dense_kernel(cuda_device):
    """No bounds: the dense call's attention, up to both calls' roundings."""
    q, k, v = _inputs(1, 500, 900, 3, 3, 128, seed=3)
    _, _, bound, _, _, _ = _definition(q, k, v, right=None)
    a = solb200.window_attn(q.cuda(), k.cuda(), v.cuda(), left=None, right=None)
    b = solb200.dense_attn(q.cuda(), k.cuda(), v.cuda())
    _check(a, b.double().cpu(), 2 * bound, "dense")


def test_strided_inputs(cuda_device):
    B, T, H, Hk, D = 2, 90, 6, 2, 64
    qkv = torch.randn(B, T, (H + 2 * Hk), D, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    q, k, v = qkv.split((H, Hk, Hk), dim=2)
    how = dict(left=20, sinks=2)
    want = solb200.window_attn(q.contiguous(), k.contiguous(), v.contiguous(), return_lse=True, **how)
    dout = torch.randn(B, H, T, D, device="cuda").bfloat16().transpose(1, 2)
    grads = solb200.window_attn_backward(dout.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), *want, **how)
    bhnd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = [torch.empty(*t.shape[:-1], D + 1, dtype=t.dtype, device=t.device)[..., 1:].copy_(t) for t in (q, k, v)]
    for form in ((q, k, v), bhnd, odd):
        assert torch.equal(solb200.window_attn(*form, **how), want[0])
        got = solb200.window_attn_backward(dout, *form, *want, **how)
        assert all(torch.equal(a, b) for a, b in zip(got, grads))
    one = k[:, :, :1].expand(-1, -1, H, -1)       # one key head repeated by expand()
    assert torch.equal(solb200.window_attn(q, one, one, **how),
                       solb200.window_attn(q, one.contiguous(), one.contiguous(), **how))


def test_a_long_cache(cuda_device):
    """Offsets past 2^31 elements: the window at the end of a cache of 2.6e9 elements."""
    T, H, D = 510_000, 40, 128
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB of free device memory")
    k = torch.empty(1, T, H, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    k[:, -300:].normal_()
    v[:, -300:].normal_()
    k[:, :2].normal_()
    v[:, :2].normal_()
    for Tq in (1, 150):
        q = torch.randn(1, Tq, H, D, device="cuda").bfloat16()
        out = solb200.window_attn(q, k, v, left=100, sinks=2)
        kk, vv = (torch.cat((t[:, :2], t[:, -300:]), 1).cpu() for t in (k, v))
        want, _, bound, _, _, _ = _definition(q.cpu(), kk, vv, left=100, sinks=2)
        _check(out, want, bound, f"long cache, {Tq} queries")


def test_empty(cuda_device):
    q, k, v = (t.cuda() for t in _inputs(2, 5, 7, 4, 2, 64))
    out = solb200.window_attn(q[:, :0], k, v)
    assert out.shape == (2, 0, 4, 64)
    out, lse = solb200.window_attn(q, k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and (lse == -torch.inf).all() and lse.shape == (2, 4, 5)
    grads = solb200.window_attn_backward(q, q, k[:, :0], v[:, :0], out, lse)
    assert not grads[0].any() and grads[1].shape == (2, 0, 2, 64)
    assert solb200.window_attn(q[:0], k[:0], v[:0]).shape == (0, 5, 4, 64)


def test_autograd(cuda_device):
    q, k, v = (t.cuda() for t in _inputs(2, 80, 80, 4, 2, 64, seed=5))
    how = dict(left=30, sinks=2, lengths=torch.tensor([80, 50], dtype=torch.int32).cuda(),
               offsets=torch.zeros(2, dtype=torch.int32).cuda())
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = solb200.window_attn(*leaves, **how)
    plain, lse = solb200.window_attn(q, k, v, return_lse=True, **how)
    assert torch.equal(out, plain) and not plain.requires_grad
    dout = torch.randn_like(out)
    got = torch.autograd.grad(out, leaves, dout)
    want = solb200.window_attn_backward(dout, q, k, v, plain, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    out, lse2 = solb200.window_attn(*leaves, return_lse=True, **how)
    assert torch.equal(lse2, lse) and not lse2.requires_grad


def test_other_stream_and_graph(cuda_device, monkeypatch):
    """On another stream, and captured in a CUDA graph and replayed with new inputs."""
    from solb200 import layer_ops
    monkeypatch.setattr(layer_ops, "_SYNC_CHECK", False)      # reading the error word synchronises
    q, k, v = (t.cuda() for t in _inputs(2, 1, 2000, 4, 4, 128, seed=6))
    lengths = torch.tensor([1500, 7], dtype=torch.int32).cuda()
    want = solb200.window_attn(q, k, v, lengths=lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(solb200.window_attn(q, k, v, lengths=lengths), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = solb200.window_attn(q, k, v, lengths=lengths)
    lengths.copy_(torch.tensor([3, 2000], dtype=torch.int32))
    q.normal_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, solb200.window_attn(q, k, v, lengths=lengths))


def test_streaming_layer(cuda_device):
    """A sequence in one call, and the same sequence in chunks and single tokens against a cache,
    agree: both paths round to bf16 at the same places, so they differ by the attention's own
    bound on a value of about 1, carried through a projection of 256 terms of size 1/16."""
    torch.manual_seed(0)
    dim, heads, kv, D, T = 256, 4, 2, 64, 150
    layer = solb200.StreamingSelfAttention(dim, heads, kv_heads=kv, head_dim=D, left=40, sinks=3).cuda()
    layer.qkv.bfloat16()
    layer.out.bfloat16()
    x = torch.randn(2, T, dim, device="cuda").bfloat16()
    angle = torch.arange(T, device="cuda")[:, None] * 100.0 ** (-torch.arange(D // 2, device="cuda") / (D // 2))
    cos, sin = angle.cos(), angle.sin()
    with torch.no_grad():
        whole = layer(x, cos, sin)
        cache = layer.new_cache(2, T + 10)
        cache.k.fill_(float("nan"))
        cache.v.fill_(float("nan"))
        parts, t = [], 0
        for n in (70, 1, 1, 40, 1, 37):
            parts.append(layer(x[:, t:t + n], cos[t:t + n], sin[t:t + n], cache=cache))
            t += n
    assert cache.lengths.tolist() == [T, T]
    diff = (torch.cat(parts, 1).float() - whole.float()).abs().max().item()
    assert diff <= 8 * U, diff
    y = layer(x, cos, sin)
    assert torch.equal(y, whole)
    y.float().square().mean().backward()
    for name, prm in layer.named_parameters():
        assert prm.grad is not None and torch.isfinite(prm.grad).all() and prm.grad.any(), name


def test_refusals(cuda_device):
    q, k, v = (t.cuda() for t in _inputs(2, 5, 7, 4, 2, 64))
    n = torch.tensor([7, 7], dtype=torch.int32).cuda()
    for args, how in [((q.half(), k, v), {}), ((q, k.float(), v), {}), ((q[0], k, v), {}), ((q, k[:1], v[:1]), {}),
                      ((q, k, v[:, :3]), {}), ((q[..., :32], k[..., :32], v[..., :32]), {}), ((q[:, :, :3], k, v), {}),
                      ((q.cpu(), k, v), {}), ((q, k.cpu(), v.cpu()), {}), ((q, k, v), dict(left=-1)),
                      ((q, k, v), dict(right=-3)), ((q, k, v), dict(sinks=-1)), ((q, k, v), dict(scale=0.0)),
                      ((q, k, v), dict(scale=float("nan"))), ((q, k, v), dict(lengths=n.long())),
                      ((q, k, v), dict(lengths=n[:1])), ((q, k, v), dict(offsets=n.cpu())),
                      ((q, k, v), dict(lengths=[7, 7])), ((q, k[:, :, :0], v[:, :, :0]), {})]:
        with pytest.raises(RuntimeError, match="solb200"):
            solb200.window_attn(*args, **how)
    out, lse = solb200.window_attn(q, k, v, return_lse=True)
    for bad in ((q[:, :3], q, k, v, out, lse), (q, q, k, v, out[:, :3], lse), (q, q, k, v, out, lse[:, :, :3]),
                (q, q, k, v, out, lse.double())):
        with pytest.raises(RuntimeError, match="solb200"):
            solb200.window_attn_backward(*bad)


def test_c_abi_refusals(cuda_device):
    """Status codes for pointers, strides and workspaces that the Python layer never passes."""
    from ctypes import c_int64
    from solb200._lib import I64x3, lib
    q, k, v = (t.cuda() for t in _inputs(1, 1, 3000, 2, 2, 64))
    out = torch.empty_like(q)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    st = lambda t: I64x3(*t.stride()[:3])

    def call(qp=q.data_ptr(), ks=st(k), outp=out.data_ptr(), wsp=ws.data_ptr(), n=1 << 20, lens=None, scale=0.1):
        return lib().solb200_window_attn(qp, st(q), k.data_ptr(), ks, v.data_ptr(), st(v), outp, None, lens, None, 1, 1,
                                         3000, 2, 2, 64, c_int64(-1), 0, 0, scale, wsp, n,
                                         torch.cuda.current_stream().cuda_stream)
    assert call() == 0
    assert call(qp=None) == 1 and call(qp=q.data_ptr() + 2) == 2
    assert call(ks=I64x3(1, 4, 64)) == 2 and call(ks=I64x3(1, 0, 64)) == 2
    assert call(outp=None) == 2 and call(wsp=None) == 3 and call(n=256) == 3 and call(wsp=ws.data_ptr() + 4) == 2
    assert call(lens=ws.data_ptr() + 2) == 2 and call(scale=-1.0) == 1
    torch.cuda.synchronize()


@pytest.mark.parametrize("T,H,Hk,D,how", [(128, 8, 8, 128, {}), (100, 6, 2, 64, {}), (97, 4, 2, 128, dict(right=None)),
                                          (128, 40, 8, 64, dict(left=90, sinks=3))])
def test_gradient_of_sequences_of_one_key_step(cuda_device, T, H, Hk, D, how):
    """Query tiles whose keys lie in one step, many on the GPU at a time: copies of a sequence all give
    the same bits, every time, and those of the definition up to its bounds. (The row sums behind delta
    are exchanged where the first product of dQ goes.)"""
    copies = 64
    one = _inputs(1, T, T, H, Hk, D, seed=41)
    do = torch.randn(one[0].shape, generator=torch.Generator().manual_seed(42)).bfloat16()
    q, k, v, dout = (t.cuda().repeat(copies, 1, 1, 1) for t in (*one, do))
    out, lse = solb200.window_attn(q, k, v, return_lse=True, **how)
    first = None
    for _ in range(20):
        got = solb200.window_attn_backward(dout, q, k, v, out, lse, **how)
        first = first or [t[:1].clone() for t in got]
        assert all(torch.equal(t, f.expand_as(t)) for t, f in zip(got, first))
    _, _, _, _, want, bounds = _definition(*one, dout=do, **how)
    for a, w, bd, name in zip(first, want, bounds, ("dq", "dk", "dv")):
        _check(a, w, bd, name)


BELOW_SINKS = [
    # Tq, Tk, D, how (H 4, Hk 2): fewer visible keys than sinks, by the length or by the right bound
    (1, 300, 64, dict(left=50, sinks=4, lengths=[1, 3, 2])),
    (1, 2000, 128, dict(left=200, sinks=1560, lengths=[100, 1, 1501])),
    (1, 300, 64, dict(sinks=64, lengths=[10, 65, 63])),                      # no left bound
    (1, 5000, 64, dict(left=4095, sinks=4, lengths=[1, 2, 70])),             # parts of the key axis
    (20, 2000, 64, dict(left=200, sinks=1560, lengths=[100, 20, 1530])),
    (150, 700, 128, dict(left=30, sinks=400, lengths=[150, 170, 390])),
    (40, 300, 64, dict(left=20, sinks=130, offsets=[0, 10, 60])),            # keys that come later
    (40, 300, 128, dict(left=20, right=5, sinks=70, offsets=[-10, 20, 0])),
    (333, 333, 64, dict(left=127, sinks=64, lengths=[5, 63, 0], offsets=[0, 0, 0])),
]


@pytest.mark.parametrize("Tq,Tk,D,how", BELOW_SINKS)
def test_keys_past_the_visible_end_among_the_sinks_are_not_used(cuda_device, Tq, Tk, D, how):
    """NaN and infinities in every key that no query sees change nothing, also where the visible keys
    end before the last sink."""
    q, k, v = (t.cuda() for t in _inputs(3, Tq, Tk, 4, 2, D, seed=Tq + Tk))
    lengths, offsets = how.get("lengths", [Tk] * 3), how.get("offsets")
    dev = _device(how)
    clean = solb200.window_attn(q, k, v, return_lse=True, **dev)
    dout = torch.randn_like(q)
    grads = solb200.window_attn_backward(dout, q, k, v, *clean, **dev)
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        off = n - Tq if offsets is None else offsets[b]
        hidden = ~_see(Tq, Tk, n, off, how.get("left"), how.get("right", 0), how["sinks"]).any(0).cuda()
        assert hidden[:how["sinks"]].any() or n >= how["sinks"]
        k2[b, hidden], v2[b, hidden] = float("nan"), float("inf")
    dirty = solb200.window_attn(q, k2, v2, return_lse=True, **dev)
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for a, b in zip(grads, solb200.window_attn_backward(dout, q, k2, v2, *dirty, **dev)):
        assert torch.equal(a, b)


def test_streaming_from_the_first_token(cuda_device):
    """Single tokens into a cache that holds NaN, from the first one on, with more sinks than tokens:
    as the whole sequence in one call (bound as in test_streaming_layer)."""
    torch.manual_seed(1)
    layer = solb200.StreamingSelfAttention(128, 2, head_dim=64, left=6, sinks=16).cuda()
    layer.qkv.bfloat16()
    layer.out.bfloat16()
    x = torch.randn(2, 24, 128, device="cuda").bfloat16()
    angle = torch.randn(24, 32, device="cuda")
    with torch.no_grad():
        whole = layer(x, angle.cos(), angle.sin())
        cache = layer.new_cache(2, 40)
        cache.k.fill_(float("nan"))
        cache.v.fill_(float("nan"))
        parts = [layer(x[:, t:t + 1], angle[t:t + 1].cos(), angle[t:t + 1].sin(), cache=cache) for t in range(24)]
    diff = (torch.cat(parts, 1).float() - whole.float()).abs().max().item()
    assert diff <= 8 * U, diff


def test_empty_with_another_default_dtype(cuda_device):
    """The log-sum-exp is float32 whatever torch's default, and the gradient takes it."""
    q, k, v = (t.cuda() for t in _inputs(2, 5, 7, 4, 2, 64))
    before = torch.get_default_dtype()
    try:
        for dtype in (torch.float64, torch.bfloat16):
            torch.set_default_dtype(dtype)
            for kv in ((k[:, :0], v[:, :0]), (k, v)):
                out, lse = solb200.window_attn(q, *kv, return_lse=True)
                assert lse.dtype == torch.float32
                grads = solb200.window_attn_backward(q, q, *kv, out, lse)
                assert all(t.dtype == torch.bfloat16 for t in grads)
    finally:
        torch.set_default_dtype(before)
