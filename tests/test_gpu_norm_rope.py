"""Head norms with the position rotation (``solb200.qk_norm_rope``) and the gradient, against the
formula in 64 bits.

Tolerances. With u the half spacing of the result's type at 1 (2^-8 bf16, 2^-11 f16, 2^-24 f32):
y is rounded once, u |y|, from fp32 arithmetic whose relative error is at most about 24 units of
2^-24 (a sum of up to 256 squares in a tree of 8-term runs, a reciprocal root, four products) of
the pair's magnitudes |a| + |b|. dx likewise, on the magnitudes of its terms. A weight's gradient
adds |g x^| over the rows, in runs of at most 256 terms here: 2^-24 * 256 of the sum of
magnitudes. f16 results below the normal range round to multiples of 2^-24."""

import pytest
import torch

import solb200

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}
EPS = 1e-6


def _turn(x, cos, sin, interleaved):
    """x [B, T, H, D] turned by cos, sin [B, T, R / 2]."""
    half = cos.shape[-1]
    c, s = cos[:, :, None], sin[:, :, None]
    y = x.clone()
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    a, b = x[..., ia], x[..., ib]
    y[..., ia] = a * c - b * s
    y[..., ib] = a * s + b * c
    return y


def _partner(x, R, interleaved):
    """The magnitudes |a| + |b| of every element's pair."""
    m = x.abs()
    ia = torch.arange(R // 2) * 2 if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    both = m[..., ia] + m[..., ib]
    m = m.clone()
    m[..., ia] = both
    m[..., ib] = both
    return m


def _formula(x, w, cos, sin, interleaved, eps=EPS):
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return _turn(x * r * w, cos, sin, interleaved), r


def _inputs(B, T, H, Hk, D, R, dtype, wdtype=None, per_batch=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, T, H, D, generator=g).to(dtype)
    k = (3 * torch.randn(B, T, Hk, D, generator=g)).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdtype or dtype) for _ in range(2))
    angle = 50 * torch.randn(*((B, T) if per_batch else (T,)), R // 2, generator=g)
    return q, k, wq, wk, angle.cos(), angle.sin()


def _tables(cos, sin, B):
    return tuple((t if t.dim() == 3 else t.expand(B, -1, -1)).double() for t in (cos, sin))


def _check(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, f"{what}: {over:.3e} past the bound"


CASES = [
    # B, T, H, Hk, D, R, dtype, interleaved, per_batch
    (1, 1, 1, 1, 64, 64, torch.bfloat16, True, False),
    (8, 1, 40, 8, 128, 128, torch.bfloat16, False, True),
    (2, 33, 5, 3, 64, 32, torch.float32, False, False),
    (1, 130, 24, 24, 128, 64, torch.float16, True, False),
    (3, 7, 3, 1, 8, 8, torch.float32, True, True),
    (2, 9, 7, 7, 80, 80, torch.bfloat16, False, True),
    (2, 9, 3, 2, 72, 40, torch.float16, True, True),
    (1, 19, 9, 3, 256, 256, torch.bfloat16, False, False),
    (1, 5, 2, 2, 200, 16, torch.float32, False, True),
    (1, 1013, 2, 1, 128, 128, torch.bfloat16, True, False),
]


@pytest.mark.parametrize("B,T,H,Hk,D,R,dtype,interleaved,per_batch", CASES)
def test_forward(cuda_device, B, T, H, Hk, D, R, dtype, interleaved, per_batch):
    q, k, wq, wk, cos, sin = _inputs(B, T, H, Hk, D, R, dtype, per_batch=per_batch)
    got = solb200.qk_norm_rope(*(t.cuda() for t in (q, k, wq, wk, cos, sin)), eps=EPS, interleaved=interleaved)
    tc, ts = _tables(cos, sin, B)
    for y, x, w, what in ((got[0], q, wq, "q"), (got[1], k, wk, "k")):
        assert y.dtype == dtype and y.is_contiguous()
        want, r = _formula(x.double(), w.double(), tc, ts, interleaved)
        mags = _partner(x.double() * r * w.double(), R, interleaved)
        _check(y, want, U[dtype] * want.abs() + 24 * 2.0 ** -24 * mags + TINY[dtype], what)


@pytest.mark.parametrize("B,T,H,Hk,D,R,dtype,interleaved,per_batch", CASES)
@pytest.mark.parametrize("w32", [False, True])
def test_gradient(cuda_device, B, T, H, Hk, D, R, dtype, interleaved, per_batch, w32):
    wdtype = torch.float32 if w32 else dtype
    q, k, wq, wk, cos, sin = _inputs(B, T, H, Hk, D, R, dtype, wdtype, per_batch, seed=1)
    g = torch.Generator().manual_seed(2)
    dys = [torch.randn(t.shape, generator=g).to(dtype) for t in (q, k)]
    args = [t.cuda() for t in (*dys, q, k, wq, wk, cos, sin)]
    got = solb200.qk_norm_rope_backward(*args, eps=EPS, interleaved=interleaved)
    again = solb200.qk_norm_rope_backward(*args, eps=EPS, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    tc, ts = _tables(cos, sin, B)
    for dx, dw, dy, x, w, what in ((got[0], got[2], dys[0], q, wq, "q"), (got[1], got[3], dys[1], k, wk, "k")):
        assert dx.dtype == dtype and dw.dtype == wdtype
        xd, wd = x.double(), w.double()
        r = (xd.square().mean(-1, keepdim=True) + EPS).rsqrt()
        gd = _turn(dy.double(), tc, -ts, interleaved)
        gm = _partner(dy.double(), R, interleaved)            # magnitudes behind g
        xh = xd * r
        want_w = (gd * xh).sum((0, 1, 2))
        dot = (gd * wd * xh).mean(-1, keepdim=True)
        want = r * (gd * wd - xh * dot)
        mags = r * (gm * wd.abs() + xh.abs() * (gm * wd.abs() * xh.abs()).mean(-1, keepdim=True))
        _check(dx, want, U[dtype] * want.abs() + 32 * 2.0 ** -24 * mags + TINY[dtype], "d" + what)
        _check(dw, want_w, U[wdtype] * want_w.abs() + 256 * 2.0 ** -24 * (gm * xh.abs()).sum((0, 1, 2)) + TINY[wdtype],
               "dw" + what)


@pytest.mark.parametrize("interleaved", [True, False])
def test_gradient_against_differences(cuda_device, interleaved):
    """The kernels' own forward in fp32, differenced along a random direction. h = 2^-6: the
    difference's error is about h^2 |L'''| ~ 1e-3 of the scale of the sum, its rounding
    2^-24 sqrt(n) |y| / h; both far below 3 % of the derivative's magnitude sqrt(n)."""
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(2, 17, 3, 2, 64, 64, torch.float32, seed=3))
    g = torch.Generator().manual_seed(4)
    xs = [q, k, wq, wk]
    ds = [torch.randn(t.shape, generator=g).cuda() for t in xs]
    dy = [torch.randn(t.shape, generator=g).cuda() for t in (q, k)]
    grads = solb200.qk_norm_rope_backward(*dy, *xs, cos, sin, eps=EPS, interleaved=interleaved)
    h = 2.0 ** -6
    for i in range(4):
        def loss(sign):
            moved = [x + sign * h * d if j == i else x for j, (x, d) in enumerate(zip(xs, ds))]
            return sum((y.double() * g_).sum() for y, g_ in zip(
                solb200.qk_norm_rope(*moved, cos, sin, eps=EPS, interleaved=interleaved), dy))
        diff = ((loss(1) - loss(-1)) / (2 * h)).item()
        want = (grads[i].double() * ds[i]).sum().item()
        size = (grads[i].double() * ds[i]).norm().item()
        assert abs(diff - want) <= 0.03 * size, (i, diff, want, size)


def test_strided_and_broadcast_inputs(cuda_device):
    """Views of one packed projection, other orders and repeated heads give what copies give."""
    B, T, H, Hk, D = 2, 21, 6, 2, 64
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(B, T, (H + 2 * Hk) * D, generator=g).bfloat16().cuda()
    q, k = qkv[..., :H * D].view(B, T, H, D), qkv[..., H * D:(H + Hk) * D].view(B, T, Hk, D)
    _, _, wq, wk, cos, sin = (t.cuda() for t in _inputs(B, T, H, Hk, D, D, torch.bfloat16))
    want = solb200.qk_norm_rope(q.contiguous(), k.contiguous(), wq, wk, cos, sin)
    forms = [(q, k),
             (q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(0, 1).contiguous().transpose(0, 1)),
             (q.movedim(-1, 0).contiguous().movedim(0, -1), k)]
    odd = torch.empty(B, T, H, D + 1, dtype=q.dtype, device=q.device)[..., 1:]       # not 16-byte aligned
    odd.copy_(q)
    forms.append((odd, k))
    for a, b in forms:
        got = solb200.qk_norm_rope(a, b, wq, wk, cos, sin)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one key head repeated by expand(), one table row for every token
    one = k[:, :, :1].expand(-1, -1, H, -1)
    row = tuple(t[:, :1].expand(-1, T, -1) for t in (cos, sin))
    got = solb200.qk_norm_rope(q, one, wq, wk, *row)
    want = solb200.qk_norm_rope(q.contiguous(), one.contiguous(), wq, wk, *(t.contiguous() for t in row))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_autograd_and_repeated_heads(cuda_device):
    """Through autograd; a repeated key head's gradient is the sum over its repeats."""
    B, T, H, D = 1, 11, 4, 64
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(B, T, H, 1, D, D, torch.float32, seed=6))
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = solb200.qk_norm_rope(leaves[0], leaves[1].expand(-1, -1, H, -1), leaves[2], leaves[3], cos, sin)
    g = torch.Generator().manual_seed(7)
    dq, dk = (torch.randn(y.shape, generator=g).cuda() for y in (yq, yk))
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    want = solb200.qk_norm_rope_backward(dq, dk, q, k.expand(-1, -1, H, -1), wq, wk, cos, sin)
    assert torch.equal(grads[0], want[0]) and torch.equal(grads[2], want[2]) and torch.equal(grads[3], want[3])
    assert torch.equal(grads[1], want[1].sum(2, keepdim=True))
    # only one output used
    leaves = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    yq, _ = solb200.qk_norm_rope(*leaves[:2], *leaves[2:], cos, sin)
    grads = torch.autograd.grad(yq, leaves, dq)
    assert torch.equal(grads[0], want[0]) and not grads[1].any() and not grads[3].any()


def test_empty_zero_rows_and_stream(cuda_device):
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(2, 4, 3, 3, 64, 64, torch.bfloat16))
    a, b = solb200.qk_norm_rope(q[:, :0], k[:, :0], wq, wk, cos[:, :0], sin[:, :0])
    assert a.shape == (2, 0, 3, 64) and b.shape == (2, 0, 3, 64)
    grads = solb200.qk_norm_rope_backward(a, b, q[:, :0], k[:, :0], wq, wk, cos[:, :0], sin[:, :0])
    assert grads[0].numel() == 0 and not grads[2].any() and not grads[3].any()
    z = torch.zeros_like(q)                       # a row of zeros: rstd = eps^-1/2, finite
    a, _ = solb200.qk_norm_rope(z, k, wq, wk, cos, sin)
    assert not a.any()
    dx = solb200.qk_norm_rope_backward(q, k, z, k, wq, wk, cos, sin)[0]
    assert torch.isfinite(dx).all()
    want = solb200.qk_norm_rope(q, k, wq, wk, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = solb200.qk_norm_rope(q, k, wq, wk, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_nan_stays_in_its_row(cuda_device):
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(1, 3, 4, 4, 128, 128, torch.bfloat16))
    want = solb200.qk_norm_rope(q, k, wq, wk, cos, sin)[0]
    q[0, 1, 2, 5] = float("nan")
    got = solb200.qk_norm_rope(q, k, wq, wk, cos, sin)[0]
    assert torch.isnan(got[0, 1, 2]).all()
    keep = torch.ones(1, 3, 4, dtype=torch.bool, device="cuda")
    keep[0, 1, 2] = False
    assert torch.equal(got[keep], want[keep])


def test_refusals(cuda_device):
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(2, 4, 3, 3, 64, 64, torch.bfloat16))
    bad = [
        dict(q=q.double()), dict(q=q[0]), dict(k=k.float()), dict(k=k[:, :3]), dict(k=k[..., :32]), dict(k=k.cpu()),
        dict(wq=wq[:32]), dict(wk=wk.float()), dict(wq=wq.half(), wk=wk.half()), dict(wq=wq.cpu()),
        dict(cos=cos[:, :3], sin=sin[:, :3]), dict(cos=cos.double(), sin=sin.double()), dict(cos=cos[..., :16]),
        dict(cos=cos[..., :2], sin=sin[..., :2]), dict(cos=cos[:1], sin=sin[:1]), dict(k=k[:, :, :0]),
        dict(cos=torch.cat((cos, cos), -1), sin=torch.cat((sin, sin), -1)),
        dict(q=q[..., :60], k=k[..., :60], wq=wq[:60], wk=wk[:60], cos=cos[..., :8], sin=sin[..., :8]),
        dict(cos=cos.clone().requires_grad_()), dict(eps=-1.0),
    ]
    for change in bad:
        a = dict(q=q, k=k, wq=wq, wk=wk, cos=cos, sin=sin, eps=EPS)
        a.update(change)
        with pytest.raises(RuntimeError, match="solb200"):
            solb200.qk_norm_rope(a["q"], a["k"], a["wq"], a["wk"], a["cos"], a["sin"], eps=a["eps"])
    with pytest.raises(RuntimeError, match="solb200"):                 # halves need multiples of 16
        solb200.qk_norm_rope(q, k, wq, wk, cos[..., :4], sin[..., :4], interleaved=False)
    with pytest.raises(RuntimeError, match="solb200"):
        solb200.qk_norm_rope_backward(q[:, :3], k, q, k, wq, wk, cos, sin)


@pytest.mark.parametrize("T,H,Hk,D", [(710, 32, 8, 128), (709, 32, 8, 128), (1418, 32, 8, 64), (354, 32, 8, 256)])
def test_gradient_stays_in_its_workspace(cuda_device, T, H, Hk, D):
    """Sizes at which 16-bit types take every CTA of the GPU: nothing behind the workspace's bytes changes."""
    import ctypes
    from ctypes import c_int32, c_int64
    from solb200._lib import I64x2, I64x3, lib
    q, k, wq, wk, cos, sin = (t.cuda() for t in _inputs(1, T, H, Hk, D, D, torch.bfloat16, per_batch=False, seed=8))
    g = torch.Generator().manual_seed(9)
    dys = [torch.randn(t.shape, generator=g).bfloat16().cuda() for t in (q, k)]
    want = solb200.qk_norm_rope_backward(*dys, q, k, wq, wk, cos, sin)
    n = c_int64(0)
    assert lib().solb200_qk_norm_rope_backward_workspace(1, T, H, Hk, D, ctypes.byref(n)) == 0
    ws = torch.full((n.value + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    got = [torch.empty_like(t) for t in (q, k, wq, wk)]
    st = lambda t: I64x3(*t.stride()[:3])
    rc = lib().solb200_qk_norm_rope_backward(
        dys[0].data_ptr(), st(q), dys[1].data_ptr(), st(k), q.data_ptr(), st(q), k.data_ptr(), st(k), wq.data_ptr(),
        wk.data_ptr(), 0, cos.data_ptr(), sin.data_ptr(), I64x2(0, D // 2), *(t.data_ptr() for t in got), 1, T, H, Hk, D,
        D, c_int32(0), 1e-6, c_int32(1), ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (ws[n.value:] == 0xA5).all()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("B,T,H,Hk,D,R", [(1, 1, 1, 1, 64, 64), (3, 7, 5, 3, 128, 128), (2, 9, 3, 2, 80, 32),
                                          (1, 37, 9, 3, 256, 256), (1, 64, 8, 8, 64, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_gradient_without_eps(cuda_device, B, T, H, Hk, D, R, dtype, interleaved):
    """eps = 0, with numbers of rows that do and do not fill the last run: what does not exist adds
    nothing to the weights' gradients. Bounds as in test_gradient."""
    q, k, wq, wk, cos, sin = _inputs(B, T, H, Hk, D, R, dtype, seed=10)
    g = torch.Generator().manual_seed(11)
    dys = [torch.randn(t.shape, generator=g).to(dtype) for t in (q, k)]
    args = [t.cuda() for t in (q, k, wq, wk, cos, sin)]
    outs = solb200.qk_norm_rope(*args, eps=0.0, interleaved=interleaved)
    got = solb200.qk_norm_rope_backward(*(t.cuda() for t in dys), *args, eps=0.0, interleaved=interleaved)
    tc, ts = _tables(cos, sin, B)
    for y, dx, dw, dy, x, w in zip(outs, got[:2], got[2:], dys, (q, k), (wq, wk)):
        xd, wd = x.double(), w.double()
        want, r = _formula(xd, wd, tc, ts, interleaved, eps=0.0)
        _check(y, want, U[dtype] * want.abs() + 24 * 2.0 ** -24 * _partner(xd * r * wd, R, interleaved) + TINY[dtype], "y")
        gd = _turn(dy.double(), tc, -ts, interleaved)
        gm = _partner(dy.double(), R, interleaved)
        xh = xd * r
        want = r * (gd * wd - xh * (gd * wd * xh).mean(-1, keepdim=True))
        mags = r * (gm * wd.abs() + xh.abs() * (gm * wd.abs() * xh.abs()).mean(-1, keepdim=True))
        _check(dx, want, U[dtype] * want.abs() + 32 * 2.0 ** -24 * mags + TINY[dtype], "dx")
        want = (gd * xh).sum((0, 1, 2))
        _check(dw, want, U[dtype] * want.abs() + 256 * 2.0 ** -24 * (gm * xh.abs()).sum((0, 1, 2)) + TINY[dtype], "dw")
