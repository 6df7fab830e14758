"""What is measured of the streaming-attention operators: head norms with the position rotation
(``solb200.qk_norm_rope`` and its gradient) and sliding-window attention with sinks
(``solb200.window_attn``: whole sequences, its gradient, single new tokens over a cache).

Positions: query i of sequence b sits at p = offsets[b] + i and sees key j when
j < lengths[b], j <= p + right, and j >= p - left or j < sinks (a bound of None is absent).
In a case, a bound of -1 is absent, lengths is a text of one number per sequence ("": all of the
cache), and offsets are 0 (from_start) or put the last query at the last key.
"""

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one new token of each of 8 sequences in serving: latency is what counts
        dict(name="rotate_token", op="rotate", B=8, T=1, H=40, Hk=8, D=128, R=128, dtype="bf16",
             interleaved=False, per_batch=True),
        # two ragged prompts of a small text model in 32 bits, half of each head rotated
        dict(name="rotate_ragged", op="rotate", B=2, T=1013, H=12, Hk=4, D=64, R=32, dtype="f32",
             interleaved=False, per_batch=False),
        # the 480p video configuration: 21 x 30 x 52 tokens, 40 heads
        dict(name="rotate_video", op="rotate", B=1, T=32760, H=40, Hk=40, D=128, R=128, dtype="bf16",
             interleaved=True, per_batch=False),
        # a training step of a grouped-head model in f16, odd length
        dict(name="rotate_grad_odd", op="rotate_grad", B=2, T=777, H=15, Hk=5, D=64, R=64, dtype="f16",
             interleaved=False, per_batch=True),
        # a training step of the image configuration: 64 x 64 tokens, 24 heads, four images
        dict(name="rotate_grad_image", op="rotate_grad", B=4, T=4096, H=24, Hk=24, D=128, R=128,
             dtype="bf16", interleaved=True, per_batch=False),
        # four right-padded prompts of a small text model, causal, short window
        dict(name="window_text", op="window", B=4, Tq=333, Tk=333, H=16, Hk=4, D=64, left=127, right=0,
             sinks=4, lengths="333 300 97 1", from_start=True),
        # one new frame (30 x 52 tokens) of a streamed video against the window of frames before it
        # and the first frame, in a cache of 32760 tokens
        dict(name="window_chunk", op="window", B=1, Tq=1560, Tk=32760, H=40, Hk=40, D=128, left=10920,
             right=-1, sinks=1560, lengths="28080", from_start=False),
        # a whole 480p video, every token seeing one and a half frames each way and the first frame
        dict(name="window_video", op="window", B=1, Tq=32760, Tk=32760, H=40, Hk=40, D=128, left=2340,
             right=2340, sinks=1560, lengths="", from_start=False),
        # a training step on ragged right-padded sequences, one of them empty, grouped heads
        dict(name="window_grad_ragged", op="window_grad", B=4, Tq=517, Tk=517, H=12, Hk=4, D=64, left=200,
             right=0, sinks=3, lengths="517 260 1 0", from_start=True),
        # a training step of the image configuration with a causal window of a quarter of it
        dict(name="window_grad_image", op="window_grad", B=4, Tq=4096, Tk=4096, H=24, Hk=24, D=128,
             left=1023, right=0, sinks=64, lengths="", from_start=False),
        # one new token of each of 16 sequences over caches of many lengths, sliding window
        dict(name="window_tokens", op="window", B=16, Tq=1, Tk=32768, H=40, Hk=8, D=128, left=4095, right=0,
             sinks=4, lengths="32768 1 5 100 4096 4097 4101 9999 20000 31000 2 513 7777 16384 24576 3000",
             from_start=False),
        # one new token over one long cache, no window: the longest read of a single row
        dict(name="window_token_long", op="window", B=1, Tq=1, Tk=262144, H=40, Hk=40, D=128, left=-1,
             right=0, sinks=0, lengths="262001", from_start=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    Hk = _log_int(rng, 1, most)
    G = rng.choice([1, 1, 2, 3, 4, 5, 8])
    return (Hk * G, Hk) if Hk * G <= 48 else (Hk, Hk)


def draw(rng):
    op = rng.choice(["rotate", "rotate_grad", "window", "window", "window_grad", "token"])
    D = rng.choice([64, 128])
    if op in ("rotate", "rotate_grad"):
        H, Hk = _heads(rng, 40)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        B = rng.randint(1, 8)
        # up to the listed video (image) case's elements
        most = (32760 * 80 if op == "rotate" else 4 * 4096 * 48) * 128 // (2 if dtype == "f32" else 1)
        T = _log_int(rng, 1, max(1, min(32760, most // (B * (H + Hk) * D))))
        return dict(op=op, B=B, T=T, H=H, Hk=Hk, D=D, R=rng.choice([D, D, D // 2]), dtype=dtype,
                    interleaved=rng.random() < 0.5, per_batch=rng.random() < 0.5)
    if op == "token":
        B = _log_int(rng, 1, 64)
        H, Hk = _heads(rng, 40)
        # the cache: up to the listed long cache's bytes
        Tk = _log_int(rng, 1, max(1, min(262144, 262144 * 40 * 128 // (B * Hk * D))))
        left = -1 if rng.random() < 0.3 else _log_int(rng, 1, 16384)
        return dict(op="window", B=B, Tq=1, Tk=Tk, H=H, Hk=Hk, D=D, left=left, right=0,
                    sinks=rng.choice([0, 1, 4, 64]),
                    lengths=" ".join(str(_log_int(rng, 1, Tk)) for _ in range(B)), from_start=False)
    B = rng.randint(1, 4)
    H, Hk = _heads(rng, 24)
    grad = op == "window_grad"
    Tk = _log_int(rng, 2, 4096 if grad else 32760)
    whole = grad or rng.random() < 0.7
    Tq = Tk if whole else _log_int(rng, 1, min(Tk, 4096))
    left = -1 if rng.random() < 0.15 else _log_int(rng, 1, 4096)
    right = rng.choice([0, 0, -1, left])
    sinks = rng.choice([0, 1, 4, 64, 1560])
    case = dict(op=op, B=B, Tq=Tq, Tk=Tk, H=H, Hk=Hk, D=D, left=left, right=right, sinks=sinks,
                lengths="", from_start=False)
    if rng.random() < 0.5:
        case["lengths"] = " ".join(str(rng.randint(0 if whole else Tq, Tk)) for _ in range(B))
        case["from_start"] = whole
    # no more than the listed cases' products (or the plain form's temporaries)
    most = 4 * 4096 * 1088 * 24 * 128 if grad else 32760 * 6240 * 40 * 128
    while _pairs(case) * H * D > most or B * H * Tq * D > 32760 * 40 * 128:
        H = max(1, H // 2)
        Hk = max(1, min(Hk, H))
        H = Hk * max(1, H // Hk)
        if H == 1 and case["B"] > 1:
            B = case["B"] = case["B"] // 2
            case["lengths"] = " ".join(case["lengths"].split()[:B])
        case["H"], case["Hk"] = H, Hk
    return case


def _lengths(case):
    return [int(n) for n in case["lengths"].split()] or [case["Tk"]] * case["B"]


def _offsets(case):
    return [0 if case["from_start"] else n - case["Tq"] for n in _lengths(case)]


def _bounds(case):
    """(left, right) as the calls take them."""
    return tuple(None if case[n] < 0 else case[n] for n in ("left", "right"))


def _visible(case, b):
    """For sequence b: (pairs of a query and a key that it sees, keys that some query sees)."""
    L, off, Tq = _lengths(case)[b], _offsets(case)[b], case["Tq"]
    (left, right), sinks = _bounds(case), case["sinks"]
    pairs, top, low = 0, 0, L
    for i in range(Tq):
        p = off + i
        hi = L if right is None else max(0, min(L, p + right + 1))
        lo = 0 if left is None else max(0, min(hi, p - left))
        pairs += hi - lo + min(sinks, lo)
        if hi > lo:
            top, low = max(top, hi), min(low, lo)
    keys = max(0, top - low) + min(sinks, low, L)
    return pairs, keys


def _pairs(case):
    return sum(_visible(case, b)[0] for b in range(case["B"]))


def work(case):
    if case["op"] in ("rotate", "rotate_grad"):
        rows = case["B"] * case["T"] * (case["H"] + case["Hk"])
        es = DTYPES[case["dtype"]].itemsize
        table = case["T"] * (case["B"] if case["per_batch"] else 1) * case["R"] * 4
        passes = 2 if case["op"] == "rotate" else 3      # x, y; or dy, x, dx
        ops = 6 if case["op"] == "rotate" else 14
        small = 2 * case["D"] * es * (1 if case["op"] == "rotate" else 2)
        return {"bytes": passes * rows * case["D"] * es + table + small, "flops": ops * rows * case["D"]}
    seen = [_visible(case, b) for b in range(case["B"])]
    pairs, keys = sum(s[0] for s in seen), sum(s[1] for s in seen)
    q_bytes = case["B"] * case["Tq"] * case["H"] * case["D"] * 2
    kv_bytes = 2 * keys * case["Hk"] * case["D"] * 2
    if case["op"] == "window":
        return {"bytes": 2 * q_bytes + kv_bytes, "flops": 4 * pairs * case["H"] * case["D"]}
    kv_out = 2 * case["B"] * case["Tk"] * case["Hk"] * case["D"] * 2
    # q, dout read, out, dq written; k, v read, dk, dv written; 2 products forward, 4 backward
    return {"bytes": 4 * q_bytes + kv_bytes + kv_out, "flops": 12 * pairs * case["H"] * case["D"]}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = _gen(seed)
    state = dict(case=case)
    if case["op"] in ("rotate", "rotate_grad"):
        B, T, H, Hk, D, R = (case[n] for n in ("B", "T", "H", "Hk", "D", "R"))
        dtype = DTYPES[case["dtype"]]
        # q and k as a projection leaves them: views of one packed [B, T, (H + 2 Hk) * D] tensor
        qkv = torch.empty((B, T, (H + 2 * Hk) * D), device="cuda", dtype=dtype)
        for b in range(B):
            qkv[b] = _randn((T, (H + 2 * Hk) * D), gen, dtype)
        state["q"] = qkv[..., :H * D].view(B, T, H, D)
        state["k"] = qkv[..., H * D:(H + Hk) * D].view(B, T, Hk, D)
        state["wq"] = (1.0 + 0.2 * _randn((D,), gen, torch.float32)).to(dtype)
        state["wk"] = (1.0 + 0.2 * _randn((D,), gen, torch.float32)).to(dtype)
        # angles: position times a falling frequency, every sequence at a place of its own
        start = torch.randint(0, 4096, (B if case["per_batch"] else 1, 1), generator=gen, device="cuda")
        pos = (start + torch.arange(T, device="cuda")).double()
        freq = 10000.0 ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64) / (R // 2))
        angle = pos[..., None] * freq
        cos, sin = angle.cos().float(), angle.sin().float()
        state["cos"], state["sin"] = (cos, sin) if case["per_batch"] else (cos[0], sin[0])
        if case["op"] == "rotate_grad":
            state["dq"] = _randn((B, T, H, D), gen, dtype)
            state["dk"] = _randn((B, T, Hk, D), gen, dtype)
        return state
    B, Tq, Tk, H, Hk, D = (case[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
    bf16 = torch.bfloat16
    # normed heads: unit variance; what lies behind a sequence's length is left from earlier use
    state["q"] = _randn((B, Tq, H, D), gen, bf16)
    state["k"] = torch.empty((B, Tk, Hk, D), device="cuda", dtype=bf16)
    state["v"] = torch.empty((B, Tk, Hk, D), device="cuda", dtype=bf16)
    for b in range(B):
        state["k"][b] = _randn((Tk, Hk, D), gen, bf16)
        state["v"][b] = _randn((Tk, Hk, D), gen, bf16)
    state["lengths"] = state["offsets"] = None
    if case["lengths"]:
        state["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    if case["from_start"]:
        state["offsets"] = torch.tensor(_offsets(case), device="cuda", dtype=torch.int32)
    if case["op"] == "window_grad":
        state["dout"] = _randn((B, Tq, H, D), gen, bf16)
    return state


# ------------------------------------------------------ the framework's own

_solb200 = None


def _own():
    global _solb200
    if _solb200 is None:
        pkg = str(Path(__file__).resolve().parent.parent / "comfyui-solattn_triton_b200")
        if pkg not in sys.path:
            sys.path.insert(1, pkg)
        import solb200
        _solb200 = solb200
    return _solb200


def _run_own(s):
    lib, case = _own(), s["case"]
    if case["op"] == "rotate":
        return lib.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], eps=EPS,
                                interleaved=case["interleaved"])
    if case["op"] == "rotate_grad":
        return lib.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"],
                                         eps=EPS, interleaved=case["interleaved"])
    left, right = _bounds(case)
    how = dict(left=left, right=right, sinks=case["sinks"], lengths=s["lengths"],
               offsets=s["offsets"])
    if case["op"] == "window":
        return lib.window_attn(s["q"], s["k"], s["v"], **how)
    out, lse = lib.window_attn(s["q"], s["k"], s["v"], return_lse=True, **how)
    return (out, *lib.window_attn_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how))


# ------------------------------------------------------------- plain forms

def _turn(x, cos, sin, interleaved):
    """x [..., H, D] with its first R elements of each head turned by the tables' angles."""
    R = 2 * cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * c - b * s, a * s + b * c
    y = torch.stack((ya, yb), dim=-1).flatten(-2) if interleaved else torch.cat((ya, yb), dim=-1)
    return y if R == x.shape[-1] else torch.cat((y, x[..., R:]), dim=-1)


def _plain_rotate(s):
    outs = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        xf = x.float()
        n = xf * torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + EPS) * w.float()
        outs.append(_turn(n, s["cos"], s["sin"], s["case"]["interleaved"]).to(x.dtype))
    return tuple(outs)


def _plain_rotate_grad(s):
    grads, weights = [], []
    for dy, x, w in ((s["dq"], s["q"], s["wq"]), (s["dk"], s["k"], s["wk"])):
        xf, wf = x.float(), w.float()
        rstd = torch.rsqrt((xf * xf).mean(dim=-1, keepdim=True) + EPS)
        xhat = xf * rstd
        g = _turn(dy.float(), s["cos"], -s["sin"], s["case"]["interleaved"])
        weights.append((g * xhat).sum(dim=(0, 1, 2)).to(w.dtype))
        gw = g * wf
        grads.append((rstd * (gw - xhat * (gw * xhat).mean(dim=-1, keepdim=True))).to(x.dtype))
    return (*grads, *weights)


def _places(s):
    """Lengths and offsets as int64 tensors [B, 1]."""
    case = s["case"]
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    if s["lengths"] is None:
        L = torch.full((B, 1), Tk, device="cuda", dtype=torch.int64)
    else:
        L = s["lengths"].long().view(B, 1)
    return L, L - Tq if s["offsets"] is None else s["offsets"].long().view(B, 1)


def _chunks(s):
    """Per run of query rows: (first row, end row, key indices [B, n] or None for all keys, which
    of them each row sees [B, rows, n])."""
    case = s["case"]
    B, Tq, Tk, H = case["B"], case["Tq"], case["Tk"], case["H"]
    (left, right), sinks = _bounds(case), min(case["sinks"], case["Tk"])
    L, off = _places(s)
    rows = Tq
    while rows > 1:      # about 2^28 scores at a time
        n = min(Tk, Tk if None in (left, right) else sinks + left + right + rows)
        if B * H * rows * n <= 1 << 28:
            break
        rows = -(-rows // 2)
    for i0 in range(0, Tq, rows):
        i1 = min(Tq, i0 + rows)
        p = off + torch.arange(i0, i1, device="cuda")                       # [B, rows]
        span = Tk if None in (left, right) else sinks + left + right + (i1 - i0)
        if span >= Tk:
            idx, j = None, torch.arange(Tk, device="cuda").expand(B, Tk)
            good = torch.ones_like(j, dtype=torch.bool)
        else:
            first = torch.arange(sinks, device="cuda").expand(B, sinks)
            near = off + i0 - left + torch.arange(span - sinks, device="cuda")
            j = torch.cat((first, near), dim=1)
            good = torch.cat((torch.ones_like(first, dtype=torch.bool), near >= sinks), dim=1)
            idx = j.clamp(0, Tk - 1)
        jj, pp = j[:, None, :], p[:, :, None]
        see = (good[:, None, :] & (jj >= 0) & (jj < L[:, :, None])).expand(-1, i1 - i0, -1)
        if right is not None:
            see = see & (jj <= pp + right)
        if left is not None:
            see = see & ((jj >= pp - left) | (jj < sinks))
        yield i0, i1, idx, see


def _pick(x, idx):
    """Rows idx [B, n] of x [B, T, Hk, D], in 32 bits, as [B, Hk, n, D]."""
    if idx is not None:
        x = torch.gather(x, 1, idx[:, :, None, None].expand(-1, -1, x.shape[2], x.shape[3]))
    return x.float().transpose(1, 2)


def _group(x, Hk):
    """[B, rows, H, D] in 32 bits as [B, Hk, G * rows, D]."""
    B, rows, H, D = x.shape
    return x.float().view(B, rows, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)


def _ungroup(x, rows):
    B, Hk, GR, D = x.shape
    return x.view(B, Hk, GR // rows, rows, D).permute(0, 3, 1, 2, 4).reshape(B, rows, -1, D)


def _weights(q, k, see, G):
    """softmax over the seen keys of q k^T / sqrt(D); a row that sees nothing is zero."""
    B, Hk, GR, D = q.shape
    score = (q @ k.transpose(-1, -2)) * D ** -0.5
    see = see[:, None, None].expand(B, Hk, G, -1, -1).reshape(B, Hk, GR, -1)
    score.masked_fill_(~see, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_window(s):
    case, q = s["case"], s["q"]
    Hk, G = case["Hk"], case["H"] // case["Hk"]
    out = torch.empty_like(q)
    for i0, i1, idx, see in _chunks(s):
        P = _weights(_group(q[:, i0:i1], Hk), _pick(s["k"], idx), see, G)
        out[:, i0:i1] = _ungroup(P @ _pick(s["v"], idx), i1 - i0).to(q.dtype)
    return out


def _plain_window_grad(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    Hk, G, D = case["Hk"], case["H"] // case["Hk"], case["D"]
    out, dq = torch.empty_like(q), torch.empty_like(q)
    dk = torch.zeros((case["B"], case["Tk"], Hk, D), device="cuda")
    dv = torch.zeros_like(dk)
    for i0, i1, idx, see in _chunks(s):
        qc, kc, vc = _group(q[:, i0:i1], Hk), _pick(k, idx), _pick(v, idx)
        do = _group(s["dout"][:, i0:i1], Hk)
        P = _weights(qc, kc, see, G)
        o = P @ vc
        out[:, i0:i1] = _ungroup(o, i1 - i0).to(q.dtype)
        dS = P * (do @ vc.transpose(-1, -2) - (do * o).sum(dim=-1, keepdim=True)) * D ** -0.5
        dq[:, i0:i1] = _ungroup(dS @ kc, i1 - i0).to(q.dtype)
        for total, part in ((dk, dS.transpose(-1, -2) @ qc), (dv, P.transpose(-1, -2) @ do)):
            part = part.transpose(1, 2)
            if idx is None:
                total += part
            else:
                total.scatter_add_(1, idx[:, :, None, None].expand(-1, -1, Hk, D), part)
    return out, dq, dk.to(k.dtype), dv.to(v.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"rotate": _plain_rotate, "rotate_grad": _plain_rotate_grad, "window": _plain_window,
            "window_grad": _plain_window_grad}[state["case"]["op"]](state)


# ------------------------------------------------------------------ 64 bits

def _exact_rotate(s):
    """The rotation as a product of complex numbers; gradients through autograd in 64 bits."""
    case = s["case"]
    turn = torch.complex(s["cos"].double(), s["sin"].double())
    if turn.dim() == 2:
        turn = turn.expand(case["B"], -1, -1)
    R = case["R"]

    def forward(x, w, b):
        n = x / (x.square().sum(-1, keepdim=True) / case["D"] + EPS).sqrt() * w
        r = n[..., :R]
        pair = r.unflatten(-1, (R // 2, 2)) if case["interleaved"] else r.unflatten(-1, (2, R // 2)).movedim(-2, -1)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[b][:, None, :])
        y = z.flatten(-2) if case["interleaved"] else z.movedim(-1, -2).flatten(-2)
        return torch.cat((y, n[..., R:]), dim=-1)

    ys, dxs, dws = [], [], []
    grad = case["op"] == "rotate_grad"
    for name, wname in (("q", "wq"), ("k", "wk")):
        w = s[wname].double().requires_grad_(grad)
        y, dx, dw = [], [], torch.zeros_like(w)
        for b in range(case["B"]):
            x = s[name][b].double().requires_grad_(grad)
            with torch.set_grad_enabled(grad):
                yb = forward(x, w, b)
            if grad:
                gx, gw = torch.autograd.grad(yb, (x, w), s["d" + name][b].double())
                dx.append(gx)
                dw = dw + gw
            else:
                y.append(yb)
        ys.append(torch.stack(y) if y else None)
        dxs.append(torch.stack(dx) if dx else None)
        dws.append(dw.detach())
    return (*dxs, *dws) if grad else tuple(ys)


def _exact_window(s):
    """One head at a time, in runs of rows against every key up to the sequence's length."""
    case = s["case"]
    B, Tq, H, D = case["B"], case["Tq"], case["H"], case["D"]
    G = H // case["Hk"]
    left, right = _bounds(case)
    grad = case["op"] == "window_grad"
    out = torch.zeros((B, Tq, H, D), device="cuda", dtype=torch.float64)
    dq = torch.zeros_like(out) if grad else None
    dk = torch.zeros((B, case["Tk"], case["Hk"], D), device="cuda", dtype=torch.float64) if grad else None
    dv = torch.zeros_like(dk) if grad else None
    for b in range(B):
        L, off = _lengths(case)[b], _offsets(case)[b]
        if L == 0:
            continue
        j = torch.arange(L, device="cuda")
        rows = max(1, min(Tq, (1 << 26) // L))
        for i0 in range(0, Tq, rows):
            p = off + torch.arange(i0, min(Tq, i0 + rows), device="cuda")[:, None]
            hide = torch.zeros((len(p), L), device="cuda", dtype=torch.bool)
            if right is not None:
                hide |= j > p + right
            if left is not None:
                hide |= (j < p - left) & (j >= case["sinks"])
            keep = torch.nonzero(~hide.all(dim=0)).flatten()
            if len(keep) == 0:
                continue
            lo, hi = int(keep[0]), int(keep[-1]) + 1
            hide = hide[:, lo:hi]
            empty = hide.all(dim=1, keepdim=True)
            for h in range(H):
                q = s["q"][b, i0:i0 + rows, h].double()
                k, v = s["k"][b, lo:hi, h // G].double(), s["v"][b, lo:hi, h // G].double()
                z = (q @ k.T) / math.sqrt(D)
                P = torch.softmax(z.masked_fill(hide & ~empty, -math.inf), dim=-1).masked_fill(empty, 0.0)
                o = P @ v
                out[b, i0:i0 + rows, h] = o
                if grad:
                    do = s["dout"][b, i0:i0 + rows, h].double()
                    dP = do @ v.T
                    dz = P * (dP - (P * dP).sum(dim=-1, keepdim=True)) / math.sqrt(D)
                    dq[b, i0:i0 + rows, h] = dz @ k
                    dk[b, lo:hi, h // G] += dz.T @ q
                    dv[b, lo:hi, h // G] += P.T @ do
    return (out, dq, dk, dv) if grad else out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotate(s) if case["op"] in ("rotate", "rotate_grad") else _exact_window(s)
