"""Plain 64-bit forms of the attention-block operators on the inputs as they
lie in memory, with a bound on each output's error that follows from the
arithmetic: half a step of the output's type plus f32 rounding errors.

u(t) = finfo(t).eps / 2 is the largest relative error of one rounding to t."""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal step: roundings near zero are off by that much, whatever the value."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}[dtype]


def assert_close(got, ref, tol):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all(), "not finite"
    off = (got - ref).abs() - tol
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"beyond the bound by {worst:.3g} (largest difference {(got - ref).abs().max().item():.3g})"


def linear(x, w, bias=None, act=None, residual=None):
    """(value, bound). The K products of an output are summed in f32: at most
    K roundings of partial sums no larger than sum |x w|. Both activations
    have slopes within [-0.13, 1.13] and are computed from one f32
    exponential whose argument is at most ~90: relative 2^-17."""
    xd, wd = x.double(), w.double()
    pre = xd @ wd.T
    mag = xd.abs() @ wd.abs().T
    if bias is not None:
        pre, mag = pre + bias.double(), mag + bias.double().abs()
    tol = (x.shape[1] + 2) * U32 * mag
    y = pre
    if act == "silu":
        y = pre * torch.sigmoid(pre)
    elif act == "gelu":
        y = 0.5 * pre * (1 + torch.tanh(math.sqrt(2 / math.pi) * (pre + 0.044715 * pre ** 3)))
    if act:
        tol = 1.13 * tol + 2.0 ** -17 * y.abs() + 1e-30
    if residual is not None:
        y = y + residual.double()
        tol = tol + U32 * y.abs()
    return y, tol * (1 + u(x.dtype)) + u(x.dtype) * y.abs() + tiny(x.dtype)


def rope(x, coords, pairs, theta, layout, gain=None, eps=0.0):
    """(value, bound); x [rows, heads, D]. Sines and cosines are off by at
    most pi 2^-25 (the rounded half-turns) + 2^-23 (sincospi): below 2^-22.
    With the norm, the sum of D squares, its root and two products add (D + 8)
    roundings."""
    xd, d = x.double(), x.shape[-1]
    rel = 4 * U32
    if gain is not None:
        xd = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps) * gain.double()
        rel = rel + (d + 8) * U32
    angle = torch.zeros(x.shape[0], d // 2, dtype=torch.float64, device=x.device)
    at = 0
    for axis, n in enumerate(pairs):
        for j in range(n):
            angle[:, at] = coords[:, 1 + axis].double() * theta ** (-j / n)
            at += 1
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = (xd[..., 0::2], xd[..., 1::2]) if layout == "pairs" else (xd[..., :d // 2], xd[..., d // 2:])
    p, q = a * cos - b * sin, a * sin + b * cos
    mag = a.abs() + b.abs()
    y = torch.stack((p, q), -1).flatten(-2) if layout == "pairs" else torch.cat((p, q), -1)
    mag = torch.stack((mag, mag), -1).flatten(-2) if layout == "pairs" else torch.cat((mag, mag), -1)
    tol = (rel + 2.0 ** -22) * mag
    return y, tol * (1 + u(x.dtype)) + u(x.dtype) * y.abs() + tiny(x.dtype)


def attention(q, k, v, q_lens, kv_lens, scale):
    """(value, bound). An error d of a row's scores changes its weights by at
    most e^2d - 1 relative; scores are sums of D f32 products, scaled: d = (D +
    2) 2^-24 scale sum |q k| + 2^-20 |score| for the exponential's argument.
    Weights are rounded to the 16-bit type before the product with v (off by
    u relative, or by a subnormal half-step where they are kept as multiples
    of 2^8 at least), and summed in f32 (n roundings). All of that scales
    sum |p v|."""
    heads, d = q.shape[1], q.shape[2]
    out = torch.zeros(sum(q_lens), heads, d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    half = q.dtype != torch.float32
    for a, b in zip(q_lens, kv_lens):
        if a and b:
            qd, kd, vd = (t.double().transpose(0, 1) for t in (q[q0:q0 + a], k[k0:k0 + b], v[k0:k0 + b]))
            s = qd @ kd.transpose(1, 2) * scale
            p = torch.softmax(s, -1)
            mag = qd.abs() @ kd.abs().transpose(1, 2) * abs(scale)
            delta = ((d + 2) * U32 * mag + 2.0 ** -20 * s.abs()).amax(-1, keepdim=True)
            o, om = p @ vd, p @ vd.abs()
            rel = 2.5 * delta + (b + 8) * U32 + 2.0 ** -20
            under = 0.0
            if half:
                rel = rel + u(q.dtype)
                under = tiny(q.dtype) * 2.0 ** -8 * vd.abs().sum(1, keepdim=True)
            t = rel * om + under
            out[q0:q0 + a], tol[q0:q0 + a] = o.transpose(0, 1), t.transpose(0, 1)
        q0, k0 = q0 + a, k0 + b
    return out, tol * (1 + u(q.dtype)) + u(q.dtype) * out.abs() + tiny(q.dtype)
