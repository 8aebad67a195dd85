"""Float64 restatements of the decoder's operators (norm with rotation, cross
attention, 4-bit projection) and their gradients, with bounds of what 16-bit
roundings and fp32 sums may cost.  Test infrastructure only.

Functions take tensors of any device and type and compute in float64.
"""

from __future__ import annotations

import torch


# ---- norm and rotation -------------------------------------------------------------


def rotate(x, cos, sin, interleaved, back=False):
    """x [..., L, D], its first 2 * cos.shape[-1] dimensions turned by the angles of cos, sin [..., L, R / 2]."""
    half = cos.shape[-1]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    if back:
        sin = -sin
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _angles(x, cos, sin, pos):
    """cos, sin [B, 1, L, R / 2] of each token and whether it is there [B, 1, L, 1]."""
    b, _, l, _ = x.shape
    if pos is None:
        pos = torch.arange(l, device=x.device).expand(b, l)
    there = (pos >= 0).view(b, 1, l, 1)
    if cos is None:
        empty = torch.zeros(b, 1, l, 0, dtype=torch.float64, device=x.device)
        return empty, empty, there
    at = pos.long().clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at].unsqueeze(1), sin.double()[at].unsqueeze(1)
    past = (pos >= cos.shape[0]).view(b, 1, l, 1)
    return c.masked_fill(past, float("nan")), s.masked_fill(past, float("nan")), there


def norm_rotary(x, w, cos, sin, pos, eps, interleaved):
    """-> (y, size): y [B, H, L, D], and the magnitude that its fp32 arithmetic errs in proportion to."""
    x, w = x.double(), w.double()
    c, s, there = _angles(x, cos, sin, pos)
    n = torch.where(there, x, 0.0)
    n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + eps)
    y = torch.where(there, rotate(w * n, c, s, interleaved), 0.0)
    size = torch.where(there, rotate((w * n).abs(), c.abs(), -s.abs(), interleaved).abs()
                       + rotate((w * n).abs(), c.abs(), s.abs(), interleaved).abs(), 0.0)
    return y, size


def norm_rotary_grads(dy, x, w, cos, sin, pos, eps, interleaved):
    """-> (dx, size of dx, dw, size of dw)."""
    dy, x, w = dy.double(), x.double(), w.double()
    c, s, there = _angles(x, cos, sin, pos)
    x = torch.where(there, x, 0.0)
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r
    g = torch.where(there, rotate(torch.where(there, dy, 0.0), c, s, interleaved, back=True), 0.0)
    big = torch.where(there, rotate(torch.where(there, dy, 0.0).abs(), c.abs(), s.abs(), interleaved).abs()
                      + rotate(torch.where(there, dy, 0.0).abs(), c.abs(), -s.abs(), interleaved).abs(), 0.0)
    dx = r * (w * g - n * (w * g * n).mean(-1, keepdim=True))
    size = r * (w.abs() * big + n.abs() * (w.abs() * big * n.abs()).mean(-1, keepdim=True))
    return dx, size, (g * n).sum((0, 1, 2)), (big * n.abs()).sum((0, 1, 2))


# ---- cross attention ---------------------------------------------------------------


def _lengths(lens, batch, most):
    return [most] * batch if lens is None else [min(max(int(n), 0), most) for n in lens]


def cross(q, k, v, lens, q_lens, scale):
    """-> (out, softmax |v|, lse), per item over its valid queries and keys, zeros (and -inf) elsewhere."""
    b, h, l, d = q.shape
    g, s = k.shape[1], k.shape[2]
    out = torch.zeros(b, h, l, d, dtype=torch.float64, device=q.device)
    size, lse = torch.zeros_like(out), torch.full((b, h, l), float("-inf"), dtype=torch.float64, device=q.device)
    for i, (n, m) in enumerate(zip(_lengths(lens, b, s), _lengths(q_lens, b, l))):
        for j in range(h if n and m else 0):
            logits = scale * (q[i, j, :m].double() @ k[i, j // (h // g), :n].double().t())
            p, val = torch.softmax(logits, -1), v[i, j // (h // g), :n].double()
            out[i, j, :m], size[i, j, :m], lse[i, j, :m] = p @ val, p @ val.abs(), torch.logsumexp(logits, -1)
    return out, size, lse


def cross_grads(dout, q, k, v, lens, q_lens, scale, u):
    """-> {name: (gradient, bound of its error)} for roundings by ``u`` of the value.

    Scores of a few units in fp32 move a probability, and with it lse, by less than
    2^-12 of itself; P and dS are rounded by u.  delta = dout . out is off by what
    the forward call's out is, (u + 2^-12) softmax |v| + u |out|, times |dout|; dP by
    fp32's D products, under 2^-16 of sum |dout| |v|.  So
      dS is off by (u + 2^-12) |dS| + P (|delta's error| + 2^-16 |dout| . |v|),
    dq, dk by that times |k|, |q|, dv by (u + 2^-12) P^T |dout|, and each by u of itself."""
    b, h, l, d = q.shape
    g, s = k.shape[1], k.shape[2]
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    grads = {name: [zero(t), zero(t)] for name, t in (("dq", q), ("dk", k), ("dv", v))}
    e = u + 2.0 ** -12
    for i, (n, m) in enumerate(zip(_lengths(lens, b, s), _lengths(q_lens, b, l))):
        for j in range(h if n and m else 0):
            c = j // (h // g)
            qq, do, kk, vv = (t.double() for t in (q[i, j, :m], dout[i, j, :m], k[i, c, :n], v[i, c, :n]))
            p = torch.softmax(scale * (qq @ kk.t()), -1)
            o, dp = p @ vv, do @ vv.t()
            ds = p * (dp - (do * o).sum(-1, keepdim=True))
            off = (do.abs() * (e * (p @ vv.abs()) + u * o.abs())).sum(-1, keepdim=True)
            off = e * ds.abs() + p * (off + 2.0 ** -16 * (do.abs() @ vv.abs().t()))
            for name, at, value, bound in (("dq", (i, j, slice(m)), scale * (ds @ kk), scale * (off @ kk.abs())),
                                           ("dk", (i, c, slice(n)), scale * (ds.t() @ qq), scale * (off.t() @ qq.abs())),
                                           ("dv", (i, c, slice(n)), p.t() @ do, e * (p.t() @ do.abs()))):
                grads[name][0][at] += value
                grads[name][1][at] += bound
    return {name: (value, bound + u * value.abs()) for name, (value, bound) in grads.items()}


def sharp_cross_grads(dout, q, k, v, lens, q_lens, scale, u):
    """cross_grads' gradients -> {name: (gradient, bound)} with bounds that hold delta to fp32.

    Scores s of at most A = max scale |q| . |k| (over a query's keys) go through D / 16 <= 8 sums of 16 products, a
    scale, lse (its logarithm, two scalings) and an exponential: under 32 half steps of fp32 of A + 1, so
    P is off by e = 2^-19 (A + 1) of itself, dP (8 sums) by m = 2^-20 |dout| . |v|.  delta starts
    from dout . out, off by 2 u |dout| . softmax |v| at most (the forward call's roundings of P and out), and is
    corrected by the sum of P (dP - dout . out), of up to 2^11 terms one after another:
      delta is off by (e + 2^-12) (P |dP - delta| + 2 u |dout| . softmax |v|) + P m.
    dS = P (dP - delta) is off by (u + e) of itself and P (m + delta's).  fp16 holds P times 2^15, off by
    2^-40 where it is small, and dS times the power of two that brings 2 |dout| |v| of the longest rows
    (dk: of all the heads that share the key) to 1/2 or more, off by 2^-38 |dout| |v|."""
    b, h, l, d = q.shape
    g, s = k.shape[1], k.shape[2]
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    grads = {name: [zero(t), zero(t)] for name, t in (("dq", q), ("dk", k), ("dv", v))}
    small = u == 2.0 ** -11
    for i, (n, m) in enumerate(zip(_lengths(lens, b, s), _lengths(q_lens, b, l))):
        for j in range(h if n and m else 0):
            c = j // (h // g)
            qq, do, kk, vv = (t.double() for t in (q[i, j, :m], dout[i, j, :m], k[i, c, :n], v[i, c, :n]))
            p = torch.softmax(scale * (qq @ kk.t()), -1)
            e = 2.0 ** -19 * (1 + (scale * (qq.abs() @ kk.abs().t())).amax(-1, keepdim=True))
            dp, dp_off = do @ vv.t(), 2.0 ** -20 * (do.abs() @ vv.abs().t())
            from_delta = dp - (p * dp).sum(-1, keepdim=True)
            ds = p * from_delta
            start = 2 * u * (do.abs() * (p @ vv.abs())).sum(-1, keepdim=True)
            off = (e + 2.0 ** -12) * (ds.abs().sum(-1, keepdim=True) + start) + (p * dp_off).sum(-1, keepdim=True)
            off = (u + e) * ds.abs() + p * (dp_off + off)
            heads = slice(c * (h // g), (c + 1) * (h // g))
            longest_v, longest = vv.norm(dim=-1).max(), dout[i, heads, :m].double().norm(dim=-1).max()
            dq_off = off + small * 2.0 ** -38 * do.norm(dim=-1, keepdim=True) * longest_v
            dk_off = off + small * 2.0 ** -38 * longest * longest_v
            p_off = (u + e) * p + small * 2.0 ** -40
            for name, at, value, bound in (("dq", (i, j, slice(m)), scale * (ds @ kk), scale * (dq_off @ kk.abs())),
                                           ("dk", (i, c, slice(n)), scale * (ds.t() @ qq), scale * (dk_off.t() @ qq.abs())),
                                           ("dv", (i, c, slice(n)), p.t() @ do, p_off.t() @ do.abs())):
                grads[name][0][at] += value
                grads[name][1][at] += bound
    return {name: (value, bound + u * value.abs()) for name, (value, bound) in grads.items()}


# ---- 4-bit projection --------------------------------------------------------------


def int4(x, values, scales, zeros, bias, act):
    """-> (y, size): the projection in float64, and sum |x| |w - z| s for its fp32 sums."""
    group = values.shape[1] // scales.shape[1]
    w = values.double().unflatten(1, (-1, group))
    z = torch.full_like(scales, 8).double() if zeros is None else zeros.double()
    w = ((w - z.unsqueeze(-1)) * scales.double().unsqueeze(-1)).flatten(1)
    y = x.double() @ w.t()
    size = x.double().abs() @ (scales.double().abs().repeat_interleave(group, 1) * 16).t()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    if act == "silu":
        y = y / (1 + torch.exp(-y))
    return y, size
