"""The decoder oracle against torch's autograd, differences and closed forms (no GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import decoder_oracle as oracle


def _tables(places, rot, seed=0):
    angle = torch.rand(places, rot // 2, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 6
    return angle.cos(), angle.sin()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_one(interleaved):
    """Turning there and back, lengths kept, and the angles' sum."""
    x = torch.randn(2, 3, 5, 32, dtype=torch.float64)
    cos, sin = _tables(5, 16)
    y = oracle.rotate(x, cos, sin, interleaved)
    torch.testing.assert_close(oracle.rotate(y, cos, sin, interleaved, back=True), x)
    torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
    assert torch.equal(y[..., 16:], x[..., 16:])
    twice = oracle.rotate(y, cos, sin, interleaved)
    torch.testing.assert_close(twice, oracle.rotate(x, cos * cos - sin * sin, 2 * sin * cos, interleaved))
    pair = (0, 1) if interleaved else (0, 8)
    z = torch.complex(x[0, 0, 2, pair[0]], x[0, 0, 2, pair[1]]) * torch.complex(cos[2, 0], sin[2, 0])
    torch.testing.assert_close(torch.view_as_real(z), y[0, 0, 2, list(pair)])


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_gradients(interleaved):
    x = torch.randn(2, 3, 4, 32, dtype=torch.float64, requires_grad=True)
    w = torch.randn(32, dtype=torch.float64, requires_grad=True)
    cos, sin = _tables(9, 16)
    pos = torch.tensor([[3, 4, -1, 8], [0, -1, 2, 2]], dtype=torch.int32)
    dy = torch.randn(2, 3, 4, 32, dtype=torch.float64)
    y, size = oracle.norm_rotary(x, w, cos, sin, pos, 1e-3, interleaved)
    assert (y.abs() <= size + 1e-12).all() and (y[0, :, 2] == 0).all()
    want = torch.autograd.grad((y * dy).sum(), (x, w))
    dx, dx_size, dw, dw_size = oracle.norm_rotary_grads(dy, x.detach(), w.detach(), cos, sin, pos, 1e-3, interleaved)
    torch.testing.assert_close(dx, want[0])
    torch.testing.assert_close(dw, want[1])
    assert (dx.abs() <= dx_size + 1e-12).all() and (dw.abs() <= dw_size + 1e-12).all()
    with torch.no_grad():
        f = lambda x, w: (oracle.norm_rotary(x, w, cos, sin, pos, 1e-3, interleaved)[0] * dy).sum()  # noqa: E731
        step, h = torch.randn_like(x), 1e-6
        torch.testing.assert_close((f(x + h * step, w) - f(x - h * step, w)) / (2 * h), (dx * step).sum(), rtol=1e-6, atol=1e-7)
        step = torch.randn_like(w)
        torch.testing.assert_close((f(x, w + h * step) - f(x, w - h * step)) / (2 * h), (dw * step).sum(), rtol=1e-6, atol=1e-7)


def test_cross_and_gradients():
    gen = torch.Generator().manual_seed(3)
    randn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, dout = randn(3, 4, 5, 64), randn(3, 2, 7, 64), randn(3, 2, 7, 64), randn(3, 4, 5, 64)
    lens, q_lens, scale = [7, 0, 3], [5, 5, 2], 0.2
    for t in (q, k, v):
        t.requires_grad_()
    seen = (torch.arange(7) < torch.tensor(lens).view(3, 1, 1, 1))
    here = (torch.arange(5).view(5, 1) < torch.tensor(q_lens).view(3, 1, 1, 1))
    logits = scale * (q @ k.repeat_interleave(2, 1).transpose(-1, -2))
    p = torch.softmax(logits.masked_fill(~seen, -1e300), -1) * seen * here
    want = p @ v.repeat_interleave(2, 1)
    out, size, lse = oracle.cross(q.detach(), k.detach(), v.detach(), lens, q_lens, scale)
    torch.testing.assert_close(out, want.detach())
    assert (size + 1e-12 >= out.abs()).all()
    torch.testing.assert_close(lse[2, 1, 1].exp(), logits[2, 1, 1, :3].exp().sum().detach())
    assert (lse[1] == -math.inf).all() and (lse[2, :, 2:] == -math.inf).all()
    grads = oracle.cross_grads(dout, q.detach(), k.detach(), v.detach(), lens, q_lens, scale, 2.0 ** -11)
    for (name, (value, bound)), g in zip(grads.items(), torch.autograd.grad((want * dout).sum(), (q, k, v))):
        torch.testing.assert_close(value, g)
        assert (bound >= 0).all(), name
    with torch.no_grad():
        f = lambda q, k, v: (oracle.cross(q, k, v, lens, q_lens, scale)[0] * dout).sum()  # noqa: E731
        h, args = 1e-6, (q, k, v)
        for i, (value, _) in enumerate(grads.values()):
            step = torch.randn(args[i].shape, dtype=torch.float64)
            up, down = ([t + sign * h * step if j == i else t for j, t in enumerate(args)] for sign in (1, -1))
            torch.testing.assert_close((f(*up) - f(*down)) / (2 * h), (value * step).sum(), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("zeros", [False, True])
def test_int4(zeros):
    gen = torch.Generator().manual_seed(5)
    values = torch.randint(0, 16, (5, 64), generator=gen, dtype=torch.uint8)
    scales, x = torch.rand(5, 2, generator=gen).half(), torch.randn(3, 64, generator=gen).half()
    zero = torch.randint(0, 16, (5, 2), generator=gen, dtype=torch.uint8) if zeros else None
    y, size = oracle.int4(x, values, scales, zero, None, None)
    for m in range(3):
        for n in range(5):
            want = sum(float(x[m, k]) * float(scales[n, k // 32]) * (int(values[n, k]) - (int(zero[n, k // 32]) if zeros else 8))
                       for k in range(64))
            assert abs(want - float(y[m, n])) < 1e-9 and size[m, n] >= abs(want)
