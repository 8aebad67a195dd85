"""qk_norm_rotary and its gradients against the definition in float64 (needs an
MI355X).

Tolerances.  The kernel works in fp32 and rounds once: a sum of D squares over a
team of lanes goes through at most 8 + 5 additions, rsqrt is off by 2 steps, and a
value goes through some five more products and sums, so y is off by less than 32 half
steps of fp32 (2^-24 each) of its pair's magnitude, and by u = finfo(t).eps / 2 of itself.  The
same for dx, whose mean of products goes through 13 additions more.  A term of dw goes
through the additions of its team's rows (at most 64 here), the teams of a workgroup
(at most 128), the workgroups' (32 and 32): under 512 in all with what formed it."""

from __future__ import annotations

import pytest
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
EPS = 1e-6
KINDS = [torch.float16, torch.bfloat16, torch.float32]


def inputs(b, l, h, hk, d, rot, kind, seed, places=500):
    """Heads of a fused projection's rows q | k | v, tables, places with padding among them."""
    gen = torch.Generator().manual_seed(seed)
    rows = (1.5 * torch.randn(b, l, h + 2 * hk, d, generator=gen)).to(kind).to(DEV).permute(0, 2, 1, 3)
    w = [(1 + 0.3 * torch.randn(d, generator=gen)).to(DEV) for _ in range(2)]
    cos = sin = None
    if rot:
        angle = torch.rand(places, rot // 2, generator=gen) * 7
        cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    pos = torch.randint(-60 if b * l > 1 else 0, places, (b, l), generator=gen, dtype=torch.int32).to(DEV)
    return rows[:, :h], rows[:, h:h + hk], w[0], w[1], cos, sin, pos


def close(got, want, size, steps=32):
    assert torch.isfinite(got).all()
    u = torch.finfo(got.dtype).eps / 2
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -140}[got.dtype]
    err = (got.double() - want).abs()
    tol = u * want.abs() + steps * 2.0 ** -24 * size + tiny
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


def grad_like(t, seed):
    return torch.randn(t.shape, generator=torch.Generator().manual_seed(seed)).to(t.dtype).to(DEV)


CASES = [
    # (batch, tokens, heads, key heads, D, rotated): a token, odd counts, every team size, no rotation and part of it
    (1, 1, 1, 1, 16, 16), (1, 1, 16, 16, 64, 64), (3, 1, 4, 1, 128, 64), (2, 7, 5, 3, 32, 16), (1, 33, 6, 2, 48, 32),
    (2, 19, 3, 1, 80, 80), (5, 13, 8, 8, 64, 0), (1, 257, 12, 4, 96, 48), (2, 31, 2, 2, 256, 256), (1, 5, 40, 1, 240, 16),
    (2, 700, 16, 4, 64, 64), (3, 301, 17, 5, 128, 128), (1, 1500, 9, 3, 112, 64),
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_float64(sidon, case, kind, interleaved):
    b, l, h, hk, d, rot = case
    q, k, qw, kw, cos, sin, pos = inputs(*case, kind, 17 * l + d)
    padded = (pos < 0).view(b, 1, l, 1)
    dq_out, dk_out = grad_like(q, 1), grad_like(k, 2)
    for t in (q, k, dq_out, dk_out):   # what padding holds is anything
        t.masked_fill_(padded, float("nan"))
    hn = sidon.head_norm
    got = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos, EPS, interleaved)
    grads = hn.qk_norm_rotary_backward(dq_out, dk_out, q, k, qw, kw, cos, sin, pos, pos, EPS, interleaved)
    for x, w, y, dy, dx, dw in ((q, qw, got[0], dq_out, grads[0], grads[2]), (k, kw, got[1], dk_out, grads[1], grads[3])):
        want, size = oracle.norm_rotary(x, w, cos, sin, pos, EPS, interleaved)
        close(y, want, size)
        assert (y.masked_select(padded.expand_as(y)) == 0).all()
        want, size, wsum, wsize = oracle.norm_rotary_grads(dy, x, w, cos, sin, pos, EPS, interleaved)
        close(dx, want, size, 64)
        close(dw, wsum, wsize, 512)


def test_gradient_is_the_difference(sidon):
    """Along a random direction, against differences of the float64 definition."""
    q, k, qw, kw, cos, sin, pos = inputs(2, 9, 4, 2, 64, 64, torch.float32, 3)
    dy = grad_like(q, 4)
    dx, _, dw, _ = sidon.head_norm.qk_norm_rotary_backward(dy, None, q, None, qw, None, cos, sin, pos, None, EPS, True)
    f = lambda x, w: float((oracle.norm_rotary(x, w, cos, sin, pos, EPS, True)[0] * dy.double()).sum())  # noqa: E731
    step, wstep, h = grad_like(q, 5).double(), grad_like(qw, 6).double(), 1e-5
    x, w = q.double(), qw.double()
    want = (f(x + h * step, w) - f(x - h * step, w)) / (2 * h)
    # 2^-24 of 64 half steps a value, over sums of random sign
    assert abs(want - float((dx.double() * step).sum())) <= 1e-4 * float((dx.double() * step).abs().sum())
    want = (f(x, w + h * wstep) - f(x, w - h * wstep)) / (2 * h)
    assert abs(want - float((dw.double() * wstep).sum())) <= 1e-4 * float((dw.double() * wstep).abs().sum())


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_places_of_their_own(sidon, kind):
    """No places: 0, 1, ...; one past the tables: NaN where it is rotated, in that token alone."""
    q, k, qw, kw, cos, sin, _ = inputs(2, 12, 4, 2, 64, 32, kind, 8, places=20)
    hn = sidon.head_norm
    rows = torch.arange(12, dtype=torch.int32, device=DEV).expand(2, 12).contiguous()
    want = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, rows, rows)
    assert all(torch.equal(a, b) for a, b in zip(hn.qk_norm_rotary(q, k, qw, kw, cos, sin), want))
    past = rows.clone()
    past[0, 3], past[1, 0] = 20, 2 ** 31 - 1
    got = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, past, rows)[0]
    for b, l in ((0, 3), (1, 0)):
        assert got[b, :, l, :32].isnan().all() and torch.equal(got[b, :, l, 32:], want[0][b, :, l, 32:])
        got[b, :, l] = want[0][b, :, l]
    assert torch.equal(got, want[0])


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_in_place_and_strides(sidon, kind, interleaved):
    """In place on the rows of a fused projection, whose values stay; heads first; an
    output within a wider tensor; expanded gradients."""
    b, l, h, hk, d = 2, 37, 4, 2, 64
    q, k, qw, kw, cos, sin, pos = inputs(b, l, h, hk, d, d, kind, 11)
    hn = sidon.head_norm
    call = lambda q, k, **kw2: hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos, EPS, interleaved, **kw2)  # noqa: E731
    want = call(q, k)
    assert all(torch.equal(a, b) for a, b in zip(call(q.contiguous(), k.contiguous()), want))
    wide = torch.full((b, l, h * d + 64), 7.0, dtype=kind, device=DEV)
    out = wide[..., 32:-32].unflatten(-1, (h, d)).permute(0, 2, 1, 3)
    assert call(q, k, out_q=out)[0] is out
    assert torch.equal(out, want[0]) and (wide[..., :32] == 7).all() and (wide[..., -32:] == 7).all()
    one = grad_like(q[:, :1, :1], 5).expand(b, h, l, d)
    args = (qw, kw, cos, sin, pos, pos, EPS, interleaved)
    grads = hn.qk_norm_rotary_backward(one, want[1], q, k, *args)
    again = hn.qk_norm_rotary_backward(one.contiguous(), want[1], q, k, *args)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    over = one.contiguous()
    got = hn.qk_norm_rotary_backward(over, want[1], q, k, *args, dq=over)
    assert got[0] is over and torch.equal(over, grads[0])
    rows = q._base
    before = rows.clone()
    got = call(q, k, out_q=q, out_k=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(rows.view(-1, h + 2 * hk, d)[:, h + hk:], before.view(-1, h + 2 * hk, d)[:, h + hk:])


def test_queries_alone(sidon):
    q, k, qw, kw, cos, sin, pos = inputs(2, 9, 4, 2, 64, 64, torch.bfloat16, 13)
    both = sidon.head_norm.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos)
    alone = sidon.head_norm.qk_norm_rotary(k, None, kw, None, cos, sin, pos)
    assert alone[1] is None and torch.equal(alone[0], both[1])
    both = sidon.head_norm.qk_norm_rotary_backward(q, k, q, k, qw, kw, cos, sin, pos, pos)
    alone = sidon.head_norm.qk_norm_rotary_backward(k, None, k, None, kw, None, cos, sin, pos)
    assert alone[1] is None and alone[3] is None and torch.equal(alone[0], both[1]) and torch.equal(alone[2], both[3])


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32], ids=str)
def test_values_past_the_squares_range(sidon, kind):
    """Squares past 2^128 and below 2^-126, a row of zeros, and an infinity, which
    gives NaN in its own row alone."""
    q, k, qw, kw, cos, sin, _ = inputs(1, 6, 2, 1, 64, 64, kind, 19)
    q = q.contiguous()
    plain = q.clone()
    q[:, :, 1] = (q[:, :, 1].float() * 2.0 ** 100).to(kind)
    q[:, :, 2] = (q[:, :, 2].float() * 2.0 ** 124).to(kind)
    q[:, :, 3] = 0
    q[:, :, 4] = (q[:, :, 4].float() * 2.0 ** -80).to(kind)
    dy = grad_like(q, 7)
    want, size = oracle.norm_rotary(q, qw, cos, sin, None, EPS, False)
    got = sidon.head_norm.qk_norm_rotary(q, None, qw, None, cos, sin)[0]
    close(got, want, size)
    want, size, wsum, wsize = oracle.norm_rotary_grads(dy, q, qw, cos, sin, None, EPS, False)
    dx, _, dw, _ = sidon.head_norm.qk_norm_rotary_backward(dy, None, q, None, qw, None, cos, sin)
    close(dx, want, size, 64)
    close(dw, wsum, wsize, 512)
    q[0, 1, 5, 9] = float("inf")
    bad = sidon.head_norm.qk_norm_rotary(q, None, qw, None, cos, sin)[0]
    assert bad[0, 1, 5].isnan().any()
    bad[0, 1, 5] = got[0, 1, 5]
    assert torch.equal(bad, got)
    assert torch.equal(sidon.head_norm.qk_norm_rotary(plain, None, qw, None, cos, sin)[0][:, :, :1], got[:, :, :1])


def test_captured(sidon):
    """Both directions in one graph, replayed on new contents between eager calls."""
    q, k, qw, kw, cos, sin, pos = inputs(2, 50, 8, 2, 64, 64, torch.bfloat16, 23)
    q, k = q.contiguous(), k.contiguous()
    hn = sidon.head_norm

    def step():
        y = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos)
        return *y, *hn.qk_norm_rotary_backward(y[0], y[1], q, k, qw, kw, cos, sin, pos, pos)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        q.copy_(grad_like(q, 30 + i))
        pos.fill_(i)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
