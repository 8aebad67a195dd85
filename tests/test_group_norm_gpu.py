"""conformer.group_norm_act against the definition in float64 (needs an MI355X).

Tolerance, per element: half a step of the output type relative to the value
(torch.finfo(t).eps / 2; fp16's subnormal step 2^-25 absolute), plus fp32
arithmetic.  With d = |x - mean| rstd |w| and the same of |mean|, the fp32 chain
(mean, difference, two products, the activation) makes at most about 12
roundings of 2^-24 of (|x| + |mean|) rstd |w| + |b|; the activations' slope is
at most 1.13, and the hardware exponential of 16-bit outputs adds |v| 2^-23 of a
value at most |v|.  2^-19 of that sum (plus its square's 2^-22 for the
exponential) holds them with a factor of two to spare."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
KINDS = [torch.float32, torch.float16, torch.bfloat16]


def reference(x, batch, groups, w, b, eps, lens, act):
    """-> (y, the scale of the fp32 error), float64."""
    rows, c = x.shape
    t = rows // batch
    y = torch.zeros(rows, c, dtype=torch.float64, device=x.device)
    scale = torch.zeros_like(y)
    for i in range(batch):
        n = t if lens is None else min(max(int(lens[i]), 0), t)
        if n == 0:
            continue
        v = x[i * t:i * t + n].double().view(n, groups, c // groups)
        mean = v.mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt((v - mean).square().mean((0, 2), keepdim=True) + eps)
        u = ((v - mean) * rstd).reshape(n, c) * w.double() + b.double()
        size = ((v.abs() + mean.abs()) * rstd).reshape(n, c) * w.double().abs() + b.double().abs()
        scale[i * t:i * t + n] = size * 2.0 ** -19 + size * size * 2.0 ** -22
        if act == "silu":
            u = u / (1 + torch.exp(-u))
        elif act == "gelu":
            u = 0.5 * u * torch.erfc(-u / math.sqrt(2))
        elif act == "relu":
            u = u.clamp_min(0)
        y[i * t:i * t + n] = u
    return y, scale


def check(got, want, scale, kind):
    tiny = 2.0 ** -25 if kind == torch.float16 else 2.0 ** -120
    err = (got.double() - want).abs()
    tol = want.abs() * (torch.finfo(kind).eps / 2) + scale + tiny
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), float((err - tol).max())


def inputs(rows, c, kind, seed, offset=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, c, generator=gen) * 1.5 + torch.randn(1, c, generator=gen) * offset).to(kind).to(DEV)
    w = (1 + 0.2 * torch.randn(c, generator=gen)).to(DEV)
    b = (0.2 * torch.randn(c, generator=gen)).to(DEV)
    return x, w, b


SHAPES = [
    # (items, frames, channels, groups): one value; one vector; odd sizes; groups of 4 (narrower than a vector);
    # several rows of lanes; a group over everything; one channel per group; more vectors than threads
    (1, 1, 1, 1), (1, 1, 8, 1), (2, 5, 7, 7), (2, 77, 100, 25), (4, 64, 96, 24), (3, 150, 1024, 32), (2, 333, 160, 10),
    (5, 401, 72, 8), (1, 700, 1024, 1), (3, 40, 1024, 1024), (2, 19, 8192, 8192), (2, 50, 4104, 1), (1, 1463, 1024, 16),
    (1, 4800, 512, 16), (2, 2600, 1024, 8), (70, 9, 64, 4),
]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(sidon, shape, kind):
    batch, t, c, groups = shape
    x, w, b = inputs(batch * t, c, kind, 7 * t + c)
    # all lengths, none, one, more than there are, fewer than none
    lens = torch.tensor([(t, max(1, t // 3), 0, 1, t + 9, -3)[i % 6] for i in range(batch)], dtype=torch.int32, device=DEV)
    act = (None, "silu", "gelu", "relu")[(t + c) % 4]
    x.view(batch, t, c)[torch.arange(t, device=DEV).view(1, t) >= lens.view(batch, 1)] = float("nan")
    y = sidon.conformer.group_norm_act(x, batch, groups, w, b, 1e-5, lens=lens, act=act)
    want, scale = reference(x, batch, groups, w, b, 1e-5, lens.tolist(), act)
    check(y, want, scale, kind)


# (items, frames, channels, groups, types): vectors that lie in two groups, and a last column block of fewer groups
# than the others, whose threads have more row lanes than the full blocks' (the statistics' LDS has to hold them)
NARROW_LAST = [(2, 1500, 352, 8, KINDS[1:]), (3, 1700, 416, 8, KINDS[1:]), (8, 4800, 480, 8, KINDS[1:]),
               (1, 1463, 648, 6, KINDS[1:]), (1, 4800, 320, 32, KINDS[1:]), (2, 1500, 176, 8, KINDS[:1]),
               (3, 1001, 208, 8, KINDS[:1]), (1, 1463, 240, 8, KINDS[:1]), (2, 700, 36, 12, KINDS)]


@pytest.mark.parametrize("shape,kind", [(s[:4], k) for s in NARROW_LAST for k in s[4]], ids=str)
def test_narrower_last_block(sidon, shape, kind):
    batch, t, c, groups = shape
    x, w, b = inputs(batch * t, c, kind, t + c)
    lens = [(t, t - t // 3, 1, 17)[i % 4] for i in range(batch)]
    x.view(batch, t, c)[torch.arange(t, device=DEV).view(1, t) >= torch.tensor(lens, device=DEV).view(batch, 1)] = float("nan")
    y = sidon.conformer.group_norm_act(x, batch, groups, w, b, 1e-5, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                       act="silu")
    check(y, *reference(x, batch, groups, w, b, 1e-5, lens, "silu"), kind)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu"])
@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_activations(sidon, act, kind):
    x, w, b = inputs(300, 256, kind, 3)
    for groups in (8, 1):
        y = sidon.conformer.group_norm_act(x, 2, groups, w, b, 1e-3, act=act)
        want, scale = reference(x, 2, groups, w, b, 1e-3, None, act)
        check(y, want, scale, kind)


@pytest.mark.parametrize("shape", [(1, 2000, 64, 2), (2, 300, 64, 1), (1, 6000, 1024, 2)], ids=str)
def test_large_mean(sidon, shape):
    """A mean of 1000 standard deviations: no difference of large sums."""
    batch, t, c, groups = shape
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn(batch * t, c, generator=gen) + 1000).to(DEV)
    w, b = torch.ones(c, device=DEV), torch.zeros(c, device=DEV)
    y = sidon.conformer.group_norm_act(x, batch, groups, w, b, 1e-5, act=None)
    want, scale = reference(x, batch, groups, w, b, 1e-5, None, None)
    check(y, want, scale, torch.float32)


@pytest.mark.parametrize("shape", [(2, 40, 64, 4), (2, 3000, 512, 2), (1, 1463, 100, 25), (3, 1500, 36, 4)], ids=str)
def test_far_from_zero(sidon, shape):
    """Values whose squares leave fp32, whose variance does not."""
    batch, t, c, groups = shape
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(batch * t, c, generator=gen) * 1e16 + 3e20).to(DEV)
    w, b = torch.ones(c, device=DEV), torch.zeros(c, device=DEV)
    lens = [max(1, t - 37 * i) for i in range(batch)]
    y = sidon.conformer.group_norm_act(x, batch, groups, w, b, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                       act=None)
    want, _ = reference(x, batch, groups, w, b, 1e-5, lens, None)
    assert torch.isfinite(y).all()
    # the fp32 chain's share of the module's bound, 2^-19 of (|x| + |mean|) rstd (about 6e4)
    assert ((y.double() - want).abs() <= 2.0 ** -19 * 6.2e4).all()


@pytest.mark.parametrize("c,groups", [(256, 8), (256, 1)])
def test_views(sidon, c, groups):
    """Rows of a wider tensor, unaligned columns, the output beside the input,
    in place; what lies around the output stays."""
    kind = torch.float16
    batch, t = 2, 90
    lens = torch.tensor([90, 31], dtype=torch.int32, device=DEV)
    wide, w, b = inputs(batch * t, 2 * c + 16, kind, 11)
    for lo in (0, 1, 8):
        x = wide[:, lo:lo + c]
        want, scale = reference(x, batch, groups, w[:c].contiguous(), b[:c].contiguous(), 1e-5, lens.tolist(), "silu")
        y = sidon.conformer.group_norm_act(x, batch, groups, w[:c].contiguous(), b[:c].contiguous(), 1e-5, lens=lens)
        check(y, want, scale, kind)
        beside = wide.clone()
        out = beside[:, c + 16:]
        sidon.conformer.group_norm_act(beside[:, lo:lo + c], batch, groups, w[:c].contiguous(), b[:c].contiguous(), 1e-5,
                                       lens=lens, out=out)
        assert torch.equal(out, y) and torch.equal(beside[:, :c + 16], wide[:, :c + 16])
        inplace = wide.clone()
        part = inplace[:, lo:lo + c]
        sidon.conformer.group_norm_act(part, batch, groups, w[:c].contiguous(), b[:c].contiguous(), 1e-5, lens=lens,
                                       out=part)
        assert torch.equal(part, y) and torch.equal(inplace[:, lo + c:], wide[:, lo + c:])


@pytest.mark.parametrize("groups", [32, 1])
def test_streams_and_graphs(sidon, groups):
    """Another stream than the tensors' own, one workspace for consecutive calls,
    and a graph replayed on new inputs with eager work in between."""
    x, w, b = inputs(900, 512, torch.bfloat16, 5)
    lens = torch.tensor([300, 17, 300], dtype=torch.int32, device=DEV)
    call = lambda **kw: sidon.conformer.group_norm_act(x, 3, groups, w, b, 1e-5, lens=lens, **kw)  # noqa: E731
    ws = torch.empty(sidon.conformer.group_norm_workspace(3, 300, 512, groups, x.dtype), dtype=torch.uint8, device=DEV)
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(workspace=ws)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=out, workspace=ws)
    for seed in range(3):
        x.copy_(inputs(900, 512, torch.bfloat16, 50 + seed)[0])
        lens.copy_(torch.tensor([299 - seed, 0, 12 * seed], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_gradients_are_refused(sidon):
    x, w, b = inputs(8, 16, torch.float32, 1)
    with pytest.raises(ValueError, match="no_grad"):
        sidon.conformer.group_norm_act(x, 1, 2, torch.nn.Parameter(w), b)
    with torch.no_grad():
        sidon.conformer.group_norm_act(x, 1, 2, torch.nn.Parameter(w), b)
