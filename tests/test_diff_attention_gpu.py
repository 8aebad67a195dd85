"""diff_attention against the definition in float64 (needs an MI355X).

Tolerance, per element, before the norm.  With u the half step of the input type
(torch.finfo(t).eps / 2) and W_m = softmax_m |v| the values' weighted magnitude of
map m: probabilities are rounded once (each off by u of itself, so the sum by at
most u W_m), the fp32 scores of D products by 2^-24 sqrt(D) of |q| . |k| / sqrt D,
which moves a probability by twice that (numerator and sum); exp2 and the sums add
some 2^-22.  With the test's N(0, 1) scores sums |q| . |k| / sqrt D stay under 16
sqrt D, so the scores' share is below 2^-24 sqrt D 32 sqrt D = 2^-12 at D = 128
(2^-13 at 64) at worst; taken as 2^-12.  So o is off by at most
(u + 2^-12) (W_1 + lambda W_2) + tiny.  The norm divides by r = rms(o): the
error is that over r, plus |out| times the mean error's share of r (Cauchy: rms
of the error over r).  The output's own rounding adds u |out|."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def reference(q, k, v, lam, lam_init, lens, causal, norm_w, eps):
    """-> (out, tolerance) in float64."""
    b, h, _, l, d = q.shape
    hk, s = k.shape[1], k.shape[3]
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(b, h, l, 2 * d, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for i in range(b):
        n = s if lens is None else min(max(int(lens[i]), 0), s)
        limit = torch.full((l,), n, device=q.device)
        if causal:
            limit = (torch.arange(l, device=q.device) + n - l + 1).clamp(0, n)
        hidden = torch.arange(n, device=q.device) >= limit.view(l, 1)
        for j in range(h):
            lm = (lam if lam.dim() == 2 else lam[j]).double()
            weight = math.exp(float(lm[0] @ lm[1])) - math.exp(float(lm[2] @ lm[3])) + lam_init
            vals = v[i, j // (h // hk), :n].double()
            o = torch.zeros(l, 2 * d, dtype=torch.float64, device=q.device)
            err = torch.zeros_like(o)
            for m, f in ((0, 1.0), (1, -weight)):
                logits = q[i, j, m].double() @ k[i, j // (h // hk), m, :n].double().t() / math.sqrt(d)
                p = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
                o += f * (p @ vals)
                err += abs(f) * (p @ vals.abs()) * (u + 2.0 ** -12)
            if norm_w is not None:
                r = torch.sqrt(o.square().mean(-1, keepdim=True) + eps)
                gain = (norm_w.double() * (1 - lam_init)) / r
                spread = torch.sqrt(err.square().mean(-1, keepdim=True)) / r
                o = o * gain
                err = err * gain.abs() + o.abs() * spread
            out[i, j] = o
            tol[i, j] = err + o.abs() * u
    return out, tol + (2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -100)


def inputs(b, h, hk, l, s, d, kind, seed, per_head=False):
    """Views of fused projections: [B*L, H*2*D] rows and a cache [B, S, Hk, 4*D]."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(b, l, h, 2, d, generator=gen).to(kind).to(DEV).permute(0, 2, 3, 1, 4)
    kv = torch.randn(b, s, hk, 4 * d, generator=gen).to(kind).to(DEV)
    k = kv[..., :2 * d].unflatten(-1, (2, d)).permute(0, 2, 3, 1, 4)
    v = kv[..., 2 * d:].permute(0, 2, 1, 3)
    lam = (0.1 * torch.randn(*((h, 4, d) if per_head else (4, d)), generator=gen)).to(DEV)
    norm_w = (1 + 0.1 * torch.randn(2 * d, generator=gen)).to(DEV)
    return q, k, v, lam, norm_w


def check(got, want, tol):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


def poison(k, v, lens):
    """What lies past the valid keys is anything."""
    for i, n in enumerate(lens):
        n = max(n, 0)
        k[i, :, :, n:] = float("nan")
        v[i, :, n:] = float("inf")


SHAPES = [
    # (batch, heads, key heads, queries, keys, D): one of each; single tokens against short, odd and long caches,
    # with and without groups; a few tokens; prompts around the 32- and 128-row blocks; groups whose rows straddle heads
    (1, 1, 1, 1, 1, 64), (2, 2, 1, 1, 31, 64), (3, 8, 2, 1, 33, 64), (1, 8, 8, 1, 4800, 64), (5, 4, 4, 1, 1000, 128),
    (2, 8, 1, 1, 2049, 128), (2, 40, 1, 1, 77, 64), (2, 4, 2, 5, 300, 64), (2, 6, 2, 13, 515, 128), (1, 2, 2, 32, 32, 64),
    (1, 1, 1, 33, 65, 128), (3, 4, 2, 150, 150, 64), (1, 2, 1, 127, 400, 64), (9, 8, 8, 517, 517, 64),
    (9, 8, 4, 300, 333, 128), (40, 8, 8, 129, 129, 64), (70, 4, 4, 128, 64, 128), (32, 8, 8, 3, 129, 64),
]


@pytest.mark.parametrize("causal", [False, True], ids=["both", "causal"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(sidon, shape, kind, causal):
    b, h, hk, l, s, d = shape
    seed = 31 * l + s + d
    q, k, v, lam, norm_w = inputs(b, h, hk, l, s, d, kind, seed, per_head=seed % 2 == 0)
    some = (s, max(1, s // 2), 0, 1, s + 5, -2, min(s, 32), min(s, 33))
    lens = [some[i % len(some)] for i in range(b)]
    if b == 1 and l > 1:
        lens = [s - s // 3]
    poison(k, v, lens)
    if seed % 3 == 0:
        norm_w = None
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                              causal=causal, norm_w=norm_w)
    check(got, *reference(q, k, v, lam, 0.3, lens, causal, norm_w, 1e-5))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 2, 200, 300, 64), (6, 8, 8, 700, 700, 64), (6, 8, 8, 700, 700, 128),
                                   (2, 4, 1, 1, 900, 128)], ids=str)
def test_rising_scores(sidon, shape, kind):
    """Scores that grow along the keys by far more than the fp16 range of the
    probabilities, so that running maxima are raised again and again."""
    b, h, hk, l, s, d = shape
    q, k, v, lam, norm_w = inputs(b, h, hk, l, s, d, kind, 5)
    q = (q.abs() * 0.25).contiguous()
    ramp = torch.linspace(-3, 3, s, device=DEV).view(1, 1, 1, s, 1)
    k = (k.float() * 0.1 + ramp).to(kind)
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, norm_w=None)
    check(got, *reference(q, k, v, lam, 0.3, None, False, None, 1e-5))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 2, 1, 20000, 64), (1, 2, 1, 3, 3000, 128), (6, 8, 8, 700, 1900, 64),
                                   (6, 8, 8, 300, 1900, 128)], ids=str)
def test_small_probabilities(sidon, shape, kind):
    """A key with no value in every 128 that takes nearly all of the weight, and an
    output that comes from the others: e^-15 of it each (under fp16's smallest
    normal number), and each still rounded by half a step of itself."""
    b, h, hk, l, s, d = shape
    q, k, v, lam, _ = inputs(*shape, kind, 7)
    q = torch.zeros_like(q)
    q[..., 0] = 8.0   # (scores: k at D = 64, k / sqrt 2 at 128)
    k = torch.zeros_like(k)
    k[..., 0] = -15.125 if d == 64 else -21.375
    k[:, :, :, ::128] = 0
    v = v.abs().clone()
    v[:, :, ::128] = 0
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3)
    check(got, *reference(q, k, v, lam, 0.3, None, False, None, 1e-5))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(64, 1, 1, 1, 8, 64), (16, 8, 2, 5, 7, 128), (16, 2, 2, 32, 8, 64), (20, 3, 1, 9, 33, 64)],
                         ids=str)
def test_few_rows_keep_two_summands(sidon, shape, kind):
    """Up to 32 rows of a key head: two maps that nearly cancel, so that what the
    probabilities lose is far more than the output's rounding.  Two summands of a
    type keep u^2 of each.  Scores of products below 1 (D of them, over sqrt D, to
    2^-24 each) and exp2 move a probability by less than 2^-15 of itself.  (One
    summand would be 7 times over this bound in fp16, 30 times in bf16.)"""
    b, h, hk, l, s, d = shape
    q, k, v, lam, _ = inputs(*shape, kind, 21)
    q, k = (0.5 * q.float()).to(kind), (0.5 * k.float()).to(kind)
    gen = torch.Generator().manual_seed(22)
    q[:, :, 1], k[:, :, 1] = q[:, :, 0], k[:, :, 0] + (0.01 * torch.randn(b, hk, s, d, generator=gen)).to(kind).to(DEV)
    lam = torch.zeros_like(lam)
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 1.0).double()
    u = torch.finfo(kind).eps / 2
    maps = torch.softmax(torch.matmul(q.double(), k.double().repeat_interleave(h // hk, 1).transpose(-1, -2).contiguous())
                         / math.sqrt(d), -1)
    vals = v.double().repeat_interleave(h // hk, 1)
    want = torch.matmul(maps[:, :, 0] - maps[:, :, 1], vals)
    size = torch.matmul(maps[:, :, 0] + maps[:, :, 1], vals.abs())
    tiny = 2.0 ** -24 if kind == torch.float16 else 2.0 ** -100
    assert ((got - want).abs() <= (u * u + 2.0 ** -15) * size + u * want.abs() + tiny).all()


@pytest.mark.parametrize("l", [1, 300])
def test_strides_and_out(sidon, l):
    """[B, H, 2, L, D] contiguous, key rows and heads in other orders, an output
    inside a wider tensor, shared keys by a zero stride; what lies around the
    output stays."""
    b, h, hk, s, d, kind = 2, 4, 2, 333, 64, torch.float16
    q, k, v, lam, norm_w = inputs(b, h, hk, l, s, d, kind, 9)
    lens = torch.tensor([333, 100], dtype=torch.int32, device=DEV)
    call = lambda q, k, v, **kw: sidon.diff_attention.diff_attention(  # noqa: E731
        q, k, v, lam, 0.3, lens=lens, causal=True, norm_w=norm_w, **kw)
    want = call(q, k, v)
    check(want, *reference(q, k, v, lam, 0.3, lens.tolist(), True, norm_w, 1e-5))
    assert torch.equal(call(q.contiguous(), k.contiguous(), v.contiguous()), want)
    maps_first = k.permute(2, 1, 0, 3, 4).contiguous().permute(2, 1, 0, 3, 4)
    keys_first = v.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    assert torch.equal(call(q, maps_first, keys_first), want)
    wide = torch.full((b, l, h * 2 * d + 64), 7.0, dtype=kind, device=DEV)
    out = wide[..., 32:-32].unflatten(-1, (h, 2 * d)).permute(0, 2, 1, 3)
    assert call(q, k, v, out=out) is out
    assert torch.equal(out, want) and (wide[..., :32] == 7).all() and (wide[..., -32:] == 7).all()
    one = k[:, :1].expand(b, hk, 2, s, d)
    assert torch.equal(call(q, one, v), call(q, one.contiguous(), v))


def test_a_row_does_not_depend_on_the_others(sidon):
    """The same queries alone and among others, and other items' lengths: equal
    to the last bit where the keys are split alike."""
    q, k, v, lam, norm_w = inputs(4, 8, 8, 600, 600, 64, torch.float16, 3)
    lens = torch.tensor([600, 600, 600, 600], dtype=torch.int32, device=DEV)
    a = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, lens=lens, norm_w=norm_w)
    lens[1:] = torch.tensor([0, 17, 300], dtype=torch.int32)
    q2 = q.clone()
    q2[1:] *= 20
    c = sidon.diff_attention.diff_attention(q2, k, v, lam, 0.3, lens=lens, norm_w=norm_w)
    assert torch.equal(a[0], c[0]) and (c[1] == 0).all()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 2, 32, 200, 64), (2, 8, 2, 5, 900, 128), (9, 8, 8, 517, 517, 64),
                                   (9, 8, 4, 300, 333, 128), (1, 8, 8, 30, 4800, 64)], ids=str)
def test_queries_that_are_no_numbers(sidon, shape, kind):
    """NaN and infinities in some queries (the padding of a batch, say) come back
    as NaN and reach no other query, head or item."""
    b, h, hk, l, s, d = shape
    q, k, v, lam, norm_w = inputs(*shape, kind, 12)
    want, tol = reference(q, k, v, lam, 0.3, None, False, norm_w, 1e-5)
    bad = torch.zeros(b, h, l, dtype=torch.bool, device=DEV)
    bad[:, :, 1::5] = True
    bad[:, 0, 0] = True
    q = q.clone()
    q[:, :, 0][bad] = float("nan")
    q[:, :, 1, 1::10] = float("inf")
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, norm_w=norm_w)
    check(got[~bad], want[~bad], tol[~bad])
    assert torch.isnan(got[bad]).all()


def test_repeats_are_equal(sidon):
    for shape in ((1, 8, 8, 1, 4800, 64), (2, 8, 8, 1037, 1037, 64), (6, 8, 8, 700, 700, 128)):
        q, k, v, lam, norm_w = inputs(*shape, torch.bfloat16, 2)
        first = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, norm_w=norm_w)
        for _ in range(20):
            assert torch.equal(sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, norm_w=norm_w), first)


@pytest.mark.parametrize("l", [1, 200])
def test_streams_and_graphs(sidon, l):
    q, k, v, lam, norm_w = inputs(2, 8, 4, l, 700, 64, torch.bfloat16, 4)
    lens = torch.tensor([700, 211], dtype=torch.int32, device=DEV)
    need = sidon.diff_attention.workspace_bytes(2, 8, 4, l, 700, 64, DEV)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    call = lambda **kw: sidon.diff_attention.diff_attention(  # noqa: E731
        q, k, v, lam, 0.3, lens=lens, causal=True, norm_w=norm_w, **kw)
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(workspace=ws)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=out, workspace=ws)
    for i in range(3):
        q.copy_(inputs(2, 8, 4, l, 700, 64, torch.bfloat16, 40 + i)[0])
        lens.copy_(torch.tensor([700 - 40 * i, 300 * i], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_gradients_are_refused(sidon):
    q, k, v, lam, norm_w = inputs(1, 1, 1, 2, 2, 64, torch.float16, 1)
    with pytest.raises(ValueError, match="no_grad"):
        sidon.diff_attention.diff_attention(q, k, v, torch.nn.Parameter(lam), 0.3)
