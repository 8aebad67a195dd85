"""cross_attention and its gradients against the definition in float64 (needs an
MI355X).

Forward tolerance, per element, as differential attention's: with u the half step of
the type and W = softmax |v|, probabilities are rounded once (u W), the fp32 scores
of N(0, 1) operands move one by less than 2^-12 of itself: (u + 2^-12) W, and the output's own
rounding, u |out|.  Up to 32 rows of a key head keep two summands, u^2 W for u W.  lse:
2^-12 for the scores, and fp32 sums and logarithms of some 2^-20 of max(1, |lse|).

Gradients: decoder_oracle.cross_grads derives their bounds.  They add roundings of
every term at its worst; beside them the error as a whole (root of the sum of
squares) is held to 2 u of the gradient: dS's and the output's roundings, each
uniform within u, are u / sqrt 3 apiece where the terms' signs are random, which makes
0.82 u, and delta's, P's and the scores' stay below that again."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
KINDS = [torch.float16, torch.bfloat16]


def inputs(b, h, hk, l, s, d, kind, seed):
    """Views of fused projections: [B*L, H*D] rows, and frames' rows k | v."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(b, l, h, d, generator=gen).to(kind).to(DEV).permute(0, 2, 1, 3)
    kv = torch.randn(b, s, 2, hk, d, generator=gen).to(kind).to(DEV).permute(2, 0, 3, 1, 4)
    dout = torch.randn(b, l, h, d, generator=gen).to(kind).to(DEV).permute(0, 2, 1, 3)
    return q, kv[0], kv[1], dout


def int32(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device=DEV)


def tiny(kind):
    return 2.0 ** -24 if kind == torch.float16 else 2.0 ** -100


def within(got, want, tol):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


def check_forward(got, lse, q, k, v, lens, q_lens, scale):
    want, size, want_lse = oracle.cross(q, k, v, lens, q_lens, scale)
    u = torch.finfo(q.dtype).eps / 2
    p = u * u if q.shape[1] // k.shape[1] * q.shape[2] <= 32 else u
    within(got, want, (p + 2.0 ** -12) * size + u * want.abs() + tiny(q.dtype))
    if lse is not None:
        none = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        assert ((lse.double() - want_lse).abs() <= 2.0 ** -12 + 2.0 ** -20 * want_lse.abs())[~none].all()


def check_backward(grads, dout, q, k, v, lens, q_lens, scale, whole=True):
    u = torch.finfo(q.dtype).eps / 2
    want = oracle.cross_grads(dout, q, k, v, lens, q_lens, scale, u)
    for got, (name, (value, tol)) in zip(grads, want.items()):
        assert got.dtype == q.dtype and got.shape == value.shape, name
        within(got, value, tol + tiny(q.dtype))
        if whole:
            assert (got.double() - value).norm() <= 2 * u * value.norm() + tiny(q.dtype), name


def poison(lens, q_lens, q, k, v, dout):
    """What lies past the valid keys and queries is anything."""
    for i in range(q.shape[0]):
        if lens is not None:
            k[i, :, max(lens[i], 0):], v[i, :, max(lens[i], 0):] = float("nan"), float("inf")
        if q_lens is not None:
            q[i, :, max(q_lens[i], 0):], dout[i, :, max(q_lens[i], 0):] = float("nan"), float("-inf")


SHAPES = [
    # (batch, heads, key heads, queries, keys, D): one of each; single tokens against short, odd and long keys;
    # a few tokens; prompts around the 32-, 64- and 128-row blocks; groups whose rows straddle heads
    (1, 1, 1, 1, 1, 64), (2, 2, 1, 1, 31, 64), (3, 8, 2, 1, 33, 64), (1, 8, 8, 1, 4800, 64), (5, 4, 4, 1, 1000, 128),
    (2, 8, 1, 1, 2049, 128), (2, 40, 1, 1, 77, 64), (2, 4, 2, 5, 300, 64), (2, 6, 2, 13, 515, 128), (1, 2, 2, 32, 32, 64),
    (1, 1, 1, 33, 65, 128), (3, 4, 2, 150, 150, 64), (1, 2, 1, 127, 400, 64), (9, 8, 8, 517, 129, 64),
    (9, 8, 4, 300, 333, 128), (40, 8, 8, 129, 129, 64), (70, 4, 4, 128, 64, 128), (32, 8, 8, 3, 129, 64),
    (2, 3, 3, 65, 96, 64), (2, 6, 1, 64, 31, 128), (1, 16, 16, 200, 1463, 64),
]


def lengths(b, l, s, seed):
    some = (s, max(1, s // 2), 0, 1, s + 5, -2, min(s, 32), min(s, 33))
    few = (l, l, max(1, l - 1), l + 9, 0, min(l, 33), -1, (l + 1) // 2)
    lens = [some[(i + seed) % len(some) if i else 0] for i in range(b)]
    q_lens = [few[i % len(few)] for i in range(b)]
    return [s - s // 3] if b == 1 and l > 1 else lens, q_lens


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(sidon, shape, kind):
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, kind, 31 * l + s + d)
    lens, q_lens = lengths(b, l, s, l)
    if (l + s) % 3 == 0:
        q_lens = None
    poison(lens, q_lens, q, k, v, dout)
    lse = torch.full((b, h, l), 5.0, device=DEV)
    got = sidon.cross_attention.cross_attention(q, k, v, int32(lens), int32(q_lens), lse=lse)
    check_forward(got, lse, q, k, v, lens, q_lens, d ** -0.5)
    assert torch.equal(got, sidon.cross_attention.cross_attention(q, k, v, int32(lens), int32(q_lens)))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", [(1, 4, 4, 4136, 1330, 128), (2, 4, 4, 2060, 1300, 64), (1, 8, 8, 4110, 1409, 64),
                                   (2, 8, 2, 1037, 2600, 128), (1, 4, 4, 4136, 2650, 128), (2, 4, 4, 2060, 3300, 64),
                                   (1, 8, 8, 4110, 3299, 64), (2, 8, 2, 1037, 4800, 128)], ids=str)
def test_row_blocks_left_over(sidon, shape, kind):
    """A few row blocks more than 256 CUs take at once, whose keys are split, where there are many, while the others' are not."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, kind, 31 * l + s + d)
    lens, q_lens = ([s - 3], [l - 5]) if b == 1 else ([s, s - 70], [l - 11, l])
    poison(lens, q_lens, q, k, v, dout)
    ca = sidon.cross_attention
    if s > 2600 and torch.cuda.get_device_properties(DEV).multi_processor_count == 256:
        # parts of fewer rows than there are (16 + 4 D bytes each)
        assert 0 < ca.workspace_bytes(b, h, hk, l, s, d, DEV) < b * h * l * (16 + 4 * d)
    lse = torch.full((b, h, l), 5.0, device=DEV)
    got = ca.cross_attention(q, k, v, int32(lens), int32(q_lens), lse=lse)
    check_forward(got, lse, q, k, v, lens, q_lens, d ** -0.5)
    assert torch.equal(got, ca.cross_attention(q, k, v, int32(lens), int32(q_lens)))
    lse.zero_()
    got = ca.cross_attention(q, k, v, int32([0] * b), int32(q_lens), lse=lse)
    assert (got == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 2, 200, 300, 64), (6, 8, 8, 700, 700, 64), (6, 8, 8, 700, 700, 128),
                                   (2, 4, 1, 1, 900, 128)], ids=str)
def test_rising_scores(sidon, shape, kind):
    """Scores that grow along the keys by far more than the fp16 range of the
    probabilities, so that running maxima are raised again and again; a scale."""
    b, h, hk, l, s, d = shape
    q, k, v, _ = inputs(*shape, kind, 5)
    q = (q.abs() * 0.25).contiguous()
    k = (k.float() * 0.1 + torch.linspace(-3, 3, s, device=DEV).view(1, 1, s, 1)).to(kind)
    lse = torch.empty(b, h, l, device=DEV)
    got = sidon.cross_attention.cross_attention(q, k, v, scale=0.2, lse=lse)
    check_forward(got, lse, q, k, v, None, None, 0.2)


BACKWARD = [
    (1, 1, 1, 1, 1, 64), (2, 2, 1, 1, 31, 64), (3, 4, 2, 5, 33, 128), (2, 4, 2, 32, 65, 64), (1, 2, 2, 33, 128, 128),
    (3, 6, 2, 31, 129, 64), (2, 4, 4, 150, 300, 64), (2, 8, 2, 127, 97, 128), (9, 2, 1, 64, 64, 64), (1, 3, 1, 260, 515, 64),
    (2, 16, 16, 100, 400, 64), (1, 4, 1, 300, 200, 128), (40, 2, 2, 3, 300, 64),
]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", BACKWARD, ids=str)
def test_backward(sidon, shape, kind):
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, kind, 7 * l + s + d)
    lens, q_lens = lengths(b, l, s, s)
    poison(lens, q_lens, q, k, v, dout)
    lens32, q_lens32 = int32(lens), int32(q_lens)
    lse = torch.empty(b, h, l, device=DEV)
    ca = sidon.cross_attention
    out = ca.cross_attention(q, k, v, lens32, q_lens32, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, lens32, q_lens32)
    check_backward(grads, dout, q, k, v, lens, q_lens, d ** -0.5, whole=min(l, s) >= 31 and b < 3)
    for i in range(b):
        n, m = min(max(lens[i], 0), s), min(max(q_lens[i], 0), l)
        assert (grads[0][i, :, m:] == 0).all() and (grads[1][i, :, n:] == 0).all() and (grads[2][i, :, n:] == 0).all()
    again = ca.cross_attention_backward(dout, q, k, v, out, lse, lens32, q_lens32)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


# (batch, heads, key heads, queries, keys, D): one for each form of the gradients' launch, on 256 CUs (blocks of keys, of
# queries, and whose come first)
FORMS = [
    (20, 8, 8, 42, 44, 64), (19, 8, 8, 49, 129, 64), (10, 4, 4, 41, 72, 64), (2, 1, 1, 42, 820, 64), (17, 16, 8, 41, 36, 64),
    (11, 8, 8, 112, 101, 64), (2, 1, 1, 39, 36, 64), (2, 1, 1, 48, 312, 64), (2, 3, 1, 594, 38, 64), (13, 8, 8, 68, 37, 64),
    (2, 2, 1, 37, 36, 64), (2, 2, 1, 107, 296, 64), (34, 2, 2, 40, 74, 128), (27, 2, 2, 34, 207, 128),
    (38, 8, 4, 37, 35, 128), (2, 1, 1, 37, 34, 128), (2, 1, 1, 35, 79, 128),
]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", FORMS, ids=str)
def test_backward_forms(sidon, shape, kind):
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, kind, l + s + b)
    lens, q_lens = lengths(b, l, s, 0)
    poison(lens, q_lens, q, k, v, dout)
    lens32, q_lens32 = int32(lens), int32(q_lens)
    lse, ca = torch.empty(b, h, l, device=DEV), sidon.cross_attention
    out = ca.cross_attention(q, k, v, lens32, q_lens32, lse=lse)
    outs = [torch.full_like(t, 7.0) for t in (q, k, v)]
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, lens32, q_lens32, dq=outs[0], dk=outs[1], dv=outs[2])
    assert all(x is y for x, y in zip(grads, outs))
    check_backward(grads, dout, q, k, v, lens, q_lens, d ** -0.5, whole=False)
    for i in range(b):
        n, m = min(max(lens[i], 0), s), min(max(q_lens[i], 0), l)
        assert (grads[0][i, :, m:] == 0).all() and (grads[1][i, :, n:] == 0).all() and (grads[2][i, :, n:] == 0).all()
    again = ca.cross_attention_backward(dout, q, k, v, out, lse, lens32, q_lens32)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_gradient_is_the_difference(sidon, kind):
    """Along random directions, against differences of the float64 definition: each
    gradient is off by 2 u of its length, so its product with a direction by that times the direction's."""
    q, k, v, dout = inputs(2, 4, 2, 70, 90, 64, kind, 3)
    ca = sidon.cross_attention
    lse = torch.empty(2, 4, 70, device=DEV)
    out = ca.cross_attention(q, k, v, scale=0.1, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, scale=0.1)
    f = lambda *a: float((oracle.cross(*a, None, None, 0.1)[0] * dout.double()).sum())  # noqa: E731
    args, h = [t.double() for t in (q, k, v)], 1e-5
    for i, g in enumerate(grads):
        step = torch.randn(g.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(DEV)
        up, down = ([t + sign * h * step if j == i else t for j, t in enumerate(args)] for sign in (1, -1))
        want = (f(*up) - f(*down)) / (2 * h)
        assert abs(want - float((g.double() * step).sum())) <= torch.finfo(kind).eps * float(g.double().norm() * step.norm())


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -9, 1.0, 2000.0], ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 300, 64), (1, 2, 1, 40, 96, 128)], ids=str)
def test_fp16_gradients_of_any_size(sidon, shape, size):
    """dout far from 1, and rows of very different size: products past 65504 and below
    fp16's smallest, from which the gradients come out right (up to what they can hold)."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, torch.float16, 11)
    v, k = (4 * v).contiguous(), (k / 4).contiguous()
    dout = (size * dout).contiguous()
    dout[:, :, ::2] /= 64
    ca = sidon.cross_attention
    lse = torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse)
    u = 2.0 ** -11
    want = oracle.cross_grads(dout, q, k, v, None, None, d ** -0.5, u)
    for got, (name, (value, tol)) in zip(grads, want.items()):
        tol = tol + 2.0 ** -24
        far = value.abs() + tol > 65504
        assert torch.isfinite(got[~far]).all(), name
        assert ((got.double() - value).abs() <= tol)[~far].all(), name


@pytest.mark.parametrize("l", [1, 150])
def test_strides_and_out(sidon, l):
    """Contiguous and other orders of q, k, v; outputs inside wider tensors; shared
    keys by a zero stride; an expanded dout; what lies around the outputs stays."""
    b, h, hk, s, d, kind = 2, 4, 2, 233, 64, torch.float16
    q, k, v, dout = inputs(b, h, hk, l, s, d, kind, 9)
    lens = int32([233, 100])
    ca = sidon.cross_attention
    lse = torch.empty(b, h, l, device=DEV)
    want = ca.cross_attention(q, k, v, lens, lse=lse)
    assert torch.equal(ca.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), lens), want)
    keys_first = v.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    heads_first = k.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)
    assert torch.equal(ca.cross_attention(q, heads_first, keys_first, lens), want)
    # q and out as column blocks of one tensor
    wide = torch.full((b, l, 2 * h * d + 64), 7.0, dtype=kind, device=DEV)
    both = wide[..., :-64].unflatten(-1, (2 * h, d)).permute(0, 2, 1, 3)
    both[:, :h] = q
    assert ca.cross_attention(both[:, :h], k, v, lens, out=both[:, h:]).data_ptr() == both[:, h:].data_ptr()
    assert torch.equal(both[:, h:], want) and torch.equal(both[:, :h], q) and (wide[..., -64:] == 7).all()
    one = k[:, :1].expand(b, hk, s, d)
    assert torch.equal(ca.cross_attention(q, one, v, lens), ca.cross_attention(q, one.contiguous(), v, lens))
    grads = ca.cross_attention_backward(dout, q, k, v, want, lse, lens)
    again = ca.cross_attention_backward(dout.contiguous(), q.contiguous(), heads_first, keys_first, want, lse, lens)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
    flat = dout[:, :1, :1].expand(b, h, l, d)
    some = ca.cross_attention_backward(flat, q, k, v, want, lse, lens)
    assert all(torch.equal(x, y) for x, y in zip(some, ca.cross_attention_backward(flat.contiguous(), q, k, v, want, lse, lens)))
    # the gradients of k | v rows in one tensor, as the projection's backward reads them
    rows = torch.full((b, s, 2 * hk * d + 32), 3.0, dtype=kind, device=DEV)
    dkv = rows[..., :-32].unflatten(-1, (2, hk, d)).permute(2, 0, 3, 1, 4)
    got = ca.cross_attention_backward(dout, q, k, v, want, lse, lens, dk=dkv[0], dv=dkv[1])
    assert torch.equal(got[0], grads[0]) and torch.equal(dkv[0], grads[1]) and torch.equal(dkv[1], grads[2])
    assert (rows[..., -32:] == 3).all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("l", [1, 200])
def test_a_query_that_is_no_number(sidon, l, kind):
    """NaN in its own row.  A row whose sum the matrix core takes in one with it has its
    sum taken apart, its 32 fp32 terms in another order: off by less than 32 2^-24 of
    itself, so the result moves by less than 2^-19 of itself, which its rounding turns into
    one step (2 u) at most; every other row keeps its bits."""
    q, k, v, _ = inputs(2, 4, 2, l, 300, 64, kind, 13)
    want = sidon.cross_attention.cross_attention(q, k, v)
    q[1, 2, l // 2, 5] = float("nan")
    got = sidon.cross_attention.cross_attention(q, k, v)
    assert got[1, 2, l // 2].isnan().all()
    got[1, 2, l // 2] = want[1, 2, l // 2]
    err = (got.double() - want.double()).abs()
    assert (err <= torch.finfo(kind).eps * want.double().abs() + tiny(kind)).all()
    assert int((err.amax(-1) > 0).sum()) <= 1   # (of the rows)


@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_captured(sidon, kind):
    """A training step in one graph, replayed on new contents and lengths between eager calls."""
    b, h, hk, l, s, d = 2, 4, 2, 60, 200, 64
    q, k, v, dout = inputs(b, h, hk, l, s, d, kind, 17)
    lens, q_lens = int32([200, 77]), int32([60, 31])
    lse = torch.empty(b, h, l, device=DEV)
    ca = sidon.cross_attention

    def step():
        out = ca.cross_attention(q, k, v, lens, q_lens, lse=lse)
        return out, *ca.cross_attention_backward(dout, q, k, v, out, lse, lens, q_lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        lens.copy_(torch.tensor([50 * i, 200 - i], dtype=torch.int32))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", [(1, 8, 8, 1, 4800, 64), (2, 4, 1, 1, 3000, 128), (3, 8, 4, 100, 900, 64), (4, 16, 4, 500, 1100, 64),
                                   (3, 8, 8, 517, 700, 128)], ids=str)
def test_repeated_calls(sidon, shape, kind):
    """The same bits from every launch, with and without lse, both directions."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = inputs(*shape, kind, 19)
    lens = int32([s - 37 * i for i in range(b)])
    ca = sidon.cross_attention
    lse = torch.empty(b, h, l, device=DEV)
    want = ca.cross_attention(q, k, v, lens, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, want, lse, lens)
    first = lse.clone()
    differ = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(40):
        differ += (ca.cross_attention(q, k, v, lens, lse=lse if i % 2 else None) != want).sum()
        differ += (lse != first).sum()
        if i % 4 == 0:
            for x, y in zip(ca.cross_attention_backward(dout, q, k, v, want, lse, lens), grads):
                differ += (x != y).sum()
    assert int(differ) == 0
