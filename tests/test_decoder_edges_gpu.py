"""The decoder's operators at the ends of their ranges (needs an MI355X): offsets
past 32 bits, long caches, many rows, calls side by side, captured calls that share
a workspace, and what they refuse on a device.  Values are held against float64, with
the tolerances of the operators' own tests, or against the same call on an ordinary
layout, which those tests hold against float64."""

from __future__ import annotations

import threading

import pytest
import test_cross_attention_gpu as cross_test
import test_head_norm_gpu as norm_test
import test_int4_gpu as int4_test
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


# ---- offsets past 32 bits, large and small counts --------------------------------------


def far_like(t, row, head, item, at=64):
    """t's values in a tensor whose rows, heads and items lie far apart."""
    b, h, l, d = t.shape
    buf = torch.empty((b - 1) * item + (h - 1) * head + (l - 1) * row + d + at, dtype=t.dtype, device=DEV)
    far = buf.as_strided(t.shape, (item, head, row, 1), at)
    far.copy_(t)
    return far


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("l", [1, 40])
def test_cross_attention_past_32_bits(sidon, l, kind):
    """Queries, a cache, outputs and gradients whose rows, heads and items lie gibibytes apart."""
    q, k, v, dout = cross_test.inputs(2, 2, 1, l, 37, 64, kind, 4)
    lens, ca = cross_test.int32([37, 20]), sidon.cross_attention
    lse = torch.empty(2, 2, l, device=DEV)
    want = ca.cross_attention(q, k, v, lens, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, want, lse, lens)
    row = (1 << 25) - 8   # rows as far apart as they may be; items 4 GiB and more
    k, v = far_like(k, row, 64, 1 << 31), far_like(v, row, 64, (1 << 31) + 64)
    q, dout = far_like(q, row, 128, (1 << 31) - 8 * 9), far_like(dout, row, 1 << 31, 1 << 32)
    out = far_like(torch.zeros_like(want), 1 << 26, 64, 1 << 32)
    far = torch.empty_like(lse)
    ca.cross_attention(q, k, v, lens, out=out, lse=far)
    assert torch.equal(out, want) and torch.equal(far, lse)
    del want
    dq = far_like(torch.zeros_like(grads[0]), 1 << 26, 64, 1 << 32)
    dk, dv = (far_like(torch.zeros_like(g), row, 64, 1 << 32) for g in grads[1:])
    ca.cross_attention_backward(dout, q, k, v, out, lse, lens, dq=dq, dk=dk, dv=dv)
    assert torch.equal(dq, grads[0]) and torch.equal(dk, grads[1]) and torch.equal(dv, grads[2])


@pytest.mark.parametrize("kind", norm_test.KINDS, ids=str)
def test_head_norm_past_32_bits(sidon, kind):
    q, k, qw, kw, cos, sin, pos = norm_test.inputs(2, 30, 2, 1, 64, 64, kind, 6)
    hn = sidon.head_norm
    want = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos)
    grads = hn.qk_norm_rotary_backward(want[0], want[1], q, k, qw, kw, cos, sin, pos, pos)
    dy = [far_like(t, 1 << 26, 256, 1 << 32) for t in want]
    fq, fk = far_like(q, 1 << 26, 64, 1 << 32), far_like(k, 1 << 26, 64, 1 << 32)
    out = far_like(torch.zeros_like(q), 1 << 26, 1 << 31, 1 << 32)
    got = hn.qk_norm_rotary(fq, fk, qw, kw, cos, sin, pos, pos, out_q=out)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = hn.qk_norm_rotary_backward(dy[0], dy[1], fq, fk, qw, kw, cos, sin, pos, pos, dq=dy[0])
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_head_norm_of_many_rows(sidon):
    """More than 2^31 values: sampled tokens and the weights' gradient against float64."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    b, l, h, d = 3, 180000, 64, 64
    rows = torch.randn(b, l, h, d, generator=gen, device=DEV, dtype=torch.bfloat16)
    x = rows.transpose(1, 2)
    w = 1 + 0.1 * torch.randn(d, generator=gen, device=DEV)
    angle = torch.rand(l, 16, generator=gen, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    out = torch.empty_like(rows).transpose(1, 2)
    hn = sidon.head_norm
    hn.qk_norm_rotary(x, None, w, None, cos, sin, out_q=out)
    some = torch.tensor([0, 1, 4095, 4096, 65535, 65536, 131072, l - 1], device=DEV)
    places = some.int().expand(b, -1)
    want, size = oracle.norm_rotary(x[:, :, some], w, cos, sin, places, norm_test.EPS, False)
    norm_test.close(out[:, :, some], want, size)
    dout = out[:, :, some].clone()
    got = hn.qk_norm_rotary_backward(out, None, x, None, w, None, cos, sin, dq=out)
    want, size, _, _ = oracle.norm_rotary_grads(dout, x[:, :, some], w, cos, sin, places, norm_test.EPS, False)
    norm_test.close(got[0][:, :, some], want, size, 64)
    # dout = R (w n) turned back is w n, so dw = w sum n^2 but for dout's roundings, 2^-9 of a term at most and of
    # random sign: 2^-9 / sqrt(3.4e7) of the sum, under 2^-18.  The sum's fp32: a team's 3.4e7 / (1024 * 32) = 1055 rows and
    # under 900 additions behind it, 2^-13 of terms of one sign
    n2 = torch.zeros(d, dtype=torch.float64, device=DEV)
    for at in range(0, l, 10000):
        part = rows[:, at:at + 10000].double().square()
        n2 += (part / (part.mean(-1, keepdim=True) + norm_test.EPS)).sum((0, 1, 2))
    assert ((got[2].double() - w.double() * n2).abs() <= (2.0 ** -13 + 2.0 ** -18) * w.double().abs() * n2).all()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_int4_past_32_bits(sidon, kind):
    """x and y of more than 4 GiB, a block of rows at the far end; weights of many rows."""
    x, values, scales, zero, bias = int4_test.inputs(70, 48, 256, 64, True, kind, 3)
    packed = sidon.int4.pack_int4(values, scales, zero)
    want = sidon.int4.int4_linear(x, packed, bias)
    wide = torch.empty(70, 1 << 26, dtype=kind, device=DEV)
    wide[:, :256] = x
    out = wide[:, 1 << 25:(1 << 25) + 48]
    sidon.int4.int4_linear(wide[:, :256], packed, bias, out=out)
    assert torch.equal(out, want)
    del wide, out
    n, k = 1 << 22, 2560   # words past 4 GiB
    gen = torch.Generator(device=DEV).manual_seed(2)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (n // 16, k // 128, 64, 4), generator=gen, device=DEV, dtype=torch.int32)
    scales = torch.full((n // 16, k // 128, 4, 16), 0.0625, dtype=kind, device=DEV)
    off = torch.full_like(scales, 136.0 if kind == torch.bfloat16 else 0.0)
    pair = torch.stack((scales, off), -1).view(torch.int32).squeeze(-1)
    big = sidon.int4.Int4Weight(words, pair, n, k, 32, kind, False)
    x = torch.randn(3, k, generator=gen, device=DEV).to(kind)
    got = sidon.int4.int4_linear(x, big)
    for first in (0, n // 2, n - 32):   # the same weights from a tensor of their own
        tiles = slice(first // 16, first // 16 + 2)
        few = sidon.int4.Int4Weight(words[tiles].contiguous(), pair[tiles].contiguous(), 32, k, 32, kind, False)
        part, far = sidon.int4.int4_linear(x, few).double(), got[:, first:first + 32].double()
        # (the rule may divide K otherwise: two results of the operator's own tolerance)
        size = x.double().abs().sum(1, keepdim=True) * 16 * 0.0625
        tol = torch.finfo(kind).eps / 2 * (part.abs() + far.abs()) + 2 * 2.0 ** -13 * size
        assert ((far - part).abs() <= tol).all() and part.abs().mean() > 8 * tol.mean()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 1, 1, 262144, 64), (2, 2, 2, 1, 40000, 128), (1, 1, 1, 9000, 9001, 64),
                                   (1, 1, 1, 70, 120000, 128)], ids=str)
def test_cross_attention_of_long_caches(sidon, shape, kind):
    """Scores of a few standard deviations more than the others' in some keys: what
    the rest is worth lies below fp16's smallest normal number relative to them."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = cross_test.inputs(*shape, kind, 9)
    k[:, :, ::911] *= 3
    lens = [s, s - 4321][:b]
    cross_test.poison(lens, None, q, k, v, dout)
    lse = torch.empty(b, h, l, device=DEV)
    got = sidon.cross_attention.cross_attention(q, k, v, cross_test.int32(lens), lse=lse)
    cross_test.check_forward(got, lse, q, k, v, lens, None, d ** -0.5)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 1, 3, 40000, 64), (1, 1, 1, 2000, 4500, 64), (1, 2, 1, 4500, 40, 128)], ids=str)
def test_gradients_of_long_sequences(sidon, shape, kind):
    b, h, hk, l, s, d = shape
    q, k, v, dout = cross_test.inputs(*shape, kind, 10)
    lens = [s - 7]
    cross_test.poison(lens, None, q, k, v, dout)
    lse, ca = torch.empty(b, h, l, device=DEV), sidon.cross_attention
    out = ca.cross_attention(q, k, v, cross_test.int32(lens), lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, cross_test.int32(lens))
    cross_test.check_backward(grads, dout, q, k, v, lens, None, d ** -0.5, whole=False)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_many_items(sidon, kind):
    """Many items of a few tokens and keys, some without any."""
    b, h, hk, l, s, d = 30000, 4, 2, 2, 5, 64
    q, k, v, dout = cross_test.inputs(b, h, hk, l, s, d, kind, 12)
    lens = torch.arange(b, device=DEV).remainder(s + 1).int()
    lse, ca = torch.empty(b, h, l, device=DEV), sidon.cross_attention
    out = ca.cross_attention(q, k, v, lens, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, lens)
    for at in (0, 1, 12345, b - 6):
        few = slice(at, at + 6)
        some = lens[few].tolist()
        cross_test.check_forward(out[few], lse[few], q[few], k[few], v[few], some, None, d ** -0.5)
        cross_test.check_backward([g[few] for g in grads], dout[few], q[few], k[few], v[few], some, None, d ** -0.5, False)
    assert all(torch.isfinite(t).all() for t in (out, *grads)) and (out[lens == 0] == 0).all()


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s", [1, 15, 32, 33, 64, 65, 129])
def test_every_length_of_keys(sidon, s, d, kind):
    """Items with every number of valid keys up to S, and lengths out of range, in one call."""
    lens = [*range(0, s + 1)][::max(1, s // 20)] + [s, -1, -2 ** 31, 2 ** 31 - 1]
    b, l = len(lens), 5
    q, k, v, dout = cross_test.inputs(b, 2, 1, l, s, d, kind, s)
    q_lens = [(3 * i) % (l + 2) - 1 for i in range(b)]
    cross_test.poison(lens, q_lens, q, k, v, dout)
    lse, ca = torch.empty(b, 2, l, device=DEV), sidon.cross_attention
    n, m = cross_test.int32(lens), cross_test.int32(q_lens)
    out = ca.cross_attention(q, k, v, n, m, lse=lse)
    cross_test.check_forward(out, lse, q, k, v, lens, q_lens, d ** -0.5)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, n, m)
    cross_test.check_backward(grads, dout, q, k, v, lens, q_lens, d ** -0.5, False)


# ---- refusals that need a device -------------------------------------------------------


def test_sizes_and_strides_past_the_range_are_refused(sidon):
    ca, hn = sidon.cross_attention, sidon.head_norm
    q, k, v, dout = cross_test.inputs(1, 1, 1, 2, 3, 64, torch.float16, 1)
    lse = torch.empty(1, 1, 2, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    with pytest.raises(ValueError, match="32 bits"):
        ca.cross_attention(q, *(t[:, :, :1].expand(1, 1, (1 << 32) + 3, 64) for t in (k, v)))
    far = torch.empty((1 << 26) + 64, dtype=torch.float16, device=DEV).as_strided((1, 1, 2, 64), (0, 0, 1 << 25, 1))
    with pytest.raises(RuntimeError, match="sidon_cross_attention"):
        ca.cross_attention(q, far, far)
    with pytest.raises(RuntimeError, match="sidon_cross_attention_bwd"):
        ca.cross_attention_backward(far, q, k, v, out, lse)
    with pytest.raises(ValueError, match="32 bits"):
        hn.qk_norm_rotary(q[:, :, :1, :16].expand(1, 1, (1 << 32) + 1, 16), None, torch.ones(16, device=DEV), None)
    # a row of its own: the stride means nothing
    w = torch.ones(64, device=DEV)
    one = q[:, :, :1]
    far_row = one.as_strided((1, 1, 1, 64), (3, 5, 7, 1))
    assert torch.equal(hn.qk_norm_rotary(far_row, None, w, None)[0], hn.qk_norm_rotary(one.contiguous(), None, w, None)[0])
    assert torch.equal(ca.cross_attention(far_row, k, v), ca.cross_attention(one, k, v))
    x, values, scales, zero, bias = int4_test.inputs(1, 48, 96, 32, True, torch.float16, 3)
    packed = sidon.int4.pack_int4(values, scales, zero)
    got = sidon.int4.int4_linear(x.as_strided((1, 96), (5, 1)), packed, bias,
                                 out=torch.empty(48, dtype=torch.float16, device=DEV).as_strided((1, 48), (0, 1)))
    assert torch.equal(got, sidon.int4.int4_linear(x, packed, bias))


@pytest.mark.parametrize("l", [1, 200])
def test_workspaces_over_operands_are_refused(sidon, l):
    ca = sidon.cross_attention
    b, h, hk, s, d = 1, 8, 8, 4800, 64
    q, k, v, dout = cross_test.inputs(b, h, hk, l, s, d, torch.float16, 3)
    need, bneed = ca.workspace_bytes(b, h, hk, l, s, d, DEV), ca.backward_workspace_bytes(b, h, hk, l, s, d, q.dtype)
    lens, q_lens, lse = cross_test.int32([s]), cross_test.int32([l]), torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, lens, q_lens, lse=lse).clone()
    outs = {"dq": torch.empty_like(q), "dk": torch.empty_like(k), "dv": torch.empty_like(v)}
    forward = {"q": q, "k": k, "v": v, "lens": lens, "q_lens": q_lens, "out": out, "lse": lse}
    assert bneed > 0 and (l > 1 or need > 0)
    for need, call, a in ((need, ca.cross_attention, forward), (bneed, ca.cross_attention_backward, {"dout": dout, **forward, **outs})):
        if need == 0:
            continue
        for name, t in a.items():
            n = t.numel() * t.element_size()
            buf = torch.empty(need + n + 4096, dtype=torch.uint8, device=DEV)
            moved = buf[:n].view(t.dtype).view(t.shape).copy_(t)
            with pytest.raises(RuntimeError, match="apart"):
                call(**{**a, name: moved}, workspace=buf)
        with pytest.raises(ValueError, match="workspace"):
            call(**a, workspace=torch.empty(need - 1, dtype=torch.uint8, device=DEV))
        with pytest.raises(ValueError, match="workspace"):
            call(**a, workspace=torch.empty(need, device=DEV))
        with pytest.raises(RuntimeError, match="aligned"):
            call(**a, workspace=torch.empty(need + 16, dtype=torch.uint8, device=DEV)[4:])


def test_tensors_that_need_a_gradient_are_refused(sidon):
    ca, hn = sidon.cross_attention, sidon.head_norm
    q, k, v, dout = cross_test.inputs(1, 2, 1, 4, 9, 64, torch.float16, 1)
    lse, w = torch.empty(1, 2, 4, device=DEV), torch.ones(64, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    needs = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    for i in range(3):
        a = [needs(t) if i == j else t for j, t in enumerate((q, k, v))]
        with pytest.raises(ValueError, match="no_grad"):
            ca.cross_attention(*a)
        with pytest.raises(ValueError, match="no_grad"):
            ca.cross_attention_backward(dout, *a, out, lse)
        with torch.no_grad():
            assert torch.equal(ca.cross_attention(*a), out)
    for a in ((needs(q), k, w, w), (q, needs(k), w, w), (q, k, needs(w), w), (q, k, w, needs(w))):
        with pytest.raises(ValueError, match="no_grad"):
            hn.qk_norm_rotary(*a)
        with pytest.raises(ValueError, match="no_grad"):
            hn.qk_norm_rotary_backward(q, k, *a)
    x, values, scales, zero, bias = int4_test.inputs(2, 48, 96, 32, True, torch.float16, 3)
    packed = sidon.int4.pack_int4(values, scales, zero)
    for a in ((needs(x), packed, bias), (x, packed, needs(bias))):
        with pytest.raises(ValueError, match="no_grad"):
            sidon.int4.int4_linear(*a)


# ---- calls side by side ----------------------------------------------------------------


def calls(sidon, seed):
    """Calls of each operator with their workspaces -> [(call, workspace bytes)]; call(workspace) -> the outputs."""
    ca, hn = sidon.cross_attention, sidon.head_norm
    one = cross_test.inputs(2, 8, 4, 1, 3000, 64, torch.float16, seed)
    pro = cross_test.inputs(2, 4, 4, 300, 300, 128, torch.bfloat16, seed)
    back = cross_test.inputs(2, 4, 2, 130, 300, 64, torch.float16, seed)
    small = cross_test.inputs(1, 4, 2, 20, 500, 64, torch.bfloat16, seed)
    q, k, qw, kw, cos, sin, pos = norm_test.inputs(2, 333, 8, 2, 64, 64, torch.bfloat16, seed)
    x, values, scales, zero, bias = int4_test.inputs(20, 1024, 1024, 64, True, torch.float16, seed)
    packed = sidon.int4.pack_int4(values, scales, zero)

    def train(q, k, v, dout, ws):
        lse = torch.empty(q.shape[:3], device=DEV)
        out = ca.cross_attention(q, k, v, lse=lse)
        return out, *ca.cross_attention_backward(dout, q, k, v, out, lse, workspace=ws)

    def bytes_of(q, k):
        return ca.backward_workspace_bytes(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], q.dtype)

    return [
        (lambda ws: (ca.cross_attention(*one[:3], workspace=ws),), ca.workspace_bytes(2, 8, 4, 1, 3000, 64, DEV)),
        (lambda ws: (ca.cross_attention(*pro[:3], workspace=ws),), ca.workspace_bytes(2, 4, 4, 300, 300, 128, DEV)),
        (lambda ws: train(*back, ws), bytes_of(*back[:2])),
        (lambda ws: train(*small, ws), bytes_of(*small[:2])),
        (lambda ws: hn.qk_norm_rotary_backward(q, k, q, k, qw, kw, cos, sin, pos, pos, workspace=ws),
         hn.workspace_bytes(2, 8, 2, 333, 333, 64)),
        (lambda ws: hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos), 0),
        (lambda ws: (sidon.int4.int4_linear(x, packed, bias, "silu"),), 0),
    ]


def buffer(size):
    return torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_that_share_a_workspace(sidon):
    """Captured calls of every operator over one buffer, replayed in turn with
    eager calls over the same buffer between them."""
    todo = calls(sidon, 3)
    ws = buffer(max(size for _, size in todo))
    wants = [call(None) for call, _ in todo]
    torch.cuda.synchronize()
    graphs = []
    for call, _ in todo:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call(ws)
        graphs.append((graph, outs))
    for turn in range(3):
        for i, (graph, outs) in enumerate(graphs):
            for out in outs:
                out.zero_()
            ws.fill_(255)
            graph.replay()
            other, _ = todo[(i + turn) % len(todo)]
            assert same(other(ws), wants[(i + turn) % len(todo)])
        torch.cuda.synchronize()
        for (_, outs), want in zip(graphs, wants):
            assert same(outs, want)


def test_streams_and_threads_at_once(sidon):
    """Calls side by side, each stream and thread with its own workspaces."""
    todo = calls(sidon, 5)
    wants = [call(None) for call, _ in todo]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        stream = torch.cuda.Stream()
        spaces = [buffer(size) for _, size in todo]
        with torch.cuda.stream(stream):
            for turn in range(14):
                i = (first + turn) % len(todo)
                outs = todo[i][0](spaces[i])
                stream.synchronize()
                if not same(outs, wants[i]):
                    wrong.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_calls_of_other_layouts_are_checked_again(sidon):
    """What one call's checks found serves only calls of the same shapes,
    strides, types and devices."""
    ca, hn = sidon.cross_attention, sidon.head_norm
    q, k, v, dout = cross_test.inputs(2, 4, 2, 3, 50, 64, torch.float16, 7)
    lens, lse = cross_test.int32([50, 20]), torch.empty(2, 4, 3, device=DEV)
    want = ca.cross_attention(q, k, v, lens, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, want, lse, lens)
    assert torch.equal(ca.cross_attention(q.contiguous(), k, v.contiguous(), lens), want)
    for bad in (dict(q=q.float()), dict(k=k[..., :32]), dict(v=v[:1]), dict(lens=lens.long()), dict(lens=lens[:1]),
                dict(lens=lens.cpu()), dict(q_lens=lens.float()), dict(k=k.cpu()), dict(v=v.bfloat16()),
                dict(lse=lse.half()), dict(lse=lse[:, :2]), dict(out=want.float()), dict(out=want[:1])):
        a = {"q": q, "k": k, "v": v, "lens": lens, "lse": lse, **bad}
        with pytest.raises((ValueError, TypeError)):
            ca.cross_attention(**a)
        if "out" not in bad:
            with pytest.raises((ValueError, TypeError)):
                ca.cross_attention_backward(dout, **{"out": want, **a})
    for bad in (dict(dout=dout.bfloat16()), dict(out=want[:, :2]), dict(dq=q.float()), dict(dk=q), dict(dv=v.cpu())):
        with pytest.raises((ValueError, TypeError)):
            ca.cross_attention_backward(**{"dout": dout, "q": q, "k": k, "v": v, "out": want, "lse": lse, "lens": lens, **bad})
    assert torch.equal(ca.cross_attention(q, k, v, lens), want)
    assert same(ca.cross_attention_backward(dout, q, k, v, want, lse, lens), grads)

    q, k, qw, kw, cos, sin, pos = norm_test.inputs(2, 12, 4, 2, 64, 32, torch.float16, 8)
    want = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos)
    names = ("q", "k", "q_w", "k_w", "cos", "sin", "q_pos", "k_pos")
    for name, bad in (("q", q.bfloat16()), ("k", k[:1]), ("q_w", qw.half()), ("k_w", kw[:32]), ("k_w", None),
                      ("cos", cos[:5]), ("sin", sin.double()), ("q_pos", pos.long()), ("k_pos", pos[:, :5]),
                      ("sin", sin.cpu()), ("k", k.cpu()), ("q_pos", pos.t())):
        with pytest.raises((ValueError, TypeError)):
            hn.qk_norm_rotary(**{**dict(zip(names, (q, k, qw, kw, cos, sin, pos, pos))), name: bad})
    assert same(hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos), want)
