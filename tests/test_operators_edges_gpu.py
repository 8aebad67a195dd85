"""The language-model operators at the ends of their ranges (needs an MI355X):
offsets past 32 bits, launches of many workgroups, every tile of the adapters,
two calls at once, captured calls that share a workspace.  Values are held against
float64, with the tolerances of the operators' own tests, or against the same call
on an ordinary layout, which those tests hold against float64."""

from __future__ import annotations

import threading

import pytest
import test_adapters_gpu as adapters_test
import test_diff_attention_gpu as attention_test
import test_group_norm_gpu as norm_test
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def test_group_norm_of_many_groups(sidon):
    """More (item, group) pairs than a launch has workgroups of 256 threads."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    batch, c, groups = 65535, 2056, 257
    x = torch.randn(batch, c, generator=gen, device=DEV, dtype=torch.float16)
    w = 1 + 0.2 * torch.randn(c, generator=gen, device=DEV)
    b = 0.2 * torch.randn(c, generator=gen, device=DEV)
    got = sidon.conformer.group_norm_act(x, batch, groups, w, b, act=None)
    some = torch.tensor([0, 1, 255, 256, 32767, 65000, 65534], device=DEV)
    v = x[some].double().view(len(some), groups, 8)
    v = (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5)
    want = v.view(len(some), c) * w.double() + b.double()
    # one fp16 rounding; fp32 arithmetic on values below 8
    assert ((got[some].double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -18).all()
    assert torch.isfinite(got).all()


# (items, rows, N, K, R, adapters): every tile of the adapters' second launch, one output type or both (of 16-bit
# outputs 32 x 64, 64 x 64, 64 x 128, 128 x 128, 192 x 128, 128 x 256, 160 x 256, 192 x 256, 320 x 256), with ranks
# that are a power of two and not, items shorter and longer than a tile, and as many as a tile holds
TILES = [(2, 90, 256, 64, 16, 2), (2, 1037, 256, 64, 40, 3), (3, 1037, 512, 64, 16, 2), (3, 1037, 1024, 64, 24, 3),
         (5, 1037, 1024, 64, 64, 2), (13, 90, 4096, 64, 16, 3), (3, 1037, 2048, 64, 40, 2), (2, 1037, 4096, 64, 16, 2),
         (5, 1037, 2048, 64, 64, 6), (8, 600, 4096, 128, 48, 3), (37, 130, 4096, 64, 32, 3), (40, 96, 1024, 64, 128, 5),
         (24, 64, 2048, 128, 64, 2), (9, 333, 2048, 192, 104, 4)]


@pytest.mark.parametrize("kind", adapters_test.KINDS, ids=str)
@pytest.mark.parametrize("shape", TILES, ids=str)
def test_adapter_tiles(sidon, shape, kind):
    s = adapters_test.inputs(*shape, kind, sum(shape))
    # what another adapter's rows would drag in, and rows without one whose low-rank products are left as they are
    ws = torch.full((sidon.adapters.workspace_bytes(s["x"].shape[0], shape[4], True, kind),), 255, dtype=torch.uint8,
                    device=DEV)
    adapters_test.check(adapters_test.linear(sidon, s, workspace=ws), *adapters_test.reference(s, False))
    ws.fill_(255)
    want, tol = adapters_test.reference(s, True)
    adapters_test.check(adapters_test.residual(sidon, s, workspace=ws), want, tol)


def test_adapters_past_32_bits(sidon):
    """Adapters, outputs and the stream at offsets of more than 4 GiB."""
    s = adapters_test.inputs(7, 30, 1024, 1024, 64, 3, torch.float16, 5)
    want, tol = adapters_test.reference(s, False)
    res, res_tol = adapters_test.reference(s, True)
    many = 40000
    a = torch.empty(many, 64, 1024, dtype=torch.float16, device=DEV)
    b = torch.empty(many, 1024, 64, dtype=torch.float16, device=DEV)
    scale = torch.zeros(many, device=DEV)
    a[-3:], b[-3:], scale[-3:] = s["a"], s["b"], s["scale"]
    s.update(a=a, b=b, scale=scale, ids=torch.where(s["ids"] < 0, -1, s["ids"] + many - 3).int())
    adapters_test.check(adapters_test.linear(sidon, s), want, tol)
    del a, b
    s.update(a=s["a"][-3:].clone(), b=s["b"][-3:].clone(), scale=scale[-3:].clone(),
             ids=torch.where(s["ids"] < 0, -1, s["ids"] - many + 3).int())
    out = torch.empty(210, 1 << 24, dtype=torch.float16, device=DEV)[:, :1024]
    adapters_test.check(adapters_test.linear(sidon, s, out=out), want, tol)
    del out
    stream = torch.empty(210, 1 << 23, device=DEV)[:, 64:1088]
    stream.copy_(s["y"])
    s["y"] = stream
    adapters_test.check(adapters_test.residual(sidon, s), res, res_tol)


def test_attention_past_32_bits(sidon):
    """Queries, a cache and an output whose rows, heads and items lie gibibytes apart."""
    q, k, v, lam, norm_w = attention_test.inputs(2, 2, 1, 40, 33, 64, torch.bfloat16, 4)
    lens = torch.tensor([33, 20], dtype=torch.int32, device=DEV)
    for length in (40, 1):
        want = sidon.diff_attention.diff_attention(q[:, :, :, :length], k, v, lam, 0.3, lens=lens, norm_w=norm_w)
        row = (1 << 25) - 8
        cache = torch.empty(35 * row + (1 << 31), dtype=torch.bfloat16, device=DEV)
        far_k = cache.as_strided(k.shape, (1 << 31, 0, row // 2 // 8 * 8, row, 1), 64)
        far_v = cache.as_strided(v.shape, (1 << 31, 0, row, 1), 4096)
        far_k.copy_(k)
        far_v.copy_(v)
        q_row = 1 << 26
        far_q = torch.empty(41 * q_row, dtype=torch.bfloat16, device=DEV).as_strided(
            (2, 2, 2, length, 64), (256, 1 << 25, 128, q_row, 1))
        far_q.copy_(q[:, :, :, :length])
        out = torch.empty(41 * q_row, dtype=torch.bfloat16, device=DEV).as_strided(
            (2, 2, length, 128), (q_row // 4, q_row // 2, q_row, 1))
        sidon.diff_attention.diff_attention(far_q, far_k, far_v, lam, 0.3, lens=lens, norm_w=norm_w, out=out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("shape", [(1, 2, 1, 1, 131072, 64), (2, 2, 2, 1, 40000, 128), (1, 1, 1, 9000, 9001, 64)],
                         ids=str)
def test_attention_of_long_caches(sidon, shape):
    b, h, hk, l, s, d = shape
    q, k, v, lam, norm_w = attention_test.inputs(b, h, hk, l, s, d, torch.bfloat16, 9)
    lens = [s, s - 4321][:b]
    attention_test.poison(k, v, lens)
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                              causal=True, norm_w=norm_w)
    attention_test.check(got, *attention_test.reference(q, k, v, lam, 0.3, lens, True, norm_w, 1e-5))


@pytest.mark.parametrize("shape", [(1, 2, 1, 1, 262144, 64), (2, 2, 2, 1, 40000, 128), (1, 1, 1, 70, 120000, 64)], ids=str)
def test_attention_of_long_fp16_caches(sidon, shape):
    """Scores of a few standard deviations more than the others' in some keys: what
    the rest is worth lies below fp16's smallest normal number relative to them."""
    b, h, hk, l, s, d = shape
    q, k, v, lam, norm_w = attention_test.inputs(b, h, hk, l, s, d, torch.float16, 9)
    k[:, :, :, ::911] *= 3
    lens = [s, s - 4321][:b]
    attention_test.poison(k, v, lens)
    got = sidon.diff_attention.diff_attention(q, k, v, lam, 0.3, lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                              causal=True, norm_w=norm_w)
    attention_test.check(got, *attention_test.reference(q, k, v, lam, 0.3, lens, True, norm_w, 1e-5))


def test_group_norm_past_32_bits(sidon):
    x, w, b = norm_test.inputs(60, 256, torch.float16, 6)
    lens = torch.tensor([30, 17], dtype=torch.int32, device=DEV)
    for groups in (8, 2, 64):
        want = sidon.conformer.group_norm_act(x, 2, groups, w, b, lens=lens)
        far = torch.empty(60, 1 << 26, dtype=torch.float16, device=DEV)
        far[:, 512:768] = x
        got = sidon.conformer.group_norm_act(far[:, 512:768], 2, groups, w, b, lens=lens, out=far[:, 1024:1280])
        assert torch.equal(got, want)
        sidon.conformer.group_norm_act(far[:, 512:768], 2, groups, w, b, lens=lens, out=far[:, 512:768])
        assert torch.equal(far[:, 512:768], want)


def test_sizes_and_strides_past_32_bits_are_refused(sidon):
    """The ABI's ints hold 32 bits: 2^32 + n would arrive as n, and the call would
    read or write other rows than it was given."""
    far = 1 << 32
    s = adapters_test.inputs(2, 1, 64, 64, 8, 2, torch.float16, 3)
    half = torch.empty(far + 256, dtype=torch.float16, device=DEV)
    rows = lambda t: t.as_strided((2, 64), (far + 64, 1))  # noqa: E731
    with pytest.raises(ValueError, match="32 bits"):
        adapters_test.linear(sidon, {**s, "x": rows(half)})
    with pytest.raises(ValueError, match="32 bits"):
        adapters_test.linear(sidon, {**s, "w": rows(half), "b": s["b"][:, :2].contiguous(), "bias": None})
    with pytest.raises(ValueError, match="32 bits"):
        adapters_test.linear(sidon, s, out=rows(half))
    x = half[:far + 64].view(1, -1)
    with pytest.raises(ValueError, match="32 bits"):
        sidon.conformer.group_norm_act(x, 1, 1, torch.empty(far + 64, device=DEV), torch.empty(far + 64, device=DEV))
    with pytest.raises(ValueError, match="32 bits"):
        sidon.conformer.group_norm_act(x.view(-1, 1), 1, 1, torch.ones(1, device=DEV), torch.zeros(1, device=DEV))
    del half, x
    full = torch.empty(far + 256, device=DEV)
    for over in (dict(out=rows(full)), dict(y=rows(full))):
        with pytest.raises(ValueError, match="32 bits"):
            adapters_test.residual(sidon, {**s, "y": over.pop("y", s["y"])}, **over)
    del full
    q, k, v, lam, _ = attention_test.inputs(1, 1, 1, 1, 1, 64, torch.float16, 1)
    with pytest.raises(ValueError, match="32 bits"):
        sidon.diff_attention.diff_attention(q, k.expand(1, 1, 2, far + 33, 64), v.expand(1, 1, far + 33, 128), lam, 0.3)


@pytest.mark.parametrize("stride", [67, 0, 1 << 33])
def test_a_single_rows_stride_means_nothing(sidon, stride):
    row = lambda t: t.as_strided((1, t.shape[1]), (stride, 1))  # noqa: E731
    s = adapters_test.inputs(1, 1, 128, 64, 8, 2, torch.float16, 3)
    want, res = adapters_test.linear(sidon, s), adapters_test.residual(sidon, s, out=torch.empty_like(s["y"]))
    out, into = torch.empty_like(want), torch.empty_like(res)
    adapters_test.linear(sidon, {**s, "x": row(s["x"])}, out=row(out))
    adapters_test.residual(sidon, {**s, "x": row(s["x"]), "y": row(s["y"])}, out=row(into))
    assert torch.equal(out, want) and torch.equal(into, res)
    x, w, b = norm_test.inputs(1, 256, torch.float16, 4)
    assert torch.equal(sidon.conformer.group_norm_act(row(x), 1, 8, w, b), sidon.conformer.group_norm_act(x, 1, 8, w, b))


def test_attention_refuses_a_workspace_over_its_operands(sidon):
    """(On a device: the workspace that a call needs depends on it.)"""
    q, k, v, lam, norm_w = attention_test.inputs(1, 8, 8, 1, 4800, 64, torch.float16, 3)
    need = sidon.diff_attention.workspace_bytes(1, 8, 8, 1, 4800, 64, DEV)
    out = torch.empty(1, 8, 1, 128, dtype=torch.float16, device=DEV)
    lens = torch.tensor([4800], dtype=torch.int32, device=DEV)
    assert need > 0
    for t in (q, k, v, lam, norm_w, lens, out):
        ws = torch.as_strided(t, (1,), (1,)).view(torch.uint8).untyped_storage()
        if ws.nbytes() < need:   # the workspace begins at the operand and goes on behind it
            buf = torch.empty(need + 4096, dtype=torch.uint8, device=DEV)
            n = t.numel() * t.element_size()
            moved = buf[:n].view(t.dtype).view(t.shape).copy_(t)
            ws = buf
        else:
            moved, ws = t, torch.empty(0, dtype=torch.uint8, device=DEV).set_(ws)
        a = {"q": q, "k": k, "v": v, "lam": lam, "norm_w": norm_w, "lens": lens, "out": out}
        name = next(n for n, x in a.items() if x is t)
        a[name] = moved
        with pytest.raises(RuntimeError, match="apart"):
            sidon.diff_attention.diff_attention(**a, lam_init=0.3, workspace=ws)


def calls(sidon, seed):
    """One call of each operator with its workspace -> [(call, workspace bytes)]; call(workspace) -> the output."""
    x, w, b = norm_test.inputs(4000, 512, torch.float16, seed)
    s = adapters_test.inputs(6, 200, 1024, 512, 32, 4, torch.float16, seed)
    one = adapters_test.inputs(40, 1, 1024, 512, 16, 30, torch.bfloat16, seed)
    att = attention_test.inputs(2, 8, 4, 1, 3000, 64, torch.float16, seed)
    pro = attention_test.inputs(2, 4, 4, 300, 300, 128, torch.bfloat16, seed)
    d = sidon.diff_attention
    return [
        (lambda ws: sidon.conformer.group_norm_act(x, 2, 4, w, b, workspace=ws),
         sidon.conformer.group_norm_workspace(2, 2000, 512, 4, torch.float16)),
        (lambda ws: adapters_test.linear(sidon, s, act="silu", workspace=ws), sidon.adapters.workspace_bytes(1200, 32)),
        (lambda ws: adapters_test.residual(sidon, one, out=torch.empty_like(one["y"]), workspace=ws),
         sidon.adapters.workspace_bytes(40, 16, True, torch.bfloat16)),
        (lambda ws: d.diff_attention(*att[:4], 0.3, norm_w=att[4], workspace=ws),
         d.workspace_bytes(2, 8, 4, 1, 3000, 64, DEV)),
        (lambda ws: d.diff_attention(*pro[:4], 0.3, causal=True, workspace=ws),
         d.workspace_bytes(2, 4, 4, 300, 300, 128, DEV)),
    ]


def buffer(size):
    return torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)


def test_graphs_that_share_a_workspace(sidon):
    """Captured calls of every operator over one buffer, replayed in turn with
    eager calls over the same buffer between them."""
    todo = calls(sidon, 3)
    ws = buffer(max(size for _, size in todo))
    wants = [call(None).clone() for call, _ in todo]
    torch.cuda.synchronize()
    graphs = []
    for call, size in todo:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(ws)
        graphs.append((graph, out))
    for turn in range(3):
        for i, (graph, out) in enumerate(graphs):
            out.zero_()
            ws.fill_(255)
            graph.replay()
            other, _ = todo[(i + turn) % len(todo)]
            assert torch.equal(other(ws), wants[(i + turn) % len(todo)])
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, wants):
            assert torch.equal(out, want)


def test_two_streams_and_threads_at_once(sidon):
    """Calls side by side, each stream and thread with its own workspaces."""
    todo = calls(sidon, 5)
    wants = [call(None).clone() for call, _ in todo]
    torch.cuda.synchronize()
    wrong = []

    def work(first):
        stream = torch.cuda.Stream()
        spaces = [buffer(size) for _, size in todo]
        with torch.cuda.stream(stream):
            for turn in range(12):
                i = (first + turn) % len(todo)
                out = todo[i][0](spaces[i])
                stream.synchronize()
                if not torch.equal(out, wants[i]):
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
    x, w, b = norm_test.inputs(64, 128, torch.float16, 2)
    lens = torch.tensor([20, 32], dtype=torch.int32, device=DEV)
    norm = sidon.conformer.group_norm_act
    want = norm(x, 2, 4, w, b, lens=lens)
    wide = torch.zeros(64, 192, dtype=torch.float16, device=DEV)
    wide[:, 32:160] = x
    assert torch.equal(norm(wide[:, 32:160], 2, 4, w, b, lens=lens), want)
    for bad in (lens.long(), lens[:1], lens.cpu(), torch.stack([lens, lens], 1)[:, 0]):
        with pytest.raises(ValueError):
            norm(x, 2, 4, w, b, lens=bad)
    for bad in (w.half(), w[:64], w.cpu(), torch.stack([w, w], 1)[:, 0]):
        with pytest.raises(ValueError):
            norm(x, 2, 4, bad, b, lens=lens)
    with pytest.raises(ValueError):
        norm(x, 2, 5, w, b, lens=lens)
    with pytest.raises(ValueError):
        norm(x.t(), 2, 4, w, b, lens=lens)
    assert torch.equal(norm(x, 2, 4, w, b, lens=lens), want)

    s = adapters_test.inputs(6, 3, 128, 64, 8, 2, torch.float16, 3)
    want = adapters_test.linear(sidon, s)
    for name, bad in (("x", s["x"].float()), ("w", s["w"].bfloat16()), ("scale", s["scale"].double()),
                      ("ids", s["ids"].long()), ("a", s["a"].transpose(1, 2)), ("bias", s["bias"][:64]),
                      ("ids", s["ids"][:4]), ("b", s["b"][:1]), ("w", s["w"].cpu())):
        with pytest.raises((ValueError, TypeError)):
            adapters_test.linear(sidon, {**s, name: bad})
    assert torch.equal(adapters_test.linear(sidon, s), want)

    q, k, v, lam, norm_w = attention_test.inputs(2, 4, 2, 3, 50, 64, torch.float16, 7)
    call = sidon.diff_attention.diff_attention
    want = call(q, k, v, lam, 0.3, norm_w=norm_w)
    assert torch.equal(call(q.contiguous(), k, v.contiguous(), lam, 0.3, norm_w=norm_w), want)
    out = torch.zeros(2, 3, 4, 128, dtype=torch.float16, device=DEV)
    assert torch.equal(call(q, k, v, lam, 0.3, norm_w=norm_w, out=out.transpose(1, 2)), want)
    assert torch.equal(call(q, k, v, lam, 0.3, norm_w=norm_w), want)
    for bad in (dict(q=q.float()), dict(k=k[..., :32]), dict(v=v[:1]), dict(lam=lam.half()), dict(lam=lam[:3]),
                dict(norm_w=norm_w[:64]), dict(k=k.cpu()), dict(v=v.bfloat16())):
        a = {"q": q, "k": k, "v": v, "lam": lam, "lam_init": 0.3, "norm_w": norm_w, **bad}
        with pytest.raises((ValueError, TypeError)):
            call(**a)
