"""adapters.adapter_linear / adapter_residual against the definition in float64
(needs an MI355X).

Tolerance, per element, with u = torch.finfo(t).eps / 2 and S = sum |x w| + |scale|
sum |x a| |b| (+ |bias|, |add|): an fp32 sum of K products taken 32 at a time rounds
K / 32 times between the groups and at most 32 times inside one, each 2^-24 of at
most S, and the shared and the low-rank sums, the bias and the stream join in a
few more: (K / 32 + 64) 2^-24 S.  linear also rounds the low-rank products once,
u of each: u |scale| sum_r |x . a_r| |b_r|, and its output: u |y|.  SiLU's slope is at
most 1.1, its hardware exponential is off by at most |v| 2^-22 of a value of at
most |v|.  residual rounds no product (two fp16 or three bf16 summands keep 2^-22
of it, inside the sum's bound)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
KINDS = [torch.float16, torch.bfloat16]


def inputs(items, rows, n, k, r, e, kind, seed):
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape, std=1.0, dtype=kind):
        return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)

    m = items * rows
    return {"x": randn(m, k), "w": randn(n, k, std=k ** -0.5), "bias": randn(n, std=0.1),
            "a": randn(e, r, k, std=k ** -0.5), "b": randn(e, n, r, std=r ** -0.5),
            "scale": randn(e, dtype=torch.float32).abs() + 0.5, "y": randn(m, n, dtype=torch.float32),
            "ids": torch.randint(-1, e, (items,), generator=gen, dtype=torch.int32).to(DEV)}


def reference(s, residual, act=None, bias=True):
    """-> (y, tolerance) in float64."""
    x, w = s["x"].double(), s["w"].double()
    m, k = x.shape
    items, e_all = s["ids"].numel(), s["a"].shape[0]
    u = torch.finfo(s["x"].dtype).eps / 2
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    rounded = torch.zeros_like(y)
    for i, e in enumerate(s["ids"].tolist()):
        if not 0 <= e < e_all:
            continue
        at = slice(i * (m // items), (i + 1) * (m // items))
        a, b, f = s["a"][e].double(), s["b"][e].double(), float(s["scale"][e])
        y[at] += f * (x[at] @ a.t()) @ b.t()
        size[at] += abs(f) * (x[at].abs() @ a.abs().t()) @ b.abs().t()
        rounded[at] = abs(f) * (x[at] @ a.t()).abs() @ b.abs().t() * u
    if residual:
        y, size, rounded = y + s["y"].double(), size + s["y"].double().abs(), 0
    elif bias:
        y, size = y + s["bias"].double(), size + s["bias"].double().abs()
    tol = (k / 32 + 64) * 2.0 ** -24 * size + rounded
    if act == "silu":
        tol = 1.1 * tol + y.square() * 2.0 ** -22
        y = y / (1 + torch.exp(-y))
    tiny = 2.0 ** -25 if s["x"].dtype == torch.float16 else 2.0 ** -100
    return y, tol + (y.abs() * u + tiny if not residual else 0)


def check(got, want, tol):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


def linear(sidon, s, **kw):
    return sidon.adapters.adapter_linear(s["x"], s["w"], kw.pop("bias", s["bias"]), s["a"], s["b"], s["scale"], s["ids"],
                                         **kw)


def residual(sidon, s, **kw):
    return sidon.adapters.adapter_residual(s["y"], s["x"], s["w"], s["a"], s["b"], s["scale"], s["ids"], **kw)


# (items, rows, N, K, R, adapters): one row; single tokens, few and many, an adapter each and shared; items shorter
# than a block, two in a block, as long as a tile; ranks of 8 to 128; a long K; whole chunks
SHAPES = [(1, 1, 64, 64, 8, 1), (1, 1, 1024, 1024, 16, 3), (7, 1, 320, 192, 24, 2), (48, 1, 4096, 1024, 16, 64),
          (300, 1, 256, 128, 40, 30), (700, 1, 128, 576, 64, 90), (33, 3, 512, 320, 32, 5), (5, 17, 192, 1024, 128, 3),
          (9, 64, 1024, 512, 48, 4), (4, 400, 2048, 1024, 32, 6), (2, 1463, 1024, 4096, 16, 2),
          (1, 1037, 2048, 64, 104, 1), (8, 600, 4096, 1024, 64, 8), (1300, 1, 4096, 256, 8, 3)]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_against_float64(sidon, shape, kind):
    s = inputs(*shape, kind, sum(shape))
    act = (None, "silu")[sum(shape) % 2]
    check(linear(sidon, s, act=act), *reference(s, False, act))
    check(linear(sidon, s, bias=None), *reference(s, False, bias=False))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_residual_against_float64(sidon, shape, kind):
    s = inputs(*shape, kind, sum(shape) + 1)
    before = s["y"].clone()
    want, tol = reference(s, True)
    out = residual(sidon, s, out=torch.empty_like(before))
    check(out, want, tol)
    assert torch.equal(s["y"], before)
    assert residual(sidon, s) is s["y"]
    assert torch.equal(s["y"], out)


# binary orders of x, a, w, b, scale: small products with a large b, products past fp16's largest number, small ones
# from a and from the scale, a tiny x, a large scale
ORDERS = [(0, -14, 0, 14, 0), (10, 2, -8, -16, 2), (0, -12, 0, 0, -12), (-6, 0, 0, 15, -8), (0, 0, 0, -10, 17)]
PATHS = [(40, 1, 256, 256, 16, 30), (4, 100, 512, 256, 64, 3), (10, 7, 192, 320, 40, 6), (5, 1037, 1024, 64, 64, 2),
         (9, 333, 2048, 192, 104, 4), (3, 1, 64, 64, 8, 2), (8, 600, 4096, 128, 48, 3)]


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("orders", ORDERS, ids=str)
@pytest.mark.parametrize("shape", PATHS, ids=str)
def test_low_rank_products_of_any_size(sidon, shape, orders, kind):
    s = inputs(*shape, kind, sum(shape) + 3)
    for name, p in zip(("x", "a", "w", "b", "scale"), orders):
        s[name] = (s[name].float() * 2.0 ** p).to(s[name].dtype)
    check(linear(sidon, s), *reference(s, False))
    want, tol = reference(s, True)
    check(residual(sidon, s), want, tol)


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("shape", PATHS, ids=str)
def test_rows_that_are_no_numbers(sidon, shape, kind):
    """An infinity or a NaN in a row of x stays in that row, and a row of zeros
    keeps what the stream holds."""
    s = inputs(*shape, kind, sum(shape) + 4)
    want, tol = reference(s, False)
    res, res_tol = reference(s, True)
    rows = torch.arange(s["x"].shape[0], device=DEV)
    s["x"][rows % 7 == 2, 5] = float("inf")
    s["x"][rows % 7 == 6, 9] = float("nan")
    s["x"][0] = 0
    clean = (rows % 7 != 2) & (rows % 7 != 6) & (rows != 0)
    got, got_res = linear(sidon, s), residual(sidon, s, out=torch.empty_like(s["y"]))
    check(got[clean], want[clean], tol[clean])
    check(got_res[clean], res[clean], res_tol[clean])
    bad = ~clean & (rows != 0)
    assert not torch.isfinite(got[bad]).any() and not torch.isfinite(got_res[bad]).any()
    assert torch.equal(got[0], s["bias"]) and torch.equal(got_res[0], s["y"][0])


@pytest.mark.parametrize("items,rows", [(40, 1), (10, 7), (3, 100)])
def test_ids_outside_and_adapters_of_others(sidon, items, rows):
    """Ids below, at and past the adapters leave the row as the shared
    projection makes it; an adapter full of infinities reaches only its own
    rows; a batch equals its items alone."""
    s = inputs(items, rows, 256, 320, 16, 6, torch.float16, 3)
    s["ids"] = torch.tensor([(0, -1, 1, 6, 2, -2 ** 31, 3, 2 ** 31 - 1, 4)[i % 9] for i in range(items)],
                            dtype=torch.int32, device=DEV)
    want, tol = reference(s, False)
    check(linear(sidon, s), want, tol)
    s["a"][5], s["b"][5], s["scale"][5] = float("inf"), float("nan"), float("nan")
    check(linear(sidon, s), want, tol)
    s["b"][2] = float("nan")
    got = linear(sidon, s).view(items, rows, -1)
    assert torch.equal(torch.isnan(got).any(-1).any(-1), s["ids"] == 2)
    clean = s["ids"] != 2
    check(got[clean], want.view(items, rows, -1)[clean], tol.view(items, rows, -1)[clean])


def test_views(sidon):
    """Rows inside wider tensors; what lies around the outputs stays."""
    s = inputs(6, 35, 192, 256, 24, 4, torch.bfloat16, 8)
    want, res = linear(sidon, s), residual(sidon, s, out=torch.empty_like(s["y"]))
    wide_x = torch.randn(210, 512, device=DEV).to(torch.bfloat16)
    wide_x[:, 128:384] = s["x"]
    wide_w = torch.randn(192, 264, device=DEV).to(torch.bfloat16)
    wide_w[:, :256] = s["w"]
    s["x"], s["w"] = wide_x[:, 128:384], wide_w[:, :256]
    out = torch.full((210, 256), 7.0, device=DEV, dtype=torch.bfloat16)
    linear(sidon, s, out=out[:, 32:224])
    assert torch.equal(out[:, 32:224], want) and (out[:, :32] == 7).all() and (out[:, 224:] == 7).all()
    out = torch.full((210, 256), 7.0, device=DEV)
    residual(sidon, s, out=out[:, 32:224])
    assert torch.equal(out[:, 32:224], res) and (out[:, :32] == 7).all() and (out[:, 224:] == 7).all()


def test_packing(sidon):
    """Adapters of different ranks, and three projections fused into one."""
    gen = torch.Generator().manual_seed(4)
    r = lambda *shape: torch.randn(*shape, generator=gen) * shape[-1] ** -0.5  # noqa: E731
    pairs = [sidon.adapters.stack_adapters([(r(q, 128), r(64, q)) for q in ranks]) for ranks in ((3, 5, 4), (8, 1, 2))]
    a, b, scale = sidon.adapters.pack_adapters(pairs, [0.25, 2.0], device=DEV)
    assert tuple(a.shape) == (2, 16, 128) and tuple(b.shape) == (2, 192, 16)
    s = inputs(4, 9, 192, 128, 8, 1, torch.float16, 6)
    s.update(a=a, b=b, scale=scale, ids=torch.tensor([1, 0, -1, 1], dtype=torch.int32, device=DEV))
    check(linear(sidon, s), *reference(s, False))
    x = s["x"][9:18].double().cpu()
    delta = 0.25 * x @ pairs[0][0].double().t() @ pairs[0][1].double().t()
    bare = linear(sidon, dict(s, ids=s["ids"] * 0 - 1))
    # fp16 copies of A and B and two fp16 outputs: a few 2^-11 of values below 4
    assert (linear(sidon, s)[9:18].double().cpu() - bare[9:18].double().cpu() - delta).abs().max() < 8 * 4 * 2.0 ** -11


def test_streams_and_graphs(sidon):
    for shape in ((48, 1, 1024, 512, 16, 20), (3, 150, 1024, 512, 32, 3)):
        s = inputs(*shape, torch.float16, 2)
        ws = torch.empty(sidon.adapters.workspace_bytes(s["x"].shape[0], shape[4]), dtype=torch.uint8, device=DEV)
        want = linear(sidon, s)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = linear(sidon, s, workspace=ws)
        side.synchronize()
        assert torch.equal(got, want)
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            linear(sidon, s, out=out, workspace=ws)
        for seed in range(3):
            fresh = inputs(*shape, torch.float16, 20 + seed)
            s["x"].copy_(fresh["x"])
            s["ids"].copy_(fresh["ids"])
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, linear(sidon, s))


def test_gradients_are_refused(sidon):
    s = inputs(1, 2, 64, 64, 8, 1, torch.float16, 1)
    s["a"] = torch.nn.Parameter(s["a"])
    with pytest.raises(ValueError, match="no_grad"):
        linear(sidon, s)
    with pytest.raises(ValueError, match="no_grad"):
        residual(sidon, s)
    with torch.no_grad():
        linear(sidon, s)
