"""int4_linear against the definition in float64 (needs an MI355X).

Tolerance.  Weights become operands exactly (fp16 v - 8, bf16 128 + v), products and
sums are fp32: with size = sum |x| 16 s, bf16's operands up to 143 and what goes off
them (the group's sum of x times up to 143) are at most 9 size each, in at most 8 + 3
additions of matrix instructions' rounded sums a group and K / group + 8 after it, so under
(2 * 9 * 32 + K / 32) 2^-24 size in all, taken as 2^-13 size (K <= 4096: 704 2^-24 = 2^-14.5).  The
result is rounded once, u of itself; SiLU's slope is at most 1.1."""

from __future__ import annotations

import pytest
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def inputs(m, n, k, group, zeros, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen).to(kind).to(DEV)
    values = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8).to(DEV)
    scales = (torch.rand(n, k // group, generator=gen) * k ** -0.5 + 0.01).to(kind).to(DEV)
    zero = torch.randint(0, 16, (n, k // group), generator=gen, dtype=torch.uint8).to(DEV) if zeros else None
    return x, values, scales, zero, torch.randn(n, generator=gen).to(kind).to(DEV)


def close(got, want, size):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -13 * size + 2.0 ** -25
    assert (err <= tol).all(), (float((err - tol).max()), float((err / tol).max()))


SHAPES = [
    # (M, N, K, group): a row, tails of every kind, each tile of rows and of outputs
    (1, 1, 32, 32), (1, 16, 128, 128), (1, 17, 96, 32), (3, 100, 192, 64), (16, 33, 4096, 128), (17, 1024, 1024, 64),
    (31, 15, 1056, 32), (32, 4096, 1024, 128), (33, 257, 640, 128), (64, 129, 2048, 64), (65, 64, 512, 256),
    (200, 511, 384, 128), (1, 40000, 256, 32), (20, 33000, 128, 128), (50, 32800, 160, 32), (5, 2048, 3200, 128),
]


@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_float64(sidon, shape, kind, zeros):
    m, n, k, group = shape
    x, values, scales, zero, bias = inputs(m, n, k, group, zeros, kind, m + n + k)
    act, bias = (None, bias) if m % 2 else ("silu", None if n % 2 else bias)
    packed = sidon.int4.pack_int4(values, scales, zero)
    got = sidon.int4.int4_linear(x, packed, bias, act)
    assert got.shape == (m, n) and got.dtype == kind
    close(got, *oracle.int4(x, values, scales, zero, bias, act))


@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 4500, 128, 128), (16, 8190, 1184, 32), (20, 6001, 256, 64), (50, 5000, 160, 32), (64, 8177, 2048, 128),
                                   (300, 1000, 640, 128), (33, 16500, 64, 64), (7, 16400, 256, 64)], ids=str)
def test_tiles_of_a_wavefront(sidon, shape, kind, zeros):
    """Two tiles of outputs, and four with K over eight wavefronts, with tails of rows, outputs and inputs."""
    m, n, k, group = shape
    x, values, scales, zero, bias = inputs(m, n, k, group, zeros, kind, m + n + k)
    got = sidon.int4.int4_linear(x, sidon.int4.pack_int4(values, scales, zero), bias)
    close(got, *oracle.int4(x, values, scales, zero, bias, None))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_every_value_and_place(sidon, kind):
    """One-hot rows read single weights exactly: every nibble of a word, every value."""
    k, n, group = 256, 48, 32
    values = (torch.arange(n).view(n, 1) * 7 + torch.arange(k) * 5).remainder(16).to(torch.uint8).to(DEV)
    scales = torch.ones(n, k // group, dtype=kind, device=DEV)
    zero = torch.arange(n * k // group).remainder(16).to(torch.uint8).view(n, -1).to(DEV)
    x = torch.eye(k, dtype=kind, device=DEV)
    for z in (None, zero):
        got = sidon.int4.int4_linear(x, sidon.int4.pack_int4(values, scales, z))
        want = values.float() - (8 if z is None else z.float().repeat_interleave(group, 1))
        assert torch.equal(got.float(), want.t())


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_strides_and_out(sidon, kind):
    x, values, scales, zero, bias = inputs(9, 70, 256, 64, True, kind, 3)
    packed = sidon.int4.pack_int4(values, scales, zero)
    want = sidon.int4.int4_linear(x, packed, bias)
    wide = torch.full((9, 256 + 72), 5.0, dtype=kind, device=DEV)
    wide[:, :256] = x
    out = wide[:, 257:327]   # a column block of x's tensor, 2-byte aligned
    assert sidon.int4.int4_linear(wide[:, :256], packed, bias, out=out) is out
    assert torch.equal(out, want) and (wide[:, 256] == 5).all() and (wide[:, 327:] == 5).all()
    assert torch.equal(wide[:, :256], x)
    # a row alone gives the bits it gives among others of its tile
    assert torch.equal(sidon.int4.int4_linear(x[4:5], packed, bias), want[4:5])


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_a_row_that_is_no_number(sidon, kind):
    x, values, scales, zero, bias = inputs(20, 64, 256, 128, True, kind, 5)
    packed = sidon.int4.pack_int4(values, scales, zero)
    want = sidon.int4.int4_linear(x, packed, bias)
    x[7, 3], x[18, 100] = float("nan"), float("inf")
    got = sidon.int4.int4_linear(x, packed, bias)
    assert not torch.isfinite(got[7]).any() and not torch.isfinite(got[18]).all()
    rest = [i for i in range(20) if i not in (7, 18)]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_quantized(sidon, kind, zeros):
    """quantize_int4's weights are within half a step of w (and of the scale's and the zero
    point's own roundings: a step in all), through the kernel."""
    gen = torch.Generator().manual_seed(9)
    w = (torch.randn(96, 512, generator=gen) * 0.05).to(kind).to(DEV)
    w[3, :64] = 0
    values, scales, zero = sidon.int4.quantize_int4(w, 64, zeros)
    got = sidon.int4.int4_linear(torch.eye(512, dtype=kind, device=DEV), sidon.int4.pack_int4(values, scales, zero)).t()
    step = scales.float().repeat_interleave(64, 1)
    assert ((got.float() - w.float()).abs() <= 1.1 * step).all() and (got[3, :64] == 0).all()


def test_captured(sidon):
    x, values, scales, zero, bias = inputs(4, 512, 1024, 128, True, torch.bfloat16, 7)
    packed = sidon.int4.pack_int4(values, scales, zero)
    sidon.int4.int4_linear(x, packed, bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sidon.int4.int4_linear(x, packed, bias, "silu")
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = sidon.int4.int4_linear(x, packed, bias, "silu")
        torch.cuda.synchronize()
        assert torch.equal(out, want)
