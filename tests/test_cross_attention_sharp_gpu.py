"""cross_attention's gradients where a query's softmax is nearly one key, as over speech
(needs an MI355X): dS is then what the other keys leave of dP - delta, far below
either, and delta has to be right to much less than the 16-bit output is.  Bounds:
decoder_oracle.sharp_cross_grads."""

from __future__ import annotations

import pytest
import test_cross_attention_gpu as cross_test
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("kind", cross_test.KINDS, ids=str)
@pytest.mark.parametrize("size", [1, 3, 8, 20])
@pytest.mark.parametrize("shape", [(2, 4, 2, 150, 300, 64), (3, 6, 2, 40, 129, 128), (1, 3, 1, 33, 20, 64), (2, 2, 2, 1, 77, 64),
                                   (1, 2, 1, 300, 1463, 64), (1, 1, 1, 70, 2049, 128), (8, 16, 16, 130, 200, 64)], ids=str)
def test_sharp_gradients(sidon, shape, size, kind):
    """Scores of a standard deviation of 1 to 20: the largest probability is 0.03 to 0.97 on average."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = cross_test.inputs(*shape, kind, l + s + size)
    q = (q * size).contiguous()
    lens, q_lens = [s, s - 3, s // 2, 0, 1, s, 33, s][:b], [l, max(l - 7, 1), l, l, 1, 0, l, l][:b]
    cross_test.poison(lens, q_lens, q, k, v, dout)
    ca, n, m = sidon.cross_attention, cross_test.int32(lens), cross_test.int32(q_lens)
    lse = torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, n, m, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse, n, m)
    want = oracle.sharp_cross_grads(dout, q, k, v, lens, q_lens, d ** -0.5, torch.finfo(kind).eps / 2)
    for got, (value, tol) in zip(grads, want.values()):
        cross_test.within(got, value, tol + cross_test.tiny(kind))
    again = ca.cross_attention_backward(dout, q, k, v, out, lse, n, m)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("less", [2.0 ** -6, 2.0 ** -12, 2.0 ** -20], ids=str)
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 300, 64), (1, 2, 1, 40, 96, 128), (1, 4, 4, 160, 500, 64)], ids=str)
def test_fp16_rows_far_apart_in_size(sidon, shape, less):
    """Rows of dout a million times shorter than others', and keys that only such rows see: what
    fp16's power of two leaves of them (one for all rows of a key in dk, one for a row in dq)."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = cross_test.inputs(*shape, torch.float16, 23)
    q, dout = q.contiguous(), (64 * dout).contiguous()
    dout[:, :, ::2] *= less
    # even queries see the first half of the keys, odd ones the rest
    q[..., 0], k[..., 0] = 0, 0
    q[:, :, ::2, 0], q[:, :, 1::2, 0] = 16, -16
    k[:, :, :s // 2, 0], k[:, :, s // 2:, 0] = 8, -8
    ca, lse = sidon.cross_attention, torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse)
    want = oracle.sharp_cross_grads(dout, q, k, v, None, None, d ** -0.5, 2.0 ** -11)
    for got, (value, tol) in zip(grads, want.values()):
        cross_test.within(got, value, tol + cross_test.tiny(torch.float16))


@pytest.mark.parametrize("kind", cross_test.KINDS, ids=str)
@pytest.mark.parametrize("size", [32, 512])
def test_gradients_of_large_scores(sidon, size, kind):
    """Scores of a standard deviation of ``size``, within the bounds of their fp32 values."""
    b, h, hk, l, s, d = 2, 2, 1, 40, 90, 64
    q, k, v, dout = cross_test.inputs(b, h, hk, l, s, d, kind, 29)
    q = (q * size).contiguous()
    ca, lse = sidon.cross_attention, torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    assert float(lse.max()) > 2 * size
    grads = ca.cross_attention_backward(dout, q, k, v, out, lse)
    want = oracle.sharp_cross_grads(dout, q, k, v, None, None, d ** -0.5, torch.finfo(kind).eps / 2)
    for got, (value, tol) in zip(grads, want.values()):
        cross_test.within(got, value, tol + cross_test.tiny(kind))


@pytest.mark.parametrize("kind", cross_test.KINDS, ids=str)
@pytest.mark.parametrize("shape", [(2, 2, 1, 40, 90, 64), (1, 2, 2, 33, 70, 128)], ids=str)
def test_gradients_of_the_largest_scores(sidon, shape, kind):
    """Scores of up to some 2^20, whose fp32 values are right to 2^-4: numbers, if no more than that."""
    b, h, hk, l, s, d = shape
    q, k, v, dout = cross_test.inputs(*shape, kind, 31)
    q, k = (8192 * q).contiguous(), (16 * k).contiguous()
    ca, lse = sidon.cross_attention, torch.empty(b, h, l, device=DEV)
    out = ca.cross_attention(q, k, v, scale=0.25, lse=lse)
    assert 2.0 ** 21 > float(lse.max()) > 2.0 ** 19   # (standard deviations of 2^18 and 2^18.5)
    assert all(torch.isfinite(t).all() for t in (out, *ca.cross_attention_backward(dout, q, k, v, out, lse, scale=0.25)))
