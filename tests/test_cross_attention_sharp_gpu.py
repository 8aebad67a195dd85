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
