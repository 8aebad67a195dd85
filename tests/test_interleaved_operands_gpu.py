"""The decoder's operators on tensors that lie in turn in one (needs an MI355X): q | k | v as
[B, 3, heads, tokens, D], gradients of k | v as [B, 2, key heads, keys, D]."""

from __future__ import annotations

import pytest
import test_cross_attention_gpu as cross_test
import test_head_norm_gpu as norm_test
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("kind", norm_test.KINDS, ids=str)
def test_norms_in_place_of_heads_first_rows(sidon, kind):
    b, h, l, d = 3, 4, 21, 64
    hn = sidon.head_norm
    rows = torch.randn(b, 3, h, l, d, generator=torch.Generator().manual_seed(3)).to(kind).to(DEV)
    _, _, qw, kw, cos, sin, pos = norm_test.inputs(b, l, h, h, d, 32, kind, 8)
    before = rows.clone()
    want = hn.qk_norm_rotary(before[:, 0], before[:, 1], qw, kw, cos, sin, pos, pos)
    hn.qk_norm_rotary(rows[:, 0], rows[:, 1], qw, kw, cos, sin, pos, pos, out_q=rows[:, 0], out_k=rows[:, 1])
    assert torch.equal(rows[:, 0], want[0]) and torch.equal(rows[:, 1], want[1]) and torch.equal(rows[:, 2], before[:, 2])
    grads = hn.qk_norm_rotary_backward(want[0], want[1], before[:, 0], before[:, 1], qw, kw, cos, sin, pos, pos)
    got = hn.qk_norm_rotary_backward(rows[:, 0], rows[:, 1], before[:, 0], before[:, 1], qw, kw, cos, sin, pos, pos, dq=rows[:, 0],
                                     dk=rows[:, 1])
    assert all(torch.equal(x, y) for x, y in zip(got, grads)) and torch.equal(rows[:, 2], before[:, 2])


@pytest.mark.parametrize("kind", cross_test.KINDS, ids=str)
def test_attention_and_gradients(sidon, kind):
    b, h, hk, l, s, d = 2, 4, 2, 40, 70, 64
    q, k, v, dout = cross_test.inputs(b, h, hk, l, s, d, kind, 5)
    ca, lens, lse = sidon.cross_attention, cross_test.int32([70, 33]), torch.empty(b, h, l, device=DEV)
    want = ca.cross_attention(q, k, v, lens, lse=lse)
    grads = ca.cross_attention_backward(dout, q, k, v, want, lse, lens)
    rows = torch.full((b, 3, h, l, d), 7.0, dtype=kind, device=DEV)   # q, out, dq
    rows[:, 0] = q
    kv = torch.full((b, 4, hk, s, d), 7.0, dtype=kind, device=DEV)   # k, v, dk, dv
    kv[:, 0], kv[:, 1] = k, v
    ca.cross_attention(rows[:, 0], kv[:, 0], kv[:, 1], lens, out=rows[:, 1], lse=lse)
    assert torch.equal(rows[:, 1], want) and (rows[:, 2] == 7).all() and torch.equal(rows[:, 0], q)
    ca.cross_attention_backward(dout, rows[:, 0], kv[:, 0], kv[:, 1], rows[:, 1], lse, lens, dq=rows[:, 2], dk=kv[:, 2], dv=kv[:, 3])
    for got, like in ((rows[:, 2], grads[0]), (kv[:, 2], grads[1]), (kv[:, 3], grads[2]), (rows[:, 0], q), (kv[:, 0], k), (kv[:, 1], v)):
        assert torch.equal(got, like)
