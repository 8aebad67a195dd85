"""qk_norm_rotary and its gradients where a team of lanes takes four heads, the last of them
not all there, and several tokens (needs an MI355X).  Tolerances: test_head_norm_gpu; a term of dw goes
through its team's rows (3 tokens of 4 heads at most here), the 128 teams of a workgroup at most,
and 16 and 64 of the workgroups' sums, under 512 additions with what formed it."""

from __future__ import annotations

import pytest
import test_head_norm_gpu as norm_test
import torch

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

CASES = [
    # (batch, tokens, heads, key heads, D, rotated): each width of a team, heads in fours and one, two or three more
    (4, 4800, 17, 5, 64, 64), (3, 1463, 15, 3, 128, 64), (2, 3000, 6, 2, 240, 16), (2, 12000, 9, 3, 16, 16), (3, 5000, 10, 1, 32, 32),
    (2, 4000, 7, 7, 48, 0), (1, 9000, 3, 1, 256, 256),
]


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("kind", norm_test.KINDS, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_four_heads_a_team(sidon, case, kind, interleaved):
    b, l, h, hk, d, rot = case
    hn = sidon.head_norm
    # rows of the workspace: workgroups, of which a chunk of four heads has as many as each other
    rows = hn.workspace_bytes(b, h, hk, l, l, d) // (4 * d)
    teams = 256 // max(2, 1 << (d // 8 - 1).bit_length())
    chunks = [-(-n // 4) for n in (h, hk)]
    turns = [-(-b * l // teams) for _ in chunks]
    each = [-(-t // (1024 // c)) for t, c in zip(turns, chunks)]
    assert rows == sum(c * -(-t // e) for c, t, e in zip(chunks, turns, each)) and max(each) <= 3
    q, k, qw, kw, cos, sin, pos = norm_test.inputs(b, l, h, hk, d, rot, kind, l + d)
    padded = (pos < 0).view(b, 1, l, 1)
    dq_out, dk_out = norm_test.grad_like(q, 1), norm_test.grad_like(k, 2)
    for t in (q, k, dq_out, dk_out):   # what padding holds is anything
        t.masked_fill_(padded, float("nan"))
    got = hn.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos, norm_test.EPS, interleaved)
    grads = hn.qk_norm_rotary_backward(dq_out, dk_out, q, k, qw, kw, cos, sin, pos, pos, norm_test.EPS, interleaved)
    for x, w, y, dy, dx, dw in ((q, qw, got[0], dq_out, grads[0], grads[2]), (k, kw, got[1], dk_out, grads[1], grads[3])):
        want, size = oracle.norm_rotary(x, w, cos, sin, pos, norm_test.EPS, interleaved)
        norm_test.close(y, want, size)
        assert (y.masked_select(padded.expand_as(y)) == 0).all()
        want, size, wsum, wsize = oracle.norm_rotary_grads(dy, x, w, cos, sin, pos, norm_test.EPS, interleaved)
        norm_test.close(dx, want, size, 64)
        norm_test.close(dw, wsum, wsize, 512)
    again = hn.qk_norm_rotary_backward(dq_out, dk_out, q, k, qw, kw, cos, sin, pos, pos, norm_test.EPS, interleaved)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))
