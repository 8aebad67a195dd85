"""The autograd function that a training program makes of cross_attention's two calls (needs
an MI355X): run by gradients of any layout, and with lengths that change too early."""

from __future__ import annotations

import pytest
import test_cross_attention_gpu as cross_test
import torch

pytestmark = pytest.mark.gpu


def attend_of(cross_attention):
    class Attend(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, lens):
            lse = q.new_empty(q.shape[:3], dtype=torch.float32)
            out = cross_attention.cross_attention(q, k, v, lens, lse=lse)
            ctx.save_for_backward(q, k, v, out, lse, lens)
            return out

        @staticmethod
        def backward(ctx, dout):
            q, k, v, out, lse, lens = ctx.saved_tensors
            return *cross_attention.cross_attention_backward(dout.contiguous(), q, k, v, out, lse, lens), None

    return Attend.apply


@pytest.mark.parametrize("kind", cross_test.KINDS, ids=str)
def test_gradients_of_any_layout(sidon, kind):
    """A sum's expanded gradient, a transposed one and a whole one, against the backward call on plain copies."""
    ca = sidon.cross_attention
    attend = attend_of(ca)
    q, k, v, _ = cross_test.inputs(2, 4, 2, 20, 70, 64, kind, 3)
    lens = cross_test.int32([70, 31])
    lse = torch.empty(2, 4, 20, device=q.device)
    out = ca.cross_attention(q, k, v, lens, lse=lse)
    for loss in (lambda y: y.sum(), lambda y: (y.transpose(-1, -2) * 2).sum(), lambda y: y.float().square().sum(),
                 lambda y: y[:, :, 3].sum()):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        y = attend(*leaves, lens)
        assert torch.equal(y, out)
        loss(y).backward()
        alone = out.clone().requires_grad_()
        loss(alone).backward()
        want = ca.cross_attention_backward(alone.grad.contiguous(), q, k, v, out, lse, lens)
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, want))


def test_lengths_that_change_before_the_gradients(sidon):
    attend = attend_of(sidon.cross_attention)
    q, k, v, _ = cross_test.inputs(2, 2, 2, 5, 40, 64, torch.float16, 3)
    lens = cross_test.int32([40, 31])
    y = attend(*(t.clone().requires_grad_() for t in (q, k, v)), lens)
    lens.copy_(cross_test.int32([3, 2]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
