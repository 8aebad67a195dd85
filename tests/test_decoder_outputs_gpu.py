"""What autograd has to know of the decoder operators' outputs (needs an MI355X): one that
needs a gradient is refused, as torch refuses ``out=`` there, and one that a graph has
saved counts as changed, as after torch's own in-place calls."""

from __future__ import annotations

import pytest
import test_cross_attention_gpu as cross_test
import test_head_norm_gpu as norm_test
import test_int4_gpu as int4_test
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def calls(sidon):
    """-> {name: (call, shape and type of the output)}; call(tensor) writes that output."""
    ca, hn = sidon.cross_attention, sidon.head_norm
    q, k, v, dout = cross_test.inputs(1, 2, 1, 4, 9, 64, torch.float16, 1)
    lse = torch.empty(1, 2, 4, device=DEV)
    out = ca.cross_attention(q, k, v, lse=lse)
    x, values, scales, zero, bias = int4_test.inputs(2, 48, 96, 32, True, torch.float16, 3)
    packed = sidon.int4.pack_int4(values, scales, zero)
    nq, nk, qw, kw, cos, sin, pos = norm_test.inputs(2, 5, 4, 2, 64, 32, torch.float16, 8)
    turn = (qw, kw, cos, sin, pos, pos)
    back = (dout, q, k, v, out, lse)
    return {
        "out": (lambda t: ca.cross_attention(q, k, v, out=t), q), "lse": (lambda t: ca.cross_attention(q, k, v, lse=t), lse),
        "dq": (lambda t: ca.cross_attention_backward(*back, dq=t), q), "dk": (lambda t: ca.cross_attention_backward(*back, dk=t), k),
        "dv": (lambda t: ca.cross_attention_backward(*back, dv=t), v),
        "out_q": (lambda t: hn.qk_norm_rotary(nq, nk, *turn, out_q=t), nq), "out_k": (lambda t: hn.qk_norm_rotary(nq, nk, *turn, out_k=t), nk),
        "norm dq": (lambda t: hn.qk_norm_rotary_backward(nq, nk, nq, nk, *turn, dq=t), nq),
        "norm dk": (lambda t: hn.qk_norm_rotary_backward(nq, nk, nq, nk, *turn, dk=t), nk),
        "y": (lambda t: sidon.int4.int4_linear(x, packed, bias, out=t), x.new_empty(2, 48)),
    }


NAMES = ["out", "lse", "dq", "dk", "dv", "out_q", "out_k", "norm dq", "norm dk", "y"]


@pytest.mark.parametrize("name", NAMES)
def test_outputs_that_need_a_gradient_are_refused(sidon, name):
    call, like = calls(sidon)[name]
    leaf = torch.full(like.shape, 5.0, dtype=like.dtype, device=DEV, requires_grad=True)
    for t in (leaf, leaf * 1):
        with pytest.raises(ValueError, match="no_grad"):
            call(t)
        assert (t == 5).all()
    with torch.no_grad():
        call(leaf)
        assert not (leaf == 5).any()
        with torch.inference_mode():
            call(torch.zeros(like.shape, dtype=like.dtype, device=DEV))


@pytest.mark.parametrize("name", NAMES)
def test_a_saved_output_counts_as_changed(sidon, name):
    call, like = calls(sidon)[name]
    saved = torch.ones(like.shape, dtype=like.dtype, device=DEV)
    leaf = torch.ones(like.shape, device=DEV, requires_grad=True)
    y = (leaf * saved).sum()
    before = saved._version
    call(saved)
    assert saved._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_norm_in_place_counts_as_a_change(sidon):
    """Of the tensor that the heads are a view of, too; what is only read does not count."""
    q, k, qw, kw, cos, sin, pos = norm_test.inputs(2, 5, 4, 2, 64, 32, torch.float16, 8)
    rows, weights = q._base, qw._version
    before, leaf = rows._version, torch.ones(rows.shape, device=DEV, requires_grad=True)
    y = (leaf * rows).sum()
    sidon.head_norm.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos)
    assert rows._version == before
    sidon.head_norm.qk_norm_rotary(q, k, qw, kw, cos, sin, pos, pos, out_q=q)
    assert rows._version > before and qw._version == weights
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
