"""The language-model operators at the ends of their ranges (needs an MI355X):
offsets past 32 bits, launches of many workgroups, two calls at once, captured
calls that share a workspace.  Values are held against the same call on an
ordinary layout, which the operators' own tests hold against float64."""

from __future__ import annotations

import pytest
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
