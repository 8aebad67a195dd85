"""The oracle's bounds for sharp softmaxes (no GPU): the same gradients as its other form's, and bounds that hold
for delta in 64 bits with everything else rounded, but not for delta from a rounded output."""

from __future__ import annotations

import pytest
import torch

from oracle import decoder_oracle as oracle


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
def test_bounds_of_sharp_softmaxes(kind):
    gen, u, scale = torch.Generator().manual_seed(4), torch.finfo(kind).eps / 2, 0.125
    randn = lambda *s, size=1: (size * torch.randn(*s, generator=gen)).to(kind)  # noqa: E731
    q, k, v, dout = randn(2, 4, 60, 64, size=8), randn(2, 2, 90, 64), randn(2, 2, 90, 64), randn(2, 4, 60, 64)
    lens, q_lens = [90, 40], [60, 51]
    want = oracle.sharp_cross_grads(dout, q, k, v, lens, q_lens, scale, u)
    for (value, _), (other, _) in zip(want.values(), oracle.cross_grads(dout, q, k, v, lens, q_lens, scale, u).values()):
        torch.testing.assert_close(value, other)
    rounded = lambda t: t.to(kind).double()  # noqa: E731
    worst = {}
    for j in range(4):
        qq, do, kk, vv = (t.double() for t in (q[0, j], dout[0, j], k[0, j // 2], v[0, j // 2]))
        p = torch.softmax(scale * (qq @ kk.t()), -1)
        dp = do @ vv.t()
        for name, delta in (("exact", (p * dp).sum(-1, keepdim=True)), ("rounded", (do * rounded(p @ vv)).sum(-1, keepdim=True))):
            up = 2.0 ** 15 / (4 * do.norm(dim=-1, keepdim=True) * vv.norm(dim=-1).max()).log2().ceil().exp2()   # (fp16's range)
            dq = rounded(scale * ((rounded(p * (dp - delta) * up) / up) @ kk))
            value, tol = (t[0, j] for t in want["dq"])
            worst[name] = max(worst.get(name, 0), float(((dq - value).abs() / (tol + 2.0 ** -24)).max()))
    assert worst["exact"] <= 1 < 5 < worst["rounded"]
