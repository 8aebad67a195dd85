"""The language-model operators' refusals, before any launch (no GPU)."""

from __future__ import annotations

import pytest
import torch


def _norm(lib, **over):
    a = dict(x=1 << 20, ldx=64, lens=None, w=16, b=16, eps=1e-5, y=1 << 22, ldy=64, ws=16, wsb=1 << 20, B=2, T=10, C=64,
             G=4, dtype=1, act=1)
    a.update(over)
    return lib.sidon_group_norm_act(a["x"], a["ldx"], a["lens"], a["w"], a["b"], a["eps"], a["y"], a["ldy"], a["ws"],
                                    a["wsb"], a["B"], a["T"], a["C"], a["G"], a["dtype"], a["act"], None)


@pytest.mark.parametrize("over,code", [
    (dict(x=None), -1), (dict(w=None), -1), (dict(b=None), -1), (dict(y=None), -1), (dict(ws=None), -1),
    (dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(act=4), -2), (dict(B=0), -2), (dict(T=0), -2), (dict(C=0), -2),
    (dict(G=0), -2), (dict(G=5), -2), (dict(C=8256, ldx=8256, ldy=8256, G=1), -2), (dict(B=65536), -2),
    (dict(wsb=0), -2), (dict(ldx=63), -3), (dict(ldy=0), -3), (dict(ldx=-64), -3), (dict(x=(1 << 20) + 1), -4),
    (dict(w=18), -4), (dict(lens=6), -4), (dict(ws=20), -4),
    (dict(y=(1 << 20) + 128), -2), (dict(y=1 << 20, ldy=128), -2),
])
def test_group_norm_refuses(sidon, over, code):
    # fake addresses, never dereferenced: validation returns before any HIP call
    lib = sidon._lib.load()
    assert _norm(lib, **over) == code
    assert lib.sidon_last_error().decode()


def test_group_norm_workspace(sidon):
    ws = sidon.conformer.group_norm_workspace
    assert ws(0, 10, 64, 4, torch.float16) == 0 and ws(1, 10, 64, 5, torch.float16) == 0
    for shape in ((1, 1, 8, 1), (3, 1463, 1024, 16), (65535, 2, 64, 64)):
        assert 0 < ws(*shape, torch.float32) <= 8 * shape[0] * shape[3] * min(128, shape[1])


def test_group_norm_rejects_host_tensors(sidon):
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="HIP device"):
        sidon.conformer.group_norm_act(x, 1, 2, torch.ones(8), torch.zeros(8))
