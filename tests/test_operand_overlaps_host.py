"""Which operands of the decoder's operators share memory, from their strides (no GPU): what
lies apart is taken, however interleaved, and nothing that meets is."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch
from test_decoder_operators_host import MB, _cross, _int4, _norm

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="fake addresses")

TAKEN, REFUSED, STRIDE = -6, -2, -3   # (no device here)


@pytest.mark.parametrize("over", [
    # q | k | v as [B, 3, heads, tokens, D], normed in place, and into another such tensor
    dict(q=MB, k=MB + 5120, yq=MB, yk=MB + 5120, Hk=4, S=10, qs=(7680, 640, 64), ks=(7680, 640, 64), yqs=(7680, 640, 64), yks=(7680, 640, 64)),
    # the same with tokens in front of heads, and with items innermost: [tokens, 3, B, heads, D]
    dict(q=MB, k=MB + 5120, yq=MB, yk=MB + 5120, Hk=4, S=10, qs=(7680, 64, 256), ks=(7680, 64, 256), yqs=(7680, 64, 256), yks=(7680, 64, 256)),
    dict(q=MB, k=MB + 1024, yq=MB, yk=MB + 1024, Hk=4, S=10, qs=(256, 64, 1536), ks=(256, 64, 1536), yqs=(256, 64, 1536), yks=(256, 64, 1536)),
    # heads of q and its output in turn, each head's tokens together
    dict(q=MB, yq=MB + 1280, qs=(5120, 1280, 64), yqs=(5120, 1280, 64)),
])
def test_norms_of_interleaved_tensors(sidon, over):
    lib = sidon._lib.load()
    assert _norm(lib, **over) == TAKEN, lib.sidon_last_error()


@pytest.mark.parametrize("over", [
    # dk | dv as [B, 2, key heads, keys, D], k | v so, and the queries' side beside its gradient
    dict(dk=8 * MB, dv=8 * MB + 25600, dks=(25600, 6400, 64), dvs=(25600, 6400, 64)),
    dict(k=8 * MB, v=8 * MB + 25600, dk=8 * MB + 51200, dv=8 * MB + 76800, ks=(51200, 6400, 64), vs=(51200, 6400, 64), dks=(51200, 6400, 64),
         dvs=(51200, 6400, 64)),
    dict(q=MB, dq=MB + 5120, qs=(5120, 640, 64), dqs=(5120, 640, 64)),
])
def test_gradients_of_interleaved_tensors(sidon, over):
    lib = sidon._lib.load()
    assert _cross(lib, True, **over) == TAKEN, lib.sidon_last_error()


@pytest.mark.parametrize("over", [
    dict(out=MB + 5120, qs=(5120, 640, 64), os=(5120, 640, 64)), dict(out=MB + 1280, qs=(5120, 1280, 64), os=(5120, 1280, 64)),
])
def test_outputs_beside_interleaved_queries(sidon, over):
    lib = sidon._lib.load()
    assert _cross(lib, **over) == TAKEN, lib.sidon_last_error()


def _bytes(at, n, st):
    """Addresses of a tensor's 16-byte units (D 64, 2 bytes)."""
    a = at + 2 * (np.arange(n[0]).reshape(-1, 1, 1) * st[0] + np.arange(n[1]).reshape(-1, 1) * st[1] + np.arange(n[2]) * st[2]).reshape(-1, 1)
    return set((a + 16 * np.arange(8)).reshape(-1).tolist())


def test_nothing_that_meets_is_taken(sidon):
    """Queries and an output at random places and strides, against the sets of their addresses."""
    lib, rng = sidon._lib.load(), random.Random(5)
    seen = {True: 0, False: 0}
    for _ in range(6000):
        b, h, l = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 4)
        order, step, st = rng.sample(range(3), 3), 64, [0, 0, 0]
        for d in order:   # a dense layout of two tensors in turn at some level, then shifted strides
            st[d] = step * rng.choice([1, 1, 2, 2]) + 8 * rng.choice([0, 0, 0, 1, 4])
            step = st[d] * (b, h, l)[d]
        other = list(st) if rng.random() < 0.6 else [s + 8 * rng.choice([0, 0, 8, 16]) for s in st]
        if rng.random() < 0.2:
            st[rng.randrange(3)] = 0   # (expanded queries)
        at = MB + 16 * rng.randint(0, 2 * max(1, step) // 8)
        rc = _cross(lib, q=MB, out=at, qs=st, os=other, B=b, H=h, Hk=1, L=l, k=32 * MB, v=48 * MB, lse=None, lens=None, q_lens=None, ws=64 * MB,
                    ks=(25600, 64, 256), vs=(25600, 64, 256))
        if rc == STRIDE:
            continue
        meet = bool(_bytes(MB, (b, h, l), st) & _bytes(at, (b, h, l), other))
        assert rc in (TAKEN, REFUSED) and not (meet and rc == TAKEN), (b, h, l, st, other, at - MB)
        seen[rc == TAKEN] += 1
    assert min(seen.values()) > 300, seen


def test_int4_beside_its_inputs(sidon):
    lib = sidon._lib.load()
    assert _int4(lib, ldx=512, y=MB + 512, ldy=1024) == TAKEN   # y in every other gap between x's rows
    assert _int4(lib, ldx=512, y=MB + 512, ldy=256) == REFUSED   # (its second row is x's)
    assert _int4(lib, ldx=512, y=MB + 500, ldy=1024) == REFUSED
