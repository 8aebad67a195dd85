"""int4_linear on rows that hold an infinity or a NaN (needs an MI355X): none of such a row's
outputs is a number, wherever it stands, and every other row keeps its bits."""

from __future__ import annotations

import pytest
import test_int4_gpu as int4_test
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(20, 64, 256, 128), (5, 33, 96, 32), (70, 100, 1216, 64)], ids=str)
def test_rows_that_are_no_numbers(sidon, shape, kind, act, zeros):
    m, n, k, group = shape
    x, values, scales, zero, bias = int4_test.inputs(m, n, k, group, zeros, kind, 5)
    packed = sidon.int4.pack_int4(values, scales, zero)
    want = sidon.int4.int4_linear(x, packed, bias, act)
    bad = {0: (3, "nan"), 1: (k - 1, "inf"), 3: (k // 2, "-inf"), m - 1: (k - 30, "nan")}
    for row, (at, value) in bad.items():
        x[row, at] = float(value)
    got = sidon.int4.int4_linear(x, packed, bias, act)
    # (SiLU of minus infinity is NaN here, as by its formula)
    assert not torch.isfinite(got[list(bad)]).any()
    rest = [i for i in range(m) if i not in bad]
    assert torch.equal(got[rest], want[rest]) and torch.isfinite(got[rest]).all()
