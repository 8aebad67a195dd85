"""Every form that int4_linear's rule can take, with tails of rows, outputs and inputs, in
each type and group (needs an MI355X).  Tolerances: test_int4_gpu."""

from __future__ import annotations

import pytest
import test_int4_gpu as int4_test
import torch
from test_int4_tiles import FORMS, ROWS, outputs_of, tiles

from oracle import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

INPUTS = {32: 1184, 64: 1216, 128: 1280}   # a quarter, half and a whole block of 128 past nine: one and more of each wavefront


@pytest.mark.parametrize("zeros", [False, True], ids=["plain", "zeros"])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_every_form(sidon, form, group, kind, zeros):
    m = ROWS[form[0]]
    n = outputs_of(sidon, form)
    assert n is not None and tiles(sidon, m, n) == form   # (by this device's compute units)
    x, values, scales, zero, bias = int4_test.inputs(m, n, INPUTS[group], group, zeros, kind, m + n)
    got = sidon.int4.int4_linear(x, sidon.int4.pack_int4(values, scales, zero), bias)
    int4_test.close(got, *oracle.int4(x, values, scales, zero, bias, None))


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(300, 3000, 640, 128), (130, 5003, 96, 32), (20, 12001, 160, 32), (64, 16384, 256, 64)], ids=str)
def test_blocks_of_rows(sidon, shape, kind):
    """Several blocks of 64 rows, and few blocks of inputs for the eight wavefronts."""
    m, n, k, group = shape
    assert tiles(sidon, m, n)[1] == 4 or torch.cuda.get_device_properties(0).multi_processor_count != 256
    x, values, scales, zero, bias = int4_test.inputs(m, n, k, group, True, kind, m + n)
    got = sidon.int4.int4_linear(x, sidon.int4.pack_int4(values, scales, zero), bias, "silu")
    int4_test.close(got, *oracle.int4(x, values, scales, zero, bias, "silu"))
