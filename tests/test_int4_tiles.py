"""How int4_linear's rule cuts a call, and that shapes are found for each of its forms
(no GPU; without one the library assumes 256 compute units)."""

from __future__ import annotations

import ctypes

import pytest

# (tiles of 16 rows, of 16 outputs, wavefronts that share K): all that the rule returns
FORMS = [(rows, outputs, splits) for rows in (1, 2, 4) for outputs, splits in ((1, 8), (2, 8), (4, 8), (4, 4))]
ROWS = {1: 7, 2: 20, 4: 50}


def tiles(sidon, m, n):
    found = [ctypes.c_int() for _ in range(3)]
    rc = sidon._lib.load().sidon_int4_linear_tiles(m, n, *map(ctypes.byref, found))
    return tuple(t.value for t in found) if rc == 0 else rc


def outputs_of(sidon, form):
    """The most outputs below a power of two, or so, that are cut so, an odd number."""
    return next((n - 5 for n in (1 << 15, 20000, 1 << 14, 1 << 13, 4096, 1000) if tiles(sidon, ROWS[form[0]], n - 5) == form), None)


def test_every_form_is_reached(sidon):
    for form in FORMS:
        assert outputs_of(sidon, form) is not None, form
    seen = {tiles(sidon, m, n) for m in (1, 16, 17, 32, 33, 64, 65, 300, 5000) for n in (1, 16, 1000, 4095, 5000, 8200, 12001, 16300, 40000)}
    assert seen == set(FORMS)   # (a form that the rule may return and nothing here names)


@pytest.mark.parametrize("sizes,code", [((0, 1), -2), ((1, 0), -2), (((1 << 21) + 1, 1), -2), ((1, (1 << 24) + 1), -2)])
def test_refusals(sidon, sizes, code):
    assert tiles(sidon, *sizes) == code
    assert sidon._lib.load().sidon_int4_linear_tiles(1, 1, None, None, None) == -1
