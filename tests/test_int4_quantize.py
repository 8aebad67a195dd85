"""quantize_int4 for weights of any type, as pack_int4 takes them (no GPU)."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("of", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_weights_of_any_type_are_packed(sidon, of, kind, zeros):
    """Within half a step of the rounded scale, but at the ends of a group's range: 15 steps (7 without
    zero points) of a scale that lost half a step of its type leave 15 u of a step there at most."""
    gen = torch.Generator().manual_seed(2)
    w = (0.1 * torch.randn(40, 256, generator=gen)).to(of)
    values, scales, zero = sidon.int4.quantize_int4(w, 64, zeros, dtype=kind)
    assert scales.dtype == kind and values.dtype == torch.uint8 and int(values.max()) <= 15
    packed = sidon.int4.pack_int4(values, scales, zero)
    assert packed.dtype == kind and packed.zeros is zeros
    z = zero.float().unsqueeze(-1) if zeros else 8
    back = (values.float().unflatten(1, (4, 64)) - z) * scales.float().unsqueeze(-1)
    off = ((back - w.float().unflatten(1, (4, 64))).abs() / scales.float().unsqueeze(-1))
    # (a zero point is rounded as well, which the other end of the range pays for)
    assert (off <= (1.0 if zeros else 0.5) + 15 * torch.finfo(kind).eps / 2 + 2.0 ** -10).all()
    if of == kind:
        for a, b in zip(sidon.int4.quantize_int4(w, 64, zeros), (values, scales, zero)):
            assert a is b is None or torch.equal(a, b)


def test_scales_keep_the_weights_type(sidon):
    w = torch.randn(4, 128)
    assert sidon.int4.quantize_int4(w)[1].dtype == torch.float32
    with pytest.raises(TypeError, match="dtype"):
        sidon.int4.pack_int4(*sidon.int4.quantize_int4(w))
    with pytest.raises(TypeError, match="floating point"):
        sidon.int4.quantize_int4(w, dtype=torch.int8)
    with pytest.raises(TypeError, match="floating point"):
        sidon.int4.quantize_int4(w.to(torch.int8))
