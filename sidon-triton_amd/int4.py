"""Projections with 4-bit weights and group scales on the HIP kernel
(csrc/int4_linear.hip).

The projections of a decoder that takes a token at a time read every weight for
each of a few rows; 4 bits a weight are a quarter of the bytes:

    y = act(bias + sum_g s[n, g] sum_{k in g} x[k] (w[n, k] - z[n, g]))

``pack_int4`` lays weights out once, when they are loaded; ``int4_linear`` is
``conformer.linear`` / ``conformer.linear_silu`` on them.  No counterpart in the
reference.
"""

from __future__ import annotations

import dataclasses

import torch

from . import _lib
from .conformer import plain, written
from .flexrel import _check_device_tensor, _on_device, _stream_handle

_TILE_N, _TILE_K = 16, 128


@dataclasses.dataclass(frozen=True)
class Int4Weight:
    """Weights [n, k] as the kernel reads them (``pack_int4``)."""

    words: torch.Tensor    # int32 [n / 16, k / 128, 64, 4]
    scales: torch.Tensor   # int32 [n / 16, k / 128, 128 / group, 16]
    n: int
    k: int
    group: int             # 32, 64 or 128 (larger groups are 128 with equal scales)
    dtype: torch.dtype
    zeros: bool

    def __post_init__(self):
        """The kernel reads as far as n, k and group say."""
        if self.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"weights are for float16 or bfloat16 (got {self.dtype})")
        if self.group not in (32, 64, 128) or min(self.n, self.k) < 1 or self.k % self.group:
            raise ValueError(f"weights [{self.n}, {self.k}] in groups of {self.group}: need 32, 64 or 128 that divide k")
        tiles, blocks = -(-self.n // _TILE_N), -(-self.k // _TILE_K)
        for name, t, shape in (("words", self.words, (tiles, blocks, 64, 4)),
                               ("scales", self.scales, (tiles, blocks, _TILE_K // self.group, 16))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 {shape} tensor (got {t.dtype} {tuple(t.shape)})")

    def to(self, device) -> "Int4Weight":
        return dataclasses.replace(self, words=self.words.to(device), scales=self.scales.to(device))


def quantize_int4(w: torch.Tensor, group: int = 128, zeros: bool = True, dtype: torch.dtype | None = None):
    """w [N, K] -> (values uint8 [N, K] from 0 to 15, scales [N, K / group] of ``dtype``
    (None: w's), zero points uint8 [N, K / group] or None): each group's range in 15 steps
    of the scale as it is rounded, to the nearest.  Without zero points the values are 8 + w / scale.
    ``pack_int4`` takes fp16 and bf16 scales: name one of them for weights of another type."""
    dtype = w.dtype if dtype is None else dtype
    if not dtype.is_floating_point:
        raise TypeError(f"scales must be of a floating point type (got {dtype})")
    if w.dim() != 2 or group < 1 or w.shape[1] % group:
        raise ValueError(f"w must be [N, K] with K a multiple of {group}")
    g = w.detach().float().unflatten(1, (-1, group))
    if zeros:
        low, high = g.amin(-1).clamp_max(0), g.amax(-1).clamp_min(0)
        scale = ((high - low) / 15).to(dtype)
    else:
        scale = (g.abs().amax(-1) / 7).to(dtype)
    # (a group of zeros, or one whose steps the type does not hold: any scale)
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    step = scale.float()
    zero = torch.round(-low / step).clamp(0, 15) if zeros else torch.full_like(step, 8)
    values = (torch.round(g / step.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15)
    return values.to(torch.uint8).flatten(1), scale, zero.to(torch.uint8) if zeros else None


def pack_int4(values: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None) -> Int4Weight:
    """values uint8 [N, K] from 0 to 15, scales fp16 or bf16 [N, K / group], zeros
    uint8 [N, K / group] from 0 to 15 (None: 8) -> the weights as ``int4_linear``
    takes them, on the values' device.  group 32, 64 or a multiple of 128; x and the
    result of ``int4_linear`` have the scales' type."""
    if values.dim() != 2 or scales.dim() != 2 or min(*values.shape, *scales.shape) < 1:
        raise ValueError("values must be [N, K], scales [N, K / group]")
    if values.dtype != torch.uint8:
        raise TypeError(f"values must be uint8 (got {values.dtype})")
    if scales.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"scales must be float16 or bfloat16 (got {scales.dtype}; quantize_int4's dtype)")
    scales = scales.detach()
    n, k = values.shape
    groups = scales.shape[1]
    if scales.shape[0] != n or k % groups:
        raise ValueError(f"values are {tuple(values.shape)}, scales {tuple(scales.shape)}")
    group = k // groups
    if group not in (32, 64) and group % 128:
        raise ValueError(f"groups of {group} inputs: need 32, 64 or a multiple of 128")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"zeros must be a uint8 {tuple(scales.shape)} tensor")
    if int(values.max() if zeros is None else torch.maximum(values.max(), zeros.max())) > 15:
        raise ValueError("values and zeros must be from 0 to 15")
    if group > 128:
        scales = scales.repeat_interleave(group // 128, 1)
        zeros = None if zeros is None else zeros.repeat_interleave(group // 128, 1)
        group = 128
    tiles, blocks, per = -(-n // _TILE_N), -(-k // _TILE_K), _TILE_K // group
    if n % _TILE_N or k % _TILE_K:
        def padded(t, width):
            full = t.new_zeros(tiles * _TILE_N, width)
            full[:n, :t.shape[1]] = t
            return full

        values, scales = padded(values, blocks * _TILE_K), padded(scales, blocks * per)
        zeros = None if zeros is None else padded(zeros, blocks * per)
    # input 4 a + 2 p + s of a word's eight goes to byte 2 s + a, nibble p
    nib = values.unflatten(1, (-1, 2, 2, 2))
    words = values.new_empty(*nib.shape[:2], 2, 2)
    torch.add(nib[..., 0, :], nib[..., 1, :], alpha=16, out=words.transpose(-1, -2))
    # [tile, row, block, step, lane quarter] -> [tile, block, quarter, row, step] of words
    words = words.flatten(2).view(torch.int32).view(tiles, _TILE_N, blocks, 4, 4).permute(0, 2, 4, 1, 3).contiguous()
    # the scale, and above it what goes off the operand that a value becomes: fp16 v - 8, bf16 128 + v
    less = -8.0 if scales.dtype == torch.float16 else 128.0
    pair = scales.new_empty(tiles, blocks, per, _TILE_N, 2)
    placed = lambda t: t.unflatten(1, (blocks, per)).unflatten(0, (tiles, _TILE_N)).permute(0, 2, 3, 1)  # noqa: E731
    pair[..., 0] = placed(scales)
    if zeros is None:
        pair[..., 1] = 8 + less
    else:
        torch.add(placed(zeros), less, out=pair[..., 1])
    both = pair.view(torch.int32).squeeze(-1)
    return Int4Weight(words.view(tiles, blocks, 64, 4), both, n, k, group, scales.dtype, zeros is not None)


def int4_linear(x: torch.Tensor, w: Int4Weight, bias: torch.Tensor | None = None, act: str | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x . w^T + bias) [M, N] for x [M, K] of the scales' type, K contiguous, rows
    whole 16 bytes apart; bias [N] of the same type or None; act None or "silu"; out:
    optional [M, N] of that type with rows contiguous, apart from the operands.

    For few rows: each block of up to 64 reads all the weights.  Sums and scales in
    fp32, one rounding at the end.  Forward only."""
    if not isinstance(x, torch.Tensor) or not isinstance(w, Int4Weight):
        raise TypeError("x must be a torch.Tensor, w an Int4Weight (pack_int4)")
    device = x.device
    _check_device_tensor("x", x, device)
    if x.dtype != w.dtype or x.dim() != 2 or x.shape[1] != w.k or x.shape[0] < 1 or x.stride(1) != 1:
        raise ValueError(f"x must be a {w.dtype} [rows, {w.k}] tensor with K contiguous (got {x.dtype} {tuple(x.shape)})")
    if act not in (None, "silu"):
        raise ValueError(f"act must be None or 'silu' (got {act!r})")
    for name, t in (("words", w.words), ("scales", w.scales)):
        if t.device != device:
            _check_device_tensor(name, t, device)
    if bias is not None:
        _check_device_tensor("bias", bias, device)
        if bias.dtype != w.dtype or tuple(bias.shape) != (w.n,) or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous {w.dtype} [{w.n}] tensor")
    rows, given = x.shape[0], out
    if out is None:
        out = x.new_empty((rows, w.n))
    else:
        _check_device_tensor("out", out, device)
        if out.dtype != w.dtype or tuple(out.shape) != (rows, w.n) or (out.stride(1) != 1 and w.n > 1):
            raise ValueError(f"out must be a {w.dtype} [{rows}, {w.n}] tensor with rows contiguous")
    if not plain(*[t for t in (x, bias, given) if t is not None]):
        raise ValueError("int4_linear has no backward: call it under torch.no_grad()")
    _lib.ints(rows=rows)
    lib = _lib.load()
    with _on_device(device):
        # (a single row's stride means nothing)
        rc = lib.sidon_int4_linear(x.data_ptr(), x.stride(0) if rows > 1 else (w.k + 7) // 8 * 8, w.words.data_ptr(),
                                   w.scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(),
                                   out.stride(0) if rows > 1 else w.n, rows, w.n, w.k, w.group, 1 if w.zeros else 0,
                                   _lib.ACTIVATIONS[act], _lib.DTYPES[w.dtype], _stream_handle(device))
    if rc:
        _lib.check("sidon_int4_linear", rc)
    written(given)
    return out
