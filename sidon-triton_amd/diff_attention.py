"""Differential attention on the HIP kernel (csrc/diff_attn.hip).

The attention of an encoder or cached decoder layer that takes the difference
of two softmax maps over one set of values, with a learned weight per head:

    o = softmax(q1 k1^T / sqrt D) v - lambda softmax(q2 k2^T / sqrt D) v
    lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init

next to ``flexrel.flexrel_attention``: strided views, device lengths, the
current stream, captured into HIP graphs like it.  No counterpart in the
reference.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .conformer import plain
from .flexrel import _check_device_tensor, _on_device, _stream_handle

HEAD_DIMS = (64, 128)


def workspace_bytes(batch: int, heads: int, kv_heads: int, length: int, keys: int, dim: int, device=None) -> int:
    """Bytes of ``diff_attention``'s workspace on ``device`` (0: none needed)."""
    _lib.ints(batch=batch, heads=heads, kv_heads=kv_heads, length=length, keys=keys, dim=dim)
    with _on_device(device):
        return int(_lib.load().sidon_diff_attention_workspace_bytes(batch, heads, kv_heads, length, keys, dim))


@functools.lru_cache(maxsize=256)
def _int64s(values: tuple) -> ctypes.Array:
    """The C array of these numbers (only ever read)."""
    return (ctypes.c_int64 * len(values))(*values)


def _strides(t: torch.Tensor) -> ctypes.Array:
    """Strides in front of the last dimension; that of a dimension of size 1
    means nothing and is given as 0."""
    st = t.stride()[:-1]
    if 1 in t.shape[:-1]:
        st = tuple([0 if n == 1 else s for n, s in zip(t.shape, st)])
    return _int64s(st)


_layouts = _lib.Layouts()


def _check(q, k, v, lam, lens, norm_w) -> tuple:
    """-> (sizes, the output's shape, workspace bytes, heads of lam, type code,
    strides of q, k and v, strides of a contiguous output) of operands that fit."""
    if q.dim() != 5 or k.dim() != 5 or v.dim() != 4:
        raise ValueError("q and k must be [B, heads, 2, length, D], v [B, heads, length, 2D]")
    batch, heads, two, length, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[3]
    if two != 2 or dim not in HEAD_DIMS:
        raise ValueError(f"q must be [B, H, 2, L, {HEAD_DIMS}] (got {tuple(q.shape)})")
    if min(q.shape) < 1 or min(k.shape) < 1:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must not be empty")
    if k.shape != (batch, kv_heads, 2, keys, dim) or v.shape != (batch, kv_heads, keys, 2 * dim):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if heads % kv_heads:
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads")
    device = q.device
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16 (got {q.dtype})")
    _check_device_tensor("q", q, device)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.device != device:
            _check_device_tensor(name, t, device)
        if t.dtype != q.dtype:
            raise TypeError(f"{name} is {t.dtype}, q is {q.dtype}")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
    if lam.device != device:
        _check_device_tensor("lam", lam, device)
    if lam.dtype != torch.float32 or not lam.is_contiguous() or lam.shape not in ((4, dim), (heads, 4, dim)):
        raise ValueError(f"lam must be a contiguous float32 [4, {dim}] or [{heads}, 4, {dim}] tensor")
    if lens is not None:
        if lens.device != device:
            _check_device_tensor("lens", lens, device)
        if lens.dtype != torch.int32 or lens.shape != (batch,) or not lens.is_contiguous():
            raise ValueError("lens must be a contiguous int32 tensor of shape [B]")
    if norm_w is not None:
        if norm_w.device != device:
            _check_device_tensor("norm_w", norm_w, device)
        if norm_w.dtype != torch.float32 or norm_w.shape != (2 * dim,) or not norm_w.is_contiguous():
            raise ValueError(f"norm_w must be a contiguous float32 [{2 * dim}] tensor")
    sizes, shape = (batch, heads, kv_heads, length, keys, dim), (batch, heads, length, 2 * dim)
    o_strides = _strides(torch.empty(shape, device="meta"))
    return (sizes, shape, workspace_bytes(*sizes, device), 1 if lam.dim() == 2 else heads, _lib.DTYPES[q.dtype],
            (_strides(q), _strides(k), _strides(v)), o_strides)


def diff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, lam_init: float,
                   lens: torch.Tensor | None = None, causal: bool = False, norm_w: torch.Tensor | None = None,
                   eps: float = 1e-5, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """q [B, H, 2, L, D], k [B, Hk, 2, S, D], v [B, Hk, S, 2D] fp16 or bf16 ->
    [B, H, L, 2D] of their type.

    Any strides that are multiples of 8 elements with the last dimension
    contiguous (views of fused projections or of a cache), D 64 or 128.  H / Hk
    neighbouring heads share a key head.  lam fp32 [4, D] (lq1, lk1, lq2, lk2) or
    [H, 4, D].  lens: int32 [B] valid keys on the device (None: all S); what lies
    past them is not read.  causal: the L queries are the last L of an item's
    valid positions, query i sees the keys up to its own.  A query without keys
    gives zeros.  norm_w fp32 [2D]: each head's output is divided by its root
    mean square (with eps > 0 under the root) and multiplied by (1 - lam_init)
    norm_w; None: left as it is.  out: optional [B, H, L, 2D], in memory apart from
    the inputs.  workspace: a contiguous uint8 tensor of ``workspace_bytes``, apart
    from all of them; allocated per call when None.  A single query against a long
    cache splits the keys over the chip.  Valid keys and values must be finite, also
    those that causal hides from some queries.  Probabilities are rounded to the
    inputs' type in front of v, but with H / Hk * L <= 32 (single tokens), where the
    output's rounding is the only one; with more that depends on all sizes.  Forward
    only."""
    key = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype,
           v.device, lam.shape, lam.stride(), lam.dtype, lam.device,
           None if lens is None else (lens.shape, lens.stride(), lens.dtype, lens.device),
           None if norm_w is None else (norm_w.shape, norm_w.stride(), norm_w.dtype, norm_w.device))
    sizes, shape, need, lam_heads, dtype, strides, o_strides = (
        _layouts.get(key) or _layouts.keep(key, _check(q, k, v, lam, lens, norm_w)))
    device = q.device
    if not (plain(q, k, v, lam) if norm_w is None else plain(q, k, v, lam, norm_w)):
        raise ValueError("diff_attention has no backward: call it under torch.no_grad()")
    if out is None:
        out = torch.empty(shape, device=device, dtype=q.dtype)
    else:
        _check_device_tensor("out", out, device)
        if out.dtype != q.dtype or tuple(out.shape) != shape or out.stride(-1) != 1:
            raise ValueError(f"out must be a {q.dtype} {shape} tensor with a contiguous last dimension")
        o_strides = _strides(out)
    lib = _lib.load()
    with _on_device(device):
        if workspace is None:
            workspace = torch.empty(need, device=device, dtype=torch.uint8) if need else None
        else:
            _check_device_tensor("workspace", workspace, device)
            if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
                raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes")
        rc = lib.sidon_diff_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), lam_heads, lam_init,
            None if lens is None else lens.data_ptr(), None if norm_w is None else norm_w.data_ptr(), eps,
            out.data_ptr(), None if workspace is None else workspace.data_ptr(),
            0 if workspace is None else workspace.numel(), *sizes, 1 if causal else 0, dtype, *strides, o_strides,
            _stream_handle(device))
    if rc:
        _lib.check("sidon_diff_attention", rc)
    return out
