"""Shared projections with a low-rank adapter per request (csrc/adapters.hip).

The reference merges one adapter into the weights before serving
(W + 0.25 A B, tools/convert_torchscript.py:179-205), so a batch cannot mix fine-tuned
variants.  Here the shared weights stay as they are and every item of a batch
names its adapter:

    y[m] = act(x[m] W^T + bias + scale_e (x[m] A_e^T) B_e^T),   e = ids[item of row m]

next to ``conformer.linear`` / ``conformer.linear_silu_lt`` (``adapter_linear``)
and ``conformer.residual_gemm`` (``adapter_residual``).  ``encoder.HipEncoder``
takes packed adapters for its projections.  All launch on the current stream and
allocate only the output and the workspace (neither when given).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .conformer import _row_stride, plain
from .flexrel import _check_device_tensor, _on_device, _stream_handle

MAX_RANK = 128
_TYPES = (torch.float16, torch.bfloat16)


def workspace_bytes(rows: int, rank: int, residual: bool = False, dtype: torch.dtype = torch.float16) -> int:
    """Bytes of the workspace of a call on ``rows`` rows (all items together)."""
    _lib.ints(rows=rows, rank=rank)
    return int(_lib.load().sidon_adapter_workspace_bytes(rows, rank, int(residual), _lib.DTYPES[dtype]))


def pack_adapters(pairs, scales, device=None, dtype: torch.dtype = torch.float16):
    """[(A [r, K], B [N, r]), ...] of any ranks up to 128 and their scales ->
    (a [E, R, K], b [E, N, R], scale [E]) for the calls below, R the largest rank
    rounded up to 8 and the rest zeros."""
    pairs, scales = list(pairs), [float(s) for s in scales]
    if not pairs or len(pairs) != len(scales):
        raise ValueError("pack_adapters needs one scale per (A, B) pair, and one pair at least")
    for a, b in pairs:
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or not 1 <= a.shape[0] <= MAX_RANK \
                or a.shape[1] != pairs[0][0].shape[1] or b.shape[0] != pairs[0][1].shape[0]:
            raise ValueError(f"every pair must be A [r <= {MAX_RANK}, K] and B [N, r] of one K and N "
                             f"(got {tuple(a.shape)} and {tuple(b.shape)})")
    rank = -(-max(a.shape[0] for a, _ in pairs) // 8) * 8
    device = pairs[0][0].device if device is None else device
    a_all = torch.zeros(len(pairs), rank, pairs[0][0].shape[1], dtype=dtype, device=device)
    b_all = torch.zeros(len(pairs), pairs[0][1].shape[0], rank, dtype=dtype, device=device)
    for e, (a, b) in enumerate(pairs):
        a_all[e, :a.shape[0]] = a.detach().to(device=device, dtype=dtype)
        b_all[e, :, :b.shape[1]] = b.detach().to(device=device, dtype=dtype)
    return a_all, b_all, torch.tensor(scales, dtype=torch.float32, device=device)


def stack_adapters(pairs):
    """The adapters of projections that are fused along their outputs (q, k and v
    as one): [(A_i [r_i, K], B_i [N_i, r_i]), ...] -> one pair of the fused
    projection, A stacked and B block-diagonal.  Scales that differ belong into
    the B_i."""
    pairs = list(pairs)
    if not pairs:
        raise ValueError("stack_adapters needs at least one pair")
    return torch.cat([a for a, _ in pairs]), torch.block_diag(*[b for _, b in pairs])


_layouts = _lib.Layouts()


def _operands(x, w, a, b, scale, ids, bias, residual: bool) -> tuple:
    """-> (rows, n, strides of x and w, the sizes behind them in a call, type code,
    workspace bytes) of operands that fit."""
    key = (x.shape, x.stride(), x.dtype, x.device, w.shape, w.stride(), w.dtype, w.device, a.shape, a.stride(), a.dtype,
           a.device, b.shape, b.stride(), b.dtype, b.device, scale.shape, scale.stride(), scale.dtype, scale.device,
           ids.shape, ids.stride(), ids.dtype, ids.device,
           None if bias is None else (bias.shape, bias.stride(), bias.dtype, bias.device), residual)
    return _layouts.get(key) or _layouts.keep(key, _check(x, w, a, b, scale, ids, bias, residual))


def _check(x, w, a, b, scale, ids, bias, residual):
    device = x.device
    _check_device_tensor("x", x, device)
    for name, t in (("x", x), ("w", w), ("a", a), ("b", b)):
        if t.device != device:
            _check_device_tensor(name, t, device)
        if t.dtype not in _TYPES or t.dtype != x.dtype:
            raise TypeError(f"{name} must be float16 or bfloat16, of x's type (got {t.dtype})")
    if x.dim() != 2 or x.stride(1) != 1 or w.dim() != 2 or w.stride(1) != 1:
        raise ValueError("x and w must be [rows, K] tensors with K contiguous")
    rows, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"x has {k} columns, w {w.shape[1]}")
    if a.dim() != 3 or a.shape[2] != k or not a.is_contiguous():
        raise ValueError(f"a must be a contiguous [E, R, {k}] tensor")
    if b.shape != (a.shape[0], n, a.shape[1]) or not b.is_contiguous():
        raise ValueError(f"b must be a contiguous [{a.shape[0]}, {n}, {a.shape[1]}] tensor")
    if scale.device != device:
        _check_device_tensor("scale", scale, device)
    if scale.dtype != torch.float32 or scale.shape != (a.shape[0],) or not scale.is_contiguous():
        raise ValueError(f"scale must be a contiguous float32 [{a.shape[0]}] tensor")
    if ids.device != device:
        _check_device_tensor("ids", ids, device)
    if ids.dtype != torch.int32 or ids.dim() != 1 or not ids.is_contiguous() or ids.numel() < 1:
        raise ValueError("ids must be a contiguous int32 [items] tensor")
    if rows < 1 or rows % ids.numel():
        raise ValueError(f"{rows} rows do not split into {ids.numel()} items")
    if bias is not None:
        if bias.device != device:
            _check_device_tensor("bias", bias, device)
        if bias.dtype != x.dtype or bias.shape != (n,) or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous {x.dtype} [{n}] tensor")
    _lib.ints(outputs=n, columns=k, adapters=a.shape[0], row_stride_of_x=_row_stride(x), row_stride_of_w=_row_stride(w))
    return (rows, n, _row_stride(x), _row_stride(w), (rows, n, k, a.shape[1], a.shape[0], ids.numel()),
            _lib.DTYPES[x.dtype], workspace_bytes(rows, a.shape[1], residual, x.dtype))


def _stride_of(name: str, t: torch.Tensor) -> int:
    stride = _row_stride(t)
    if stride > _lib.INT_MAX:
        raise ValueError(f"{name}'s row stride {stride} must fit 32 bits")
    return stride


def _workspace(workspace, need, device):
    if workspace is None:
        return torch.empty(max(need, 16), device=device, dtype=torch.uint8)
    _check_device_tensor("workspace", workspace, device)
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes")
    return workspace


def adapter_linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, a: torch.Tensor, b: torch.Tensor,
                   scale: torch.Tensor, ids: torch.Tensor, act: str | None = None, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + bias + scale_e (x A_e^T) B_e^T) [M, N] for x [M, K], w [N, K],
    a [E, R, K], b [E, N, R] (``pack_adapters``) and bias [N] or None, fp16 or bf16;
    scale fp32 [E].

    ids: int32 [items] on the device, M a multiple of items: rows in order, M /
    items per item (an utterance of a padded batch; items = M: single tokens).  An
    id outside [0, E) means no adapter.  act: None or "silu".  N and K multiples of
    64, R of 8 up to 128.  Sums in fp32, scale (x A_e^T) rounded to x's type (fp16: relative
    to a power of two of its row, so that it neither overflows nor loses the digits
    of small values).  Rows of x, w and out may be strided.  workspace: a contiguous uint8 tensor of ``workspace_bytes``.
    Forward only."""
    rows, n, ldx, ldw, sizes, dtype, need = _operands(x, w, a, b, scale, ids, bias, False)
    device = x.device
    if act not in (None, "silu"):
        raise ValueError(f"act must be None or 'silu' (got {act!r})")
    if not (plain(x, w, a, b, scale) if bias is None else plain(x, w, a, b, scale, bias)):
        raise ValueError("adapter_linear has no backward: call it under torch.no_grad()")
    if out is None:
        out = torch.empty(rows, n, device=device, dtype=x.dtype)
        ldy = n
    else:
        _check_device_tensor("out", out, device)
        if out.dtype != x.dtype or out.shape != (rows, n) or out.stride(1) != 1:
            raise ValueError(f"out must be a {x.dtype} [{rows}, {n}] tensor with rows contiguous")
        ldy = _stride_of("out", out)
    workspace = _workspace(workspace, need, device)
    lib = _lib.load()
    with _on_device(device):
        rc = lib.sidon_adapter_linear(
            x.data_ptr(), ldx, w.data_ptr(), ldw, None if bias is None else bias.data_ptr(), a.data_ptr(), b.data_ptr(),
            scale.data_ptr(), ids.data_ptr(), out.data_ptr(), ldy, workspace.data_ptr(), workspace.numel(), *sizes,
            _lib.ACTIVATIONS[act], dtype, _stream_handle(device))
    if rc:
        _lib.check("sidon_adapter_linear", rc)
    return out


def adapter_residual(y: torch.Tensor, x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                     scale: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y + x W^T + scale_e (x A_e^T) B_e^T into the fp32 stream y [M, N], in place
    or, with ``out`` fp32 [M, N], beside it; the other arguments as for
    ``adapter_linear``.  The low-rank term keeps fp32 accuracy."""
    rows, n, ldx, ldw, sizes, dtype, need = _operands(x, w, a, b, scale, ids, None, True)
    device = x.device
    out = y if out is None else out
    for name, t in (("y", y), ("out", out)):
        _check_device_tensor(name, t, device)
        if t.dtype != torch.float32 or t.shape != (rows, n) or t.stride(1) != 1:
            raise ValueError(f"{name} must be a float32 [{rows}, {n}] tensor with rows contiguous")
    if not plain(y, x, w, a, b, scale):
        raise ValueError("adapter_residual has no backward: call it under torch.no_grad()")
    ldadd, ldy = _stride_of("y", y), _stride_of("out", out)
    workspace = _workspace(workspace, need, device)
    lib = _lib.load()
    with _on_device(device):
        rc = lib.sidon_adapter_residual(
            x.data_ptr(), ldx, w.data_ptr(), ldw, a.data_ptr(), b.data_ptr(), scale.data_ptr(), ids.data_ptr(),
            y.data_ptr(), ldadd, out.data_ptr(), ldy, workspace.data_ptr(), workspace.numel(),
            *sizes, dtype, _stream_handle(device))
    if rc:
        _lib.check("sidon_adapter_residual", rc)
    return out
