"""Attention over states of another length on the HIP kernels
(csrc/cross_attn.hip, csrc/cross_attn_bwd.hip).

A decoder's tokens read the encoder's frames:

    out = softmax(scale q k^T) v        over the frames j < lens

next to ``flexrel.flexrel_attention`` and ``diff_attention.diff_attention``:
strided views, device lengths (the encoder's ``frames``), grouped heads, the
current stream, captured into HIP graphs like them; prompts and single tokens,
and the gradients for training.  No counterpart in the reference.
"""

from __future__ import annotations

import torch

from . import _lib
from .conformer import plain, written
from .diff_attention import _strides
from .flexrel import _check_device_tensor, _on_device, _stream_handle

HEAD_DIMS = (64, 128)

_layouts = _lib.Layouts()
_backward_layouts = _lib.Layouts()


def workspace_bytes(batch: int, heads: int, kv_heads: int, length: int, keys: int, dim: int, device=None) -> int:
    """Bytes of ``cross_attention``'s workspace on ``device`` (0: none needed)."""
    _lib.ints(batch=batch, heads=heads, kv_heads=kv_heads, length=length, keys=keys, dim=dim)
    with _on_device(device):
        return int(_lib.load().sidon_cross_attention_workspace_bytes(batch, heads, kv_heads, length, keys, dim))


def backward_workspace_bytes(batch: int, heads: int, kv_heads: int, length: int, keys: int, dim: int,
                             dtype: torch.dtype) -> int:
    """Bytes of ``cross_attention_backward``'s workspace."""
    _lib.ints(batch=batch, heads=heads, kv_heads=kv_heads, length=length, keys=keys, dim=dim)
    return int(_lib.load().sidon_cross_attention_bwd_workspace_bytes(batch, heads, kv_heads, length, keys, dim,
                                                                     _lib.DTYPES.get(dtype, -1)))


def _layout(*tensors) -> tuple:
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors])


def _check(q, k, v, lens, q_lens) -> tuple:
    """-> (sizes, type code, strides of q, k and v, of a contiguous out, workspace bytes)."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be [B, H, L, D], k and v [B, heads, S, D]")
    batch, heads, length, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    if dim not in HEAD_DIMS:
        raise ValueError(f"q must be [B, H, L, {HEAD_DIMS}] (got {tuple(q.shape)})")
    if min(q.shape) < 1 or min(k.shape) < 1:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must not be empty")
    if k.shape != (batch, kv_heads, keys, dim) or v.shape != k.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if heads % kv_heads:
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16 (got {q.dtype})")
    device = q.device
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_device_tensor(name, t, device)
        if t.dtype != q.dtype:
            raise TypeError(f"{name} is {t.dtype}, q is {q.dtype}")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
    for name, t in (("lens", lens), ("q_lens", q_lens)):
        if t is not None:
            _check_device_tensor(name, t, device)
            if t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor of shape [B]")
    sizes = (batch, heads, kv_heads, length, keys, dim)
    return (sizes, _lib.DTYPES[q.dtype], (_strides(q), _strides(k), _strides(v)),
            _strides(torch.empty(q.shape, device="meta")), workspace_bytes(*sizes, device))


def _scale(scale, dim) -> float:
    return dim ** -0.5 if scale is None else float(scale)


def _check_lse(lse, sizes, device) -> None:
    _check_device_tensor("lse", lse, device)
    shape = (sizes[0], sizes[1], sizes[3])
    if lse.dtype != torch.float32 or tuple(lse.shape) != shape or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 {shape} tensor")


def _workspace(workspace, need, like):
    if workspace is None:
        return like.new_empty(need, dtype=torch.uint8) if need else None
    device = like.device
    _check_device_tensor("workspace", workspace, device)
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes")
    return workspace


def _out(name, out, like):
    """-> (tensor, strides): ``out``, or a new contiguous tensor of ``like``'s shape."""
    if out is None:
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
    else:
        _check_device_tensor(name, out, like.device)
        if out.dtype != like.dtype or out.shape != like.shape or out.stride(-1) != 1:
            raise ValueError(f"{name} must be a {like.dtype} {tuple(like.shape)} tensor with a contiguous last dimension")
    return out, _strides(out)


def _ptr(t):
    return None if t is None else t.data_ptr()


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor | None = None,
                    q_lens: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """q [B, H, L, D], k and v [B, Hk, S, D] fp16 or bf16 -> [B, H, L, D] of their type.

    Any strides that are multiples of 8 elements with the last dimension
    contiguous (views of fused projections or of a cache), D 64 or 128.  H / Hk
    neighbouring heads share a key head.  lens: int32 [B] valid keys on the device
    (None: all S), q_lens: int32 [B] valid queries (None: all L); what lies past
    either does not matter.  A query without keys, or past q_lens, gives zeros.
    scale: of the scores, positive (None: 1 / sqrt D).  out: optional [B, H, L, D], in
    memory apart from the inputs (a column block of one tensor with q is, and items in turn with it).  lse: optional
    contiguous fp32 [B, H, L] that takes the logarithm of the sums of exponentials,
    which ``cross_attention_backward`` wants.  workspace: a contiguous uint8 tensor of
    ``workspace_bytes``, apart from all of them; allocated per call when None.
    A single query against many keys splits them over the chip.  Probabilities are
    rounded to the inputs' type in front of v, but with H / Hk * L <= 32 (single
    tokens), where the output's rounding is the only one; with more that depends on all
    sizes."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)):
        raise TypeError("q, k and v must be torch.Tensor")
    key = _layout(q, k, v, lens, q_lens)
    sizes, dtype, strides, o_strides, need = _layouts.get(key) or _layouts.keep(key, _check(q, k, v, lens, q_lens))
    device, given = q.device, out
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        out, o_strides = _out("out", out, q)
    if lse is not None:
        _check_lse(lse, sizes, device)
    if not (plain(q, k, v) if given is lse is None else plain(q, k, v, out, *(() if lse is None else (lse,)))):
        raise ValueError("cross_attention follows no gradient: call it under torch.no_grad(), and "
                         "cross_attention_backward for the gradients")
    lib = _lib.load()
    with _on_device(device):
        workspace = _workspace(workspace, need, q)
        rc = lib.sidon_cross_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(lens), _ptr(q_lens), _scale(scale, sizes[-1]), out.data_ptr(),
            _ptr(lse), _ptr(workspace), 0 if workspace is None else workspace.numel(), *sizes, dtype, *strides,
            o_strides, _stream_handle(device))
    if rc:
        _lib.check("sidon_cross_attention", rc)
    written(given, lse)
    return out


def _check_backward(dout, q, k, v, out, lse, lens, q_lens) -> tuple:
    """-> (sizes, type code, strides of dout, q, k, v and out, of contiguous dq, dk and dv, workspace bytes)."""
    sizes, dtype, strides, contiguous, _ = _check(q, k, v, lens, q_lens)
    for name, t in (("dout", dout), ("out", out)):
        _check_device_tensor(name, t, q.device)
        if t.dtype != q.dtype or t.shape != q.shape or t.stride(-1) != 1:
            raise ValueError(f"{name} must be a {q.dtype} {tuple(q.shape)} tensor with a contiguous last dimension")
    _check_lse(lse, sizes, q.device)
    like_k = _strides(torch.empty(k.shape, device="meta"))
    return (sizes, dtype, (_strides(dout), *strides, _strides(out)), (contiguous, like_k, like_k),
            backward_workspace_bytes(*sizes, q.dtype))


def cross_attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, lens: torch.Tensor | None = None, q_lens: torch.Tensor | None = None,
                             scale: float | None = None, dq: torch.Tensor | None = None,
                             dk: torch.Tensor | None = None, dv: torch.Tensor | None = None,
                             workspace: torch.Tensor | None = None):
    """The gradients (dq, dk, dv) of ``cross_attention``'s q, k and v from its output's.

    q, k, v, lens, q_lens and scale as the forward call had them, out and lse as it
    left them; dout [B, H, L, D] of the same type (any strides as q's; what it holds past
    q_lens does not matter).  dq like q, dk and dv like k, optional, in memory apart from the other operands
    (column blocks of one tensor are, and items in turn); they are written, zeros past the valid queries and
    keys.  Heads that share a key head are summed in fp32.  workspace: a contiguous uint8
    tensor of ``backward_workspace_bytes``; allocated per call when None.  Equal calls
    give equal bits."""
    if not all(isinstance(t, torch.Tensor) for t in (dout, q, k, v, out, lse)):
        raise TypeError("dout, q, k, v, out and lse must be torch.Tensor")
    key = _layout(dout, q, k, v, out, lse, lens, q_lens)
    sizes, dtype, strides, contiguous, need = (
        _backward_layouts.get(key)
        or _backward_layouts.keep(key, _check_backward(dout, q, k, v, out, lse, lens, q_lens)))
    device, given = q.device, (dq, dk, dv)
    outs = []
    for i, (name, t, like) in enumerate((("dq", dq, q), ("dk", dk, k), ("dv", dv, v))):
        outs.append((torch.empty_like(like, memory_format=torch.contiguous_format), contiguous[i]) if t is None
                    else _out(name, t, like))
    if not plain(dout, q, k, v, out, lse, *[t for t in given if t is not None]):
        raise ValueError("cross_attention_backward follows no gradient: call it under torch.no_grad()")
    lib = _lib.load()
    with _on_device(device):
        workspace = _workspace(workspace, need, q)
        rc = lib.sidon_cross_attention_bwd(
            dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(lens),
            _ptr(q_lens), _scale(scale, sizes[-1]), *[t.data_ptr() for t, _ in outs], workspace.data_ptr(),
            workspace.numel(), *sizes, dtype, *strides, *[s for _, s in outs], _stream_handle(device))
    if rc:
        _lib.check("sidon_cross_attention_bwd", rc)
    written(*given)
    return tuple(t for t, _ in outs)
