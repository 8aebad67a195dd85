"""The norm of queries and keys for each head with the position rotation in the
same pass, and its gradients, on the HIP kernels (csrc/head_norm.hip).

What a decoder layer does to the heads of its projections in front of an
attention (``cross_attention.cross_attention`` and the others of this package):

    y = R_p (w * x / sqrt(mean(x^2) + eps))

with R_p the rotation of pairs of a head's first dimensions by the angles of
its token's place p.  Strided views of fused projections, places on the device,
in place or out, captured into HIP graphs like its neighbours.  No counterpart
in the reference.
"""

from __future__ import annotations

import torch

from . import _lib
from .conformer import plain, written
from .diff_attention import _strides
from .flexrel import _check_device_tensor, _on_device, _stream_handle

_layouts = _lib.Layouts()
_NONE = _strides(torch.empty(1, 1, 1, 1, device="meta"))


def workspace_bytes(batch: int, heads: int, kv_heads: int, length: int, keys: int, dim: int) -> int:
    """Bytes of ``qk_norm_rotary_backward``'s workspace (kv_heads 0: no keys)."""
    _lib.ints(batch=batch, heads=heads, kv_heads=kv_heads, length=length, keys=keys, dim=dim)
    return int(_lib.load().sidon_qk_norm_rotary_workspace_bytes(batch, heads, kv_heads, length, keys, dim))


def _layout(*tensors) -> tuple:
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors])


def _rows(name, t, shape, like) -> None:
    _check_device_tensor(name, t, like.device)
    if t.dtype != like.dtype or tuple(t.shape) != shape or t.stride(-1) != 1:
        raise ValueError(f"{name} must be a {like.dtype} {shape} tensor with a contiguous last dimension")


def _check(q, k, q_w, k_w, cos, sin, q_pos, k_pos) -> tuple:
    """-> (sizes, type code, rotated dimensions, places, strides of q and k, of contiguous outputs)."""
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be [B, heads, tokens, D]")
    if q.dtype not in _lib.DTYPES:
        raise TypeError(f"q must be float32, float16 or bfloat16 (got {q.dtype})")
    device = q.device
    batch, heads, length, dim = q.shape
    kv_heads, keys = (0, 0) if k is None else (k.shape[1], k.shape[2])
    if min(q.shape) < 1 or (k is not None and min(k.shape) < 1):
        raise ValueError("q and k must not be empty")
    if dim % 16 or not 16 <= dim <= 256:
        raise ValueError(f"heads must have a multiple of 16 dimensions up to 256 (got {dim})")
    _rows("q", q, tuple(q.shape), q)
    if k is not None:
        _rows("k", k, (batch, kv_heads, keys, dim), q)
    if (k is None) != (k_w is None):
        raise ValueError("k and k_w belong together")
    if k is None and k_pos is not None:
        raise ValueError("k_pos without k")
    for name, t in (("q_w", q_w), ("k_w", k_w)):
        if t is None and name == "k_w":
            continue
        _check_device_tensor(name, t, device)
        if t.dtype != torch.float32 or tuple(t.shape) != (dim,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 [{dim}] tensor")
    rot = places = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin belong together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            _check_device_tensor(name, t, device)
            if t.dtype != torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.shape != cos.shape:
                raise ValueError(f"{name} must be a contiguous float32 [places, rotated dimensions / 2] tensor")
        places, rot = cos.shape[0], 2 * cos.shape[1]
        if places < 1 or rot % 16 or not 16 <= rot <= dim:
            raise ValueError(f"the tables rotate {rot} of {dim} dimensions at {places} places: need a multiple of 16")
    for name, t, tokens in (("q_pos", q_pos, length), ("k_pos", k_pos, keys)):
        if t is not None:
            _check_device_tensor(name, t, device)
            if t.dtype != torch.int32 or tuple(t.shape) != (batch, tokens) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 [{batch}, {tokens}] tensor")
        elif rot and tokens > places:
            raise ValueError(f"{tokens} tokens, the tables have {places} places")
    sizes = (batch, heads, kv_heads, length, keys, dim)
    _lib.ints(batch=batch, heads=heads, kv_heads=kv_heads, length=length, keys=keys, places=places)
    return (sizes, _lib.DTYPES[q.dtype], rot, places, (_strides(q), _NONE if k is None else _strides(k)),
            (_strides(torch.empty(q.shape, device="meta")),
             _NONE if k is None else _strides(torch.empty(k.shape, device="meta"))))


def _found(q, k, q_w, k_w, cos, sin, q_pos, k_pos) -> tuple:
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    key = _layout(q, k, q_w, k_w, cos, sin, q_pos, k_pos)
    return _layouts.get(key) or _layouts.keep(key, _check(q, k, q_w, k_w, cos, sin, q_pos, k_pos))


def _plain(name, *tensors) -> None:
    if not plain(*[t for t in tensors if t is not None]):
        raise ValueError(f"{name} takes plain tensors that need no gradient: call it under torch.no_grad()")


def _out(name, out, like, contiguous):
    """-> (tensor, strides): ``out``, or a new contiguous tensor of ``like``'s shape."""
    if like is None:
        if out is not None:
            raise ValueError(f"{name} without k")
        return None, _NONE
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format), contiguous
    _rows(name, out, tuple(like.shape), like)
    return out, _strides(out)


def _ptr(t):
    return None if t is None else t.data_ptr()


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_w: torch.Tensor, k_w: torch.Tensor | None,
                   cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                   q_pos: torch.Tensor | None = None, k_pos: torch.Tensor | None = None, eps: float = 1e-6,
                   interleaved: bool = False, out_q: torch.Tensor | None = None, out_k: torch.Tensor | None = None):
    """q [B, H, L, D], k [B, Hk, S, D] (or None) fp32, fp16 or bf16 -> the same
    shapes and type (contiguous, or out_q and out_k): each head's D values divided
    by their root mean square (with eps under the root), times q_w or k_w (fp32
    [D]), and rotated.

    Any strides of whole 16 bytes with the last dimension contiguous; D a multiple
    of 16 up to 256.  cos, sin: fp32 [places, R / 2] tables of the angles that the
    first R dimensions turn by (None: no rotation), pairs (j, j + R / 2), or
    (2j, 2j + 1) with ``interleaved``.  q_pos [B, L], k_pos [B, S]: int32 places on
    the device (None: 0, 1, ...); a negative one marks padding, which gives zeros;
    one past the tables gives NaN in the rotated dimensions.  out_q may be q itself,
    out_k k; they must not share other memory with an operand."""
    sizes, dtype, rot, places, strides, contiguous = _found(q, k, q_w, k_w, cos, sin, q_pos, k_pos)
    given = (out_q, out_k)
    out_q, oq = _out("out_q", out_q, q, contiguous[0])
    out_k, ok = _out("out_k", out_k, k, contiguous[1])
    _plain("qk_norm_rotary", q, k, q_w, k_w, cos, sin, *given)
    lib = _lib.load()
    with _on_device(q.device):
        rc = lib.sidon_qk_norm_rotary(
            q.data_ptr(), _ptr(k), out_q.data_ptr(), _ptr(out_k), q_w.data_ptr(), _ptr(k_w), _ptr(cos), _ptr(sin), places,
            rot, 1 if interleaved else 0, _ptr(q_pos), _ptr(k_pos), eps, *sizes, dtype, *strides, oq, ok,
            _stream_handle(q.device))
    if rc:
        _lib.check("sidon_qk_norm_rotary", rc)
    written(*given)
    return out_q, out_k


def qk_norm_rotary_backward(dout_q: torch.Tensor, dout_k: torch.Tensor | None, q: torch.Tensor,
                            k: torch.Tensor | None, q_w: torch.Tensor, k_w: torch.Tensor | None,
                            cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                            q_pos: torch.Tensor | None = None, k_pos: torch.Tensor | None = None, eps: float = 1e-6,
                            interleaved: bool = False, dq: torch.Tensor | None = None, dk: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None):
    """The gradients (dq, dk, dq_w, dk_w) of ``qk_norm_rotary``'s arguments from
    those of its outputs.

    The arguments are those of the forward call (q and k as they went in; an
    in-place call has overwritten them); dout_q and dout_k of q's and k's shapes and type, any
    strides of whole 16 bytes (expanded tensors too).  dq, dk: optional outputs,
    dq in dout_q's or q's own place if wanted, dk likewise.  dq_w and dk_w are fp32
    [D], sums over all heads and tokens in a fixed order.  workspace: a contiguous
    uint8 tensor of ``workspace_bytes``; allocated per call when None.  Without k the
    second and fourth are None."""
    sizes, dtype, rot, places, strides, contiguous = _found(q, k, q_w, k_w, cos, sin, q_pos, k_pos)
    given = (dq, dk)
    _rows("dout_q", dout_q, tuple(q.shape), q)
    if (dout_k is None) != (k is None):
        raise ValueError("dout_k and k belong together")
    if k is not None:
        _rows("dout_k", dout_k, tuple(k.shape), k)
    dq, sq = _out("dq", dq, q, contiguous[0])
    dk, sk = _out("dk", dk, k, contiguous[1])
    _plain("qk_norm_rotary_backward", dout_q, dout_k, q, k, q_w, k_w, cos, sin, *given)
    dim, device = sizes[-1], q.device
    dw = q_w.new_empty((1 if k is None else 2, dim))
    lib = _lib.load()
    with _on_device(device):
        need = lib.sidon_qk_norm_rotary_workspace_bytes(*sizes)
        if workspace is None:
            workspace = q.new_empty(need, dtype=torch.uint8)
        else:
            _check_device_tensor("workspace", workspace, device)
            if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
                raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes")
        rc = lib.sidon_qk_norm_rotary_bwd(
            dout_q.data_ptr(), _ptr(dout_k), q.data_ptr(), _ptr(k), dq.data_ptr(), _ptr(dk), dw.data_ptr(),
            None if k is None else dw[1].data_ptr(), q_w.data_ptr(), _ptr(k_w), _ptr(cos), _ptr(sin), places, rot,
            1 if interleaved else 0, _ptr(q_pos), _ptr(k_pos), eps, workspace.data_ptr(), workspace.numel(), *sizes,
            dtype, _strides(dout_q), _NONE if k is None else _strides(dout_k), *strides, sq, sk, _stream_handle(device))
    if rc:
        _lib.check("sidon_qk_norm_rotary_bwd", rc)
    written(*given)
    return dq, dk, dw[0], None if k is None else dw[1]
