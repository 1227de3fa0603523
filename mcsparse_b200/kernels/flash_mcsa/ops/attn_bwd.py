"""Launch of the attention's backward kernels, shared by the dense and the gather-KV entry points.

Everything here works on (B, S, H, D) tensors; the entry points own argument meaning and layouts.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch
from torch import Tensor

from mcsparse_b200 import _lib

_ARGS = struct.Struct("15Q24q8ifi")           # the fields of mcs_attn_bwd_args
assert _ARGS.size == C.sizeof(_lib.AttnBwdArgs)


def readable(t: Tensor) -> Tensor:
    """``t`` itself where the kernels can read it in place, else a contiguous copy: rows contiguous, 16-byte address and strides,
    and strides that nest without overlap (an expanded gradient, for instance, is copied)."""
    st, sz = t.stride(), t.shape
    end = sz[3]
    ok = st[3] == 1 and t.data_ptr() % 16 == 0
    for stride, size in sorted(zip(st[:3], sz[:3])):
        if size > 1:
            ok = ok and stride >= end and stride % 8 == 0
            end = stride * size
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def gradient_like(t: Tensor) -> Tensor:
    """Memory for the gradient of ``t``, in its layout where that one's rows are contiguous."""
    g = torch.empty_like(t, requires_grad=False)             # (of windows, stride 1 twice, the rows may not be)
    return g if g.stride(3) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format, requires_grad=False)


def launch_backward(entry: str, dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, dq: Tensor, dk: Tensor, dv: Tensor,
                    softmax_scale: float, gi: Optional[Tensor] = None, gl: Optional[Tensor] = None, perm: Optional[Tensor] = None,
                    group_rows: int = 128, heads_first: bool = False) -> None:
    """Fill dq, dk, dv.  All tensors are (B, S, H, D), or (B, H, S, D) with ``heads_first``; checked by the caller and readable by
    the kernels."""
    row, head = (2, 1) if heads_first else (1, 2)
    strides = []
    for t in (q, k, v, out, dout, dq, dk, dv):
        # (the stride of a dimension of extent 1 is never used, but has to be a multiple of 16 bytes)
        st, sz = t.stride(), t.shape
        strides += [st[0] if sz[0] > 1 else 0, st[row] if sz[row] > 1 else 0, st[head] if sz[head] > 1 else 0]
    shape = q.shape
    sizes = (shape[0], shape[row], k.shape[row], shape[head], shape[3], 0 if gi is None else gi.shape[-1], int(group_rows),
             _lib.MCS_DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.MCS_DTYPE_FP16, float(softmax_scale), 0)
    pointers = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                0 if gi is None else gi.data_ptr(), 0 if gl is None else gl.data_ptr(), 0 if perm is None else perm.data_ptr())
    a = _lib.packed(_lib.AttnBwdArgs, _ARGS, *pointers, 0, 0, 0, *strides, *sizes)
    need = getattr(_lib.lib(), entry + "_workspace_bytes")(a)
    if need < 0:
        _lib.raise_on_error(need, entry)
    device = q.device
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    a.status = _lib.status_word(device).data_ptr()
    if device.index == torch.cuda.current_device():
        _lib.launch(entry, a, device, entry)
    else:
        with torch.cuda.device(device):
            _lib.launch(entry, a, device, entry)


def check_saved(dout: Tensor, out: Tensor, lse: Tensor, q: Tensor, lse_shape) -> None:
    """The gradient from above and what the forward pass left must belong to q."""
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise ValueError(f"{name} must have q's shape {tuple(q.shape)} and dtype {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if tuple(lse.shape) != tuple(lse_shape) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 of shape {tuple(lse_shape)}, got {lse.dtype} {tuple(lse.shape)}")
    if any(t.device != q.device for t in (dout, out, lse)):
        raise ValueError("dout, out and lse must be on q's device")
