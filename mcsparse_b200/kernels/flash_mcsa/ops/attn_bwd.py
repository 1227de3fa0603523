"""Launch of the attention's backward kernels, shared by the dense and the gather-KV entry points.

Everything here works on (B, S, H, D) tensors; the entry points own argument meaning and layouts.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from mcsparse_b200 import _lib


def readable(t: Tensor) -> Tensor:
    """``t`` itself where the kernels can read it in place, else a contiguous copy: rows contiguous, 16-byte address and strides,
    and strides that nest without overlap (an expanded gradient, for instance, is copied)."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    end = t.shape[-1]
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride()[:-1], t.shape[:-1]) if sz > 1):
        ok = ok and stride >= end and stride % 8 == 0
        end = stride * size
    if ok:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: Tensor) -> Tuple[int, ...]:
    # (the stride of a dimension of extent 1 is never used, but has to be a multiple of 16 bytes)
    return tuple(st if sz > 1 else 0 for st, sz in zip(t.stride()[:3], t.shape[:3]))


def launch_backward(entry: str, dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, dq: Tensor, dk: Tensor, dv: Tensor,
                    softmax_scale: float, gi: Optional[Tensor] = None, gl: Optional[Tensor] = None, perm: Optional[Tensor] = None,
                    group_rows: int = 128) -> None:
    """Fill dq, dk, dv.  All tensors are (B, S, H, D), checked by the caller and readable by the kernels."""
    a = _lib.AttnBwdArgs()
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", dout), ("dq", dq), ("dk", dk), ("dv", dv)):
        setattr(a, name, t.data_ptr())
        dst = getattr(a, name + "_stride")
        dst[0], dst[1], dst[2] = _strides(t)
    a.lse = lse.data_ptr()
    a.gi, a.gl, a.perm = (None if t is None else t.data_ptr() for t in (gi, gl, perm))
    a.B, a.Sq, a.H, a.D = q.shape
    a.Sk = k.shape[1]
    a.gather_len, a.group_rows = (0 if gi is None else gi.shape[-1]), int(group_rows)
    a.dtype = _lib.MCS_DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.MCS_DTYPE_FP16
    a.softmax_scale = float(softmax_scale)
    need = getattr(_lib.lib(), entry + "_workspace_bytes")(a)
    if need < 0:
        _lib.raise_on_error(need, entry)
    with torch.cuda.device(q.device):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), need
        a.status = _lib.status_word(q.device).data_ptr()
        _lib.launch(entry, a, q.device, entry)


def check_saved(dout: Tensor, out: Tensor, lse: Tensor, q: Tensor, lse_shape) -> None:
    """The gradient from above and what the forward pass left must belong to q."""
    for name, t in (("dout", dout), ("out", out)):
        if tuple(t.shape) != tuple(q.shape) or t.dtype != q.dtype:
            raise ValueError(f"{name} must have q's shape {tuple(q.shape)} and dtype {q.dtype}, got {tuple(t.shape)} {t.dtype}")
    if tuple(lse.shape) != tuple(lse_shape) or lse.dtype != torch.float32:
        raise ValueError(f"lse must be float32 of shape {tuple(lse_shape)}, got {lse.dtype} {tuple(lse.shape)}")
    if any(t.device != q.device for t in (dout, out, lse)):
        raise ValueError("dout, out and lse must be on q's device")
