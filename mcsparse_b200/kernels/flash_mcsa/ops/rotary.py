"""Rotary positions of q and k, forward and backward, on (B, L, H, D) tensors.

The reference leaves the rotary embedding to the host model (its ``forward_op``, ``mcsparse/h3/context_parallel.py``
:165-176, gets rotated q and k); this package fuses it into the exchange of a context-parallel layer
(``h3/ulysses_layer.py``).  Here it stands alone, with its gradient, for a layer that is trained: interleaved or half
layout, the whole head or its first part, one position axis (text, frames) or several (a video grid), and the usual ways
to stretch the frequencies for longer sequences.  The kernel (``mcs_rotary``) computes the angles from integer positions
exactly, without a table, so positions have no upper limit.
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from decimal import Decimal, localcontext
from typing import Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from mcsparse_b200 import _lib

_DTYPES = {torch.bfloat16: _lib.MCS_DTYPE_BF16, torch.float16: _lib.MCS_DTYPE_FP16, torch.float32: _lib.MCS_DTYPE_FP32}
_ARGS = struct.Struct("4Q12qQ3q2Q11if")     # the fields of mcs_rotary_args
assert _ARGS.size == C.sizeof(_lib.RotaryArgs)
_TWO_PI = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582")


def _turns(freq: float) -> int:
    """round(2^64 freq / (2 pi)) modulo 2^64: the part of a turn that one step of position adds."""
    with localcontext() as ctx:
        ctx.prec = 60
        return int((Decimal(freq) * (1 << 64) / _TWO_PI).to_integral_value()) % (1 << 64)


def _per_axis(value, n: int, what: str) -> Tuple[float, ...]:
    values = tuple(float(x) for x in value) if isinstance(value, (tuple, list)) else (float(value),) * n
    if len(values) != n or not all(math.isfinite(x) and x > 0 for x in values):
        raise ValueError(f"{what} must be a positive number, or one for each of the {n} axes, got {value!r}")
    return values


class RotaryEmbedding:
    """Plan of a rotary embedding: frequencies, axes and layout.  It lives on the host and serves every device and stream.

    ``head_dim``; ``rotary_dim`` (default: all of it) is the part of the head, from its start, that is rotated; the rest
    passes through.  ``axis_pairs`` says how many of the ``rotary_dim / 2`` pairs turn with each position axis, in order
    (default: one axis; ``h3.ulysses_layer.rope_pairs(head_dim)`` for a frame / row / column grid).  Pair ``i`` of an axis
    with ``n`` pairs turns by ``position * theta**(-i/n)``.  ``layout``: ``"interleaved"`` pairs elements (2p, 2p+1),
    ``"half"`` pairs (p, p + rotary_dim/2).

    ``scaling`` stretches the frequencies by ``factor`` (> 0; one number, or one per axis):

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: theta times ``factor**(n/(n-1))``, so that the lowest frequency would be divided by ``factor`` and the highest
      stays (one pair: as ``"linear"``);
    * ``"yarn"``: with r the turns that a pair makes over ``original_length`` (one number, or one per axis), frequencies with
      r >= ``beta_fast`` stay, those with r <= ``beta_slow`` are divided by ``factor``, linear in r between (a model that was
      trained with a ramp in the pair's index instead is rotated differently by this); the rotation is scaled by
      ``magnitude``, default 0.1 ln(largest factor) + 1 (at least 1).

    ``magnitude`` (default 1 except for ``"yarn"``) multiplies the rotated part.
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, axis_pairs: Optional[Sequence[int]] = None,
                 theta: float = 10000.0, layout: str = "interleaved", scaling: Optional[str] = None,
                 factor: Union[float, Sequence[float]] = 1.0, original_length: Union[float, Sequence[float], None] = None,
                 beta_fast: float = 32.0, beta_slow: float = 1.0, magnitude: Optional[float] = None):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim or rotary_dim > 256:
            raise ValueError(f"rotary_dim must be even, at least 2 and at most head_dim and 256, got {rotary_dim} of {head_dim}")
        pairs = (rotary_dim // 2,) if axis_pairs is None else tuple(int(x) for x in axis_pairs)
        if not 1 <= len(pairs) <= 3 or min(pairs) < 0 or sum(pairs) != rotary_dim // 2:
            raise ValueError(f"axis_pairs must give 1 to 3 counts that sum to {rotary_dim // 2}, got {axis_pairs!r}")
        if layout not in ("interleaved", "half"):
            raise ValueError(f"layout must be 'interleaved' or 'half', got {layout!r}")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
        if not (math.isfinite(theta) and theta > 0):
            raise ValueError(f"theta must be positive, got {theta!r}")
        factors = _per_axis(factor, len(pairs), "factor")
        if scaling == "yarn":
            if original_length is None:
                raise ValueError("scaling='yarn' needs original_length")
            if not beta_fast > beta_slow:
                raise ValueError("beta_fast must be greater than beta_slow")
            lengths = _per_axis(original_length, len(pairs), "original_length")
        if magnitude is None:
            magnitude = max(1.0, 0.1 * math.log(max(factors)) + 1.0) if scaling == "yarn" else 1.0
        if not math.isfinite(magnitude):
            raise ValueError(f"magnitude must be finite, got {magnitude!r}")
        self.head_dim, self.rotary_dim, self.axis_pairs, self.layout = head_dim, rotary_dim, pairs, layout
        self.magnitude = float(magnitude)
        freq, axis = [], []
        for a, n in enumerate(pairs):
            base, s = theta, factors[a]
            if scaling == "ntk" and n > 1:
                base = theta * s ** (n / (n - 1))
            for i in range(n):
                f = base ** (-i / n)
                if scaling == "linear" or (scaling == "ntk" and n == 1):
                    f /= s
                elif scaling == "yarn":
                    keep = min(1.0, max(0.0, (lengths[a] * f / (2 * math.pi) - beta_slow) / (beta_fast - beta_slow)))
                    f = keep * f + (1.0 - keep) * f / s
                freq.append(f)
                axis.append(a)
        self.frequencies, self.pair_axis = tuple(freq), tuple(axis)
        self._lay_out()

    def _lay_out(self) -> None:
        """The arrays that a launch copies into its arguments."""
        n = len(self.frequencies)
        self._turns = (C.c_uint64 * n)(*[_turns(f) for f in self.frequencies])
        self._axis = (C.c_uint8 * n)(*self.pair_axis)

    def __getstate__(self):
        return {k: x for k, x in self.__dict__.items() if k not in ("_turns", "_axis")}

    def __setstate__(self, state) -> None:
        self.__dict__.update(state)
        self._lay_out()

    # ------------------------------------------------------------------------------------------ launches
    def _check(self, tensors: Sequence[Tensor], positions: Tensor) -> Tuple[int, int, int]:
        """The positions' (batch, row, axis) strides; raises on arguments that the kernel does not take."""
        if not 1 <= len(tensors) <= 2:
            raise ValueError(f"one or two tensors are rotated at a time, got {len(tensors)}")
        x = tensors[0]
        dtype, device = x.dtype, x.device
        for t in tensors:
            shape = t.shape
            if len(shape) != 4 or shape[3] != self.head_dim:
                raise ValueError(f"expected (B, L, H, {self.head_dim}) tensors, got {tuple(shape)}")
            if shape[:2] != x.shape[:2]:
                raise ValueError(f"batch and length must agree, got {tuple(x.shape)} and {tuple(shape)}")
            if t.dtype not in _DTYPES or t.dtype != dtype:
                raise TypeError(f"rotary positions need bf16, fp16 or fp32 tensors of one dtype, got {t.dtype}")
        B, L = x.shape[:2]
        axes = len(self.axis_pairs)
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        shape, strides = tuple(positions.shape), positions.stride()
        if axes == 1:
            shape, strides = shape + (1,), strides + (0,)
        if len(shape) == 2:
            shape, strides = (1,) + shape, (0,) + strides
        if len(shape) != 3 or shape[0] not in (1, B) or shape[1] != L or shape[2] != axes:
            lead = f"({L},) or ({B}, {L})" if axes == 1 else f"({L}, {axes}) or ({B}, {L}, {axes})"
            raise ValueError(f"positions must have shape {lead}, got {tuple(positions.shape)}")
        for t in tensors:
            if not t.is_cuda:
                raise RuntimeError("rotary positions run on a CUDA device only; there is no CPU path")
            if t.device != device:
                raise ValueError("tensors and positions must be on one device")
        if positions.device != device:
            raise ValueError("tensors and positions must be on one device")
        return strides if shape[0] == B else (0, strides[1], strides[2])

    def _launch(self, tensors: Sequence[Tensor], positions: Tensor, inverse: bool, inplace: bool) -> Tuple[Tensor, ...]:
        p_stride = self._check(tensors, positions)
        if inplace:
            for t in tensors:
                if t.stride(-1) != 1 or _overlaps_itself(t):
                    raise ValueError("inplace needs tensors with contiguous rows whose elements do not share memory")
            if len(tensors) == 2 and _may_share(*tensors):
                raise ValueError("inplace needs two tensors that share no element")
            src = outs = tuple(tensors)
        else:
            src = tuple(t if t.stride(3) == 1 else t.contiguous() for t in tensors)
            outs = tuple(_memory_like(t) for t in src)
        x, y = src[0], outs[0]
        B, L, H = x.shape[:3]
        if B == 0 or L == 0:
            return outs
        xs, ys = x.stride(), y.stride()
        if len(src) == 2:
            x1, y1 = src[1], outs[1]
            second = (x1.data_ptr(), y1.data_ptr(), x1.stride(), y1.stride(), x1.shape[2])
        else:
            second = (0, 0, (0, 0, 0, 0), (0, 0, 0, 0), 0)
        xs1, ys1 = second[2], second[3]
        a = _lib.packed(_lib.RotaryArgs, _ARGS, x.data_ptr(), second[0], y.data_ptr(), second[1],
                        xs[0], xs[1], xs[2], xs1[0], xs1[1], xs1[2], ys[0], ys[1], ys[2], ys1[0], ys1[1], ys1[2],
                        positions.data_ptr(), *p_stride, C.addressof(self._turns), C.addressof(self._axis),
                        H, second[4], B, L, self.head_dim, len(self.frequencies), len(self.axis_pairs), int(self.layout == "half"),
                        int(positions.dtype == torch.int64), int(inverse), _DTYPES[x.dtype], self.magnitude)
        device = x.device
        if device.index == torch.cuda.current_device():
            _lib.launch("mcs_rotary", a, device, "mcs_rotary")
        else:
            with torch.cuda.device(device):
                _lib.launch("mcs_rotary", a, device, "mcs_rotary")
        if inplace:
            for t in tensors:
                torch.autograd.graph.increment_version(t)      # what autograd saved of it is no longer there
        return outs

    def rotate(self, *tensors: Tensor, positions: Tensor, inplace: bool = False):
        """Rotated copies of one or two (B, L, H, D) tensors (q and k; the head counts may differ), from one launch.

        ``positions``: int32 or int64 on the tensors' device, any strides: (L,) or (B, L) for one axis, (L, axes) or
        (B, L, axes) for several.  Differentiable in the tensors.  ``inplace`` overwrites them instead (forward only; they share no element).
        Returns a tensor for one, a tuple for two."""
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
            if inplace:
                raise RuntimeError("inplace rotation is forward-only; detach the inputs or use torch.no_grad()")
            self._check(tensors, positions)
            outs = _Rotate.apply(self, positions, *tensors)
        else:
            outs = self._launch(tensors, positions, False, inplace)
        return outs[0] if len(tensors) == 1 else outs

    __call__ = rotate

    def rotate_backward(self, *grads: Tensor, positions: Tensor, inplace: bool = False):
        """Gradients of the rotated tensors' inputs from those of the outputs: the rotation the other way, same magnitude."""
        outs = self._launch(grads, positions, True, inplace)
        return outs[0] if len(grads) == 1 else outs


def _memory_like(t: Tensor) -> Tensor:
    """Memory for the rotated ``t``: its order of dimensions, rows contiguous."""
    y = torch.empty_like(t, requires_grad=False)             # (of windows, stride 1 twice, the rows may not be)
    return y if y.stride(3) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format, requires_grad=False)


def _overlaps_itself(t: Tensor) -> bool:
    """Whether two elements of t may share memory: dimensions in the order of their strides do not nest."""
    end = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride < end:
            return True
        end = stride * (size - 1) + end
    return False


def _may_share(a: Tensor, b: Tensor) -> bool:
    """Whether a and b, neither overlapping itself, may have an element in common.  Views of one layout are told apart (heads of a packed
    projection, say); others count as sharing where their ranges of addresses meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    extent = lambda t, dims: 1 + sum(t.stride(d) * (t.shape[d] - 1) for d in dims)
    size, offset = a.element_size(), b.data_ptr() - a.data_ptr()
    if offset >= size * extent(a, range(4)):
        return False
    dims = [d for d in range(4) if a.shape[d] > 1 or b.shape[d] > 1]
    if offset % size or any(a.stride(d) != b.stride(d) and a.shape[d] > 1 and b.shape[d] > 1 for d in dims):
        return True
    offset //= size
    stride = {d: a.stride(d) if a.shape[d] > 1 else b.stride(d) for d in dims}
    order = sorted(dims, key=stride.get)
    for i, d in enumerate(order):
        # modulo a stride that divides all greater ones only the lesser dimensions and the offset remain: apart if those are
        step, inner = stride[d], order[:i]
        if step and all(stride[e] % step == 0 for e in order[i:]):
            rest = offset % step
            if extent(a, inner) <= rest and rest + extent(b, inner) <= step:
                return False
    return True


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan: RotaryEmbedding, positions: Tensor, *tensors: Tensor):
        ctx.plan = plan
        ctx.save_for_backward(positions)
        return plan._launch(tensors, positions, False, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        return (None, None, *ctx.plan._launch(grads, positions, True, False))
