"""Gradients of softmax attention in 64 bits, with elementwise bounds of what a kernel may be off (test infrastructure).

The kernel under test forms, from 16-bit q, k, v, dout, out and an fp32 lse,
    P = exp(scale q k^T - lse), dV = P^T dO, dP = dO V^T, dS = P (dP - delta), delta = rowsum(dO o out), dQ = scale dS K,
    dK = scale dS^T Q
with fp32 products and sums, P and dS rounded once to the input type (relative step u = eps / 2) as operands.  First-order bounds:

* a score is off by 2^-21 of scale sum|q||k| (fp32 products of exact operands, summed in the tensor core) and the exponent's
  argument by as much of |lse|; the exponential itself, the logarithm in lse and their scalings by 2^-20 relative:
      err(P) = P (2^-21 (scale |q||k|^T + |lse|) + 2^-20);
* dV: u P from the rounding of the operand, err(P), both times |dO| summed over queries;
* dS: u |dS| from the rounding of the operand; err(P) |dP - delta|; P times the error of dP, 2^-20 |dO||V|^T, and of delta: the
  difference that the given (rounded) `out` makes, which is computed here, and 2^-20 sum|dO||out|; its products with |K|, |Q| are
  summed;  sums in fp32 add 2^-20 of the sums of magnitudes;
* dQ: the kernel subtracts r PK, r the sum of a row's rounded dS (zero but for the errors above, so |r| is at most their sum) and
  PK = P K: beside sum err(dS) |K| at most sum err(dS) times P |K|;
* fp16: P and dS are scaled by powers of two such that the half-step of the smallest fp16 numbers, 2^-25, stands for less than
  2^-39 of P's largest value 1 and of the bound 2 max|dO| max|V| of dS;
* the result's own rounding, u of its value;
* where an axis is short the kernel takes P and dS as two 16-bit parts each, the rounded value and the rounded rest: u becomes u^2 (`paired`).
"""

from __future__ import annotations

import math

import torch


def head_grads(q, k, v, dout, out, scale, dtype, hide=None, paired=False):
    """One head, 64-bit (n, D) queries and (m, D) keys: (dq, dk, dv) and their bounds before the final rounding.  `hide`: bool (n, m),
    keys that a query does not see.  `dtype`: the kernel's input type."""
    u = torch.finfo(dtype).eps / 2
    if paired:
        u = u * u
    s = scale * (q @ k.t())
    if hide is not None:
        s = s.masked_fill(hide, -math.inf)
    lse = torch.logsumexp(s, dim=-1, keepdim=True)
    p = torch.exp(s - lse)
    o = p @ v
    dp = dout @ v.t()
    delta = (dout * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ k, scale * ds.t() @ q, p.t() @ dout
    err_p = p * (2.0 ** -21 * (scale * (q.abs() @ k.abs().t()) + lse.abs()) + 2.0 ** -20)
    err_delta = (dout * (out - o)).sum(-1, keepdim=True).abs() + 2.0 ** -20 * (dout.abs() * out.abs()).sum(-1, keepdim=True)
    err_ds = (u + 2.0 ** -20) * ds.abs() + err_p * (dp - delta).abs() + p * (err_delta + 2.0 ** -20 * (dout.abs() @ v.abs().t()))
    err_dv = (u + 2.0 ** -20) * p + err_p
    if dtype == torch.float16:
        err_dv = err_dv + 2.0 ** -39
        err_ds = err_ds + 2.0 ** -39 * 2 * dout.norm(dim=-1).max() * v.norm(dim=-1).max()
    tol_dq = scale * (err_ds @ k.abs() + err_ds.sum(-1, keepdim=True) * (p @ k.abs()))
    tol_dk = scale * err_ds.t() @ q.abs()
    return (dq, dk, dv), (tol_dq, tol_dk, err_dv.t() @ dout.abs())


def dense_grads(q, k, v, dout, out, scale, dtype, paired=False):
    """(B, H, L, D) tensors -> ((dq, dk, dv), bounds), in 64 bits on their device."""
    res = [torch.empty(t.shape, dtype=torch.float64, device=t.device) for t in (q, k, v, q, k, v)]
    for b in range(q.shape[0]):
        for h in range(q.shape[1]):
            g, t = head_grads(*(x[b, h].double() for x in (q, k, v, dout, out)), scale, dtype, paired=paired)
            for dst, src in zip(res, (*g, *t)):
                dst[b, h] = src
    return res[:3], res[3:]


def gather_grads(q, k, v, dout, out, gi, gl, perm, group_rows, scale, dtype):
    """(B, S, H, D) tensors, indices (B, H, M, K): the key set of a group is the multiset gi[b, h, m, :128 * gl]."""
    res = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, k, v, q, k, v)]
    B, Sq, H, _ = q.shape
    for b in range(B):
        for h in range(H):
            order = torch.arange(Sq, device=q.device) if perm is None else perm[b * H + h]
            for m in range(gi.shape[2]):
                rows = order[m * group_rows:(m + 1) * group_rows]
                n = gi.shape[3] if gl is None else 128 * min(max(int(gl[b, h, m]), 1), gi.shape[3] // 128)
                idx = gi[b, h, m, :n].long().clamp(0, k.shape[1] - 1)
                x = (q[b, rows, h], k[b, idx, h], v[b, idx, h], dout[b, rows, h], out[b, rows, h])
                g, t = head_grads(*(y.double() for y in x), scale, dtype)
                for i, (dst, src) in enumerate(zip(res, (*g, *t))):
                    if i % 3 == 0:
                        dst[b, rows, h] = src
                    else:
                        dst[b, :, h].index_add_(0, idx, src)
    return res[:3], res[3:]


def check_grads(got, grads, bounds, dtype, what=""):
    """Every element of the kernel's gradients within its bound and one rounding of the value; returns the largest share of it."""
    fi = torch.finfo(dtype)
    worst = 0.0
    for name, g, ref, tol in zip(("dq", "dk", "dv"), got, grads, bounds):
        assert g.dtype == dtype and g.shape == ref.shape, (what, name)
        limit = tol * (1 + fi.eps) + fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps / 2
        d = (g.double() - ref).abs()
        assert bool(torch.isfinite(g).all()), (what, name)
        share = float((d / limit).max()) if d.numel() else 0.0
        assert share <= 1.0, f"{what} {name}: {share:.3f} of the bound, largest error {float(d.max()):.3e}"
        worst = max(worst, share)
    return worst
