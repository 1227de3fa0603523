"""GPU tests of the dense attention's backward pass over short axes, where P and dS are taken in two 16-bit parts: bounds with the square of
an operand's rounding (oracle/attn_bwd.py), which single parts would not meet."""

import math

import pytest
import torch

from oracle.attn_bwd import check_grads, dense_grads
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward, full_attention_with_lse

pytestmark = pytest.mark.gpu


def make(B, H, Lq, Lk, D, dtype, device, seed):
    """Neighbouring tokens that resemble one another: the sums cancel."""
    g = torch.Generator(device=device).manual_seed(seed)
    def mk(L):
        x = torch.randn(B, H, 1, D, generator=g, device=device) + 0.3 * torch.randn(B, H, L, D, generator=g, device=device)
        return x.to(dtype)
    return mk(Lq), mk(Lk), mk(Lk), torch.randn(B, H, Lq, D, generator=g, device=device).to(dtype)


# (up to 64 rows one or two tiles; the last three several)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 144, 256, 8, 72])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (7, 33), (33, 7), (32, 33), (64, 64), (63, 32), (65, 64), (130, 90), (256, 256)])
def test_both_axes_short(cuda_device, Lq, Lk, D, dtype):
    q, k, v, dout = make(1, 2, Lq, Lk, D, dtype, cuda_device, seed=Lq + 300 * Lk)
    out, lse = full_attention_with_lse(q, k, v)
    got = full_attention_backward(dout, q, k, v, out, lse)
    check_grads(got, *dense_grads(q, k, v, dout, out, 1 / math.sqrt(D), dtype, paired=True), dtype, (Lq, Lk, D))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 144])
def test_one_axis_short(cuda_device, D, dtype):
    """Only the sums over the short axis have the smaller bound: dq over keys, dk and dv over queries."""
    for Lq, Lk, exact in ((40, 3000, (1, 2)), (3000, 40, (0,)), (1, 5000, (1, 2)), (5000, 1, (0,))):
        q, k, v, dout = make(2, 12, Lq, Lk, D, dtype, cuda_device, seed=Lq + Lk)
        out, lse = full_attention_with_lse(q, k, v)
        got = full_attention_backward(dout, q, k, v, out, lse)
        s = 1 / math.sqrt(D)
        grads, wide = dense_grads(q, k, v, dout, out, s, dtype)
        _, close = dense_grads(q, k, v, dout, out, s, dtype, paired=True)
        check_grads(got, grads, [close[i] if i in exact else wide[i] for i in range(3)], dtype, (Lq, Lk, D))
