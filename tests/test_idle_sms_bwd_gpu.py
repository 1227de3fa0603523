"""GPU tests of the dense attention's backward pass where the call leaves most SMs idle: P and dS are taken in two 16-bit parts there, however
long the axes, and the results meet bounds with the square of an operand's rounding (oracle/attn_bwd.py)."""

import pytest
import torch

from oracle.attn_bwd import check_grads, dense_grads
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward, full_attention_with_lse

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,Lq,Lk,D", [(2, 257, 257, 64), (2, 300, 300, 128), (1, 1000, 700, 128), (1, 2000, 128, 64), (1, 100, 4500, 128),
                                       (4, 130, 700, 96), (1, 600, 500, 144), (2, 260, 300, 256)])
def test_both_sums_in_two_parts(cuda_device, H, Lq, Lk, D, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(Lq + Lk)
    def mk(L):                                               # neighbouring tokens that resemble one another: the sums cancel
        x = torch.randn(1, H, 1, D, generator=g, device=cuda_device) + 0.3 * torch.randn(1, H, L, D, generator=g, device=cuda_device)
        return x.to(dtype)
    q, k, v = mk(Lq), mk(Lk), mk(Lk)
    dout = torch.randn(1, H, Lq, D, generator=g, device=cuda_device).to(dtype)
    out, lse = full_attention_with_lse(q, k, v)
    got = full_attention_backward(dout, q, k, v, out, lse)
    check_grads(got, *dense_grads(q, k, v, dout, out, D ** -0.5, dtype, paired=True), dtype, (H, Lq, Lk, D))
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(got, full_attention_backward(dout, q, k, v, out, lse)))
