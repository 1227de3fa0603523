"""GPU tests of the attention's backward kernels where a CTA walks many short items: neighbouring items share barriers, row sums and tensor
memory.  Gradients against 64 bits with the bounds of oracle/attn_bwd.py, and the same bits from every launch."""

import pytest
import torch

from oracle.attn_bwd import check_grads, dense_grads
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward, full_attention_with_lse

pytestmark = pytest.mark.gpu

REPEATS = 20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Lk", [(128, 40), (128, 100), (64, 64), (64, 128), (144, 20), (144, 32), (256, 30)])
def test_dense_items_of_one_tile(cuda_device, D, Lk, dtype):
    """Keys that fit one streamed tile: every item of the query side has one."""
    g = torch.Generator(device=cuda_device).manual_seed(D + Lk)
    mk = lambda L: torch.randn(2, 12, L, D, generator=g, device=cuda_device).to(dtype)
    q, k, v, dout = mk(2100), mk(Lk), mk(Lk), mk(2100)
    out, lse = full_attention_with_lse(q, k, v)
    first = full_attention_backward(dout, q, k, v, out, lse)
    check_grads(first, *dense_grads(q, k, v, dout, out, D ** -0.5, dtype), dtype, (D, Lk))
    for _ in range(REPEATS):
        assert all(torch.equal(a, b) for a, b in zip(first, full_attention_backward(dout, q, k, v, out, lse)))
