"""GPU tests of the attention's backward kernels where a CTA walks many short items: neighbouring items share barriers, row sums and tensor
memory.  Gradients against 64 bits with the bounds of oracle/attn_bwd.py, and the same bits from every launch."""

import pytest
import torch

from oracle.attn_bwd import check_grads, dense_grads, gather_grads
from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_backward_func, flash_attn_gather_kv_func
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("most", [1, 2, 5])
@pytest.mark.parametrize("D", [64, 96, 128, 144, 192, 256])
def test_gathered_lists_of_few_tiles(cuda_device, D, most, dtype):
    """Lists of 1 to `most` tiles: the warps that copy rows cross from item to item at every position of their turn."""
    g = torch.Generator(device=cuda_device).manual_seed(D + most)
    B, H, Sq, Sk, rows = 2, 6, 3000, 700, 50
    M = Sq // rows
    mk = lambda L: torch.randn(B, L, H, D, generator=g, device=cuda_device).to(dtype)
    q, k, v, dout = mk(Sq), mk(Sk), mk(Sk), mk(Sq)
    gi = torch.rand(B, H, M, Sk, generator=g, device=cuda_device).argsort(dim=-1)[..., :128 * most].int().contiguous()
    gl = torch.randint(1, most + 1, (B, H, M), generator=g, device=cuda_device, dtype=torch.int32)
    kw = dict(gather_kv_lengths=gl, group_rows=rows)
    out, lse = flash_attn_gather_kv_func(q, k, v, gi, return_lse=True, **kw)
    first = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi, **kw)
    check_grads(first, *gather_grads(q, k, v, dout, out, gi, gl, None, rows, D ** -0.5, dtype), dtype, (D, most))
    for _ in range(REPEATS):
        again = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi, **kw)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
