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


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (96, torch.float16), (144, torch.bfloat16)])
def test_rows_of_dq_that_perm_does_not_name_are_zero(cuda_device, D, dtype):
    """Entries of perm out of range, and a row named twice: the rows left over have no gradient, whatever their memory held."""
    from mcsparse_b200.kernels.flash_mcsa.ops import attn_bwd
    g = torch.Generator(device=cuda_device).manual_seed(D)
    B, H, S = 2, 2, 300
    q, k, v, dout = (torch.randn(B, S, H, D, generator=g, device=cuda_device).to(dtype) for _ in range(4))
    gi = torch.rand(B, H, 3, S, generator=g, device=cuda_device).argsort(dim=-1)[..., :128].int().contiguous()
    perm = torch.stack([torch.randperm(S, generator=g, device=cuda_device) for _ in range(B * H)])
    out, lse = flash_attn_gather_kv_func(q, k, v, gi, return_lse=True, perm=perm)
    want = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi, perm=perm)
    left = perm[:, [5, 140, 299]].clone()
    bad = perm.clone()
    bad[:, 5], bad[:, 140], bad[:, 299] = S, -1, perm[:, 298]
    big = torch.full((B, S + 2, H + 2, D + 16), float("nan"), dtype=dtype, device=cuda_device)
    dq = big[:, 1:-1, 1:-1, 8:D + 8]
    attn_bwd.launch_backward("mcs_gather_attn_bwd", dout, q, k, v, out, lse, dq, torch.empty_like(k), torch.empty_like(v), D ** -0.5, gi, None, bad)
    for bh in range(B * H):
        b, h = divmod(bh, H)
        assert bool((dq[b, left[bh], h] == 0).all())
        others = torch.ones(S, dtype=torch.bool, device=cuda_device)
        others[left[bh]] = False
        others[perm[bh, 298]] = False                        # (named twice)
        assert torch.equal(dq[b, others, h], want[0][b, others, h])
    dq.fill_(float("nan"))
    assert bool(big.isnan().all())                           # nothing beside the rows was written


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (144, torch.bfloat16)])
def test_dq_of_full_lists_has_the_dense_bits(cuda_device, D, dtype):
    """Every group lists every key in order, and the dense call neither splits the keys nor takes its operands in two parts: the same products
    in the same order."""
    g = torch.Generator(device=cuda_device).manual_seed(D)
    B, H, Sq, Sk = 1, 12, 1500, 512
    mk = lambda L: torch.randn(B, L, H, D, generator=g, device=cuda_device).to(dtype)
    q, k, v, dout = mk(Sq), mk(Sk), mk(Sk), mk(Sq)
    gi = torch.arange(Sk, device=cuda_device, dtype=torch.int32).expand(B, H, 12, Sk).contiguous()
    heads = lambda x: x.transpose(1, 2)
    out, lse = full_attention_with_lse(heads(q), heads(k), heads(v))
    dense = full_attention_backward(heads(dout), heads(q), heads(k), heads(v), out, lse)
    got = flash_attn_gather_kv_backward_func(dout, q, k, v, heads(out), lse, gi)
    assert torch.equal(heads(dense[0]), got[0])
