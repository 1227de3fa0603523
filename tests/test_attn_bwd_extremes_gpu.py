"""GPU tests of the attention's backward passes where rows are not finite or far larger than the rest: what takes no part in a sum
must not change it.  Results are compared bit for bit with those of the same call without these rows."""

import math

import pytest
import torch

from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_backward_func, flash_attn_gather_kv_func
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward, full_attention_with_lse

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.inf, math.nan, 60000.0])
def test_keys_that_no_group_selects(cuda_device, value, dtype):
    """Rows of k and v outside every list hold anything.  (fp16 operands of dS are scaled by the largest rows of dout and v.)"""
    B, S, H, D, K, M = 1, 600, 2, 64, 128, 5
    g = torch.Generator(device=cuda_device).manual_seed(0)
    q, k, v, dout = (torch.randn(B, S, H, D, generator=g, device=cuda_device).to(dtype) for _ in range(4))
    q, dout = q * 4, dout * 16
    gi = torch.rand(B, H, M, S // 2, generator=g, device=cuda_device).argsort(-1)[..., :K].sort(-1).values.int() * 2     # even keys only
    out, lse = flash_attn_gather_kv_func(q, k, v, gi, return_lse=True)
    k, v = k.clone(), v.clone()
    k[:, 1::2], v[:, 1::2] = 0, 0
    want = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi)
    k[:, 1::2], v[:, 1::2] = value, value
    got = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi)
    for a, b in zip(got, want):
        assert bool(b.isfinite().all()) and torch.equal(a, b)
    assert not got[1][:, 1::2].any() and not got[2][:, 1::2].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_one_row_of_dout_is_not_finite(cuda_device, value, dtype):
    """The overflow of a scaled loss shows in dk and dv and in that row of dq; the other rows and the other head keep their bits."""
    B, H, L, D = 1, 2, 300, 64
    g = torch.Generator(device=cuda_device).manual_seed(1)
    q, k, v, dout = (torch.randn(B, H, L, D, generator=g, device=cuda_device).to(dtype) for _ in range(4))
    q, dout = q * 4, dout * 16
    out, lse = full_attention_with_lse(q, k, v)
    dout[0, 1, 7] = 0
    want = full_attention_backward(dout, q, k, v, out, lse)
    dout[0, 1, 7, 3] = value
    got = full_attention_backward(dout, q, k, v, out, lse)
    assert bool(torch.stack([t.isfinite().all() for t in want]).all())
    for a, b in zip(got, want):
        assert torch.equal(a[0, 0], b[0, 0])
    others = torch.arange(L, device=cuda_device) != 7
    assert torch.equal(got[0][0, 1, others], want[0][0, 1, others])
    assert not bool(got[0][0, 1, 7].isfinite().any())
    assert not bool(got[1][0, 1].isfinite().all()) and not bool(got[2][0, 1].isfinite().all())
