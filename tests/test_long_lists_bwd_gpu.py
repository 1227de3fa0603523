"""GPU test of the gather-KV attention's backward pass at the package's large shape (98,280 tokens, 768 groups) with lists of 8,192 keys: one
head's contributions take 6.4 GB, so offsets inside them pass 32 bits."""

import pytest
import torch

from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_backward_func, flash_attn_gather_kv_func

pytestmark = pytest.mark.gpu


def test_offsets_that_pass_32_bits(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(0)
    B, H, S, D, K, rows = 1, 2, 98280, 128, 8192, 128
    M = -(-S // rows)
    scale = D ** -0.5
    u, e = torch.finfo(torch.bfloat16).eps / 2, 2.0 ** -20
    q, k, v, dout = (torch.randn(B, S, H, D, generator=g, device=cuda_device).bfloat16() for _ in range(4))
    gi = torch.empty(B, H, M, K, dtype=torch.int32, device=cuda_device)
    for h in range(H):
        for m in range(M):
            gi[0, h, m] = torch.randperm(S, generator=g, device=cuda_device)[:K].sort().values
    gi[..., -1] = S - 1                                      # (a key that every group selects)
    out, lse = flash_attn_gather_kv_func(q, k, v, gi, return_lse=True)
    grads = flash_attn_gather_kv_backward_func(dout, q, k, v, out, lse, gi)
    # the second head alone: another place in every tensor, the same bits
    one = lambda t: t[:, :, 1:2].contiguous()
    alone = flash_attn_gather_kv_backward_func(one(dout), one(q), one(k), one(v), one(out), lse[:, 1:].contiguous(), gi[:, 1:].contiguous())
    for a, b in zip(grads, alone):
        assert torch.equal(a[:, :, 1:2], b)
    # a few keys from the definition in 64 bits, P from the given lse; bounds as in oracle/attn_bwd.py, with the error of lse beside
    for h in range(H):
        x, d, o = q[0, :, h].double(), dout[0, :, h].double(), out[0, :, h].double()
        delta = (d * o).sum(-1)
        # (delta's own error: the kernel takes it from the rounded out and corrects it by the row's sum of dS; |dout| |out - exact| either way)
        err_delta = (u + e) * (d.abs() * o.abs()).sum(-1)
        for key in (0, 1, 40000, S - 2, S - 1):
            named = (gi[0, h] == key).any(-1).repeat_interleave(rows)[:S]
            assert key != S - 1 or bool(named.all())
            kj, vj, L = k[0, key, h].double(), v[0, key, h].double(), lse[0, h].double()
            p = torch.exp(scale * x @ kj - L) * named
            err_p = p * (2 * e * (scale * x.abs() @ kj.abs() + L.abs()) + 2 * e)
            dp = d @ vj
            ds = p * (dp - delta)
            err_ds = (u + e) * ds.abs() + err_p * (dp - delta).abs() + p * (2 * err_delta + e * (d.abs() @ vj.abs()))
            for got, want, tol in ((grads[1], scale * ds @ x, scale * err_ds @ x.abs()), (grads[2], p @ d, ((u + e) * p + err_p) @ d.abs())):
                got = got[0, key, h].double()
                limit = tol * (1 + 2 * u) + u * want.abs()
                assert bool(((got - want).abs() <= limit).all()), (h, key, float(((got - want).abs() / limit).max()))
