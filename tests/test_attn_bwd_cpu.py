"""CPU tests of the attention gradients' refusals (wrappers and C entry points), workspace sizes, and of the bounds' arithmetic."""

import ctypes as C

import pytest
import torch

from mcsparse_b200 import _lib
from mcsparse_b200.kernels.flash_mcsa.ops import attn_bwd
from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_backward_func
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward
from oracle.attn_bwd import head_grads


def dense_args(B=1, H=2, Lq=5, Lk=7, D=64, dtype=torch.bfloat16):
    mk = lambda L: torch.zeros(B, H, L, D, dtype=dtype)
    return dict(dout=mk(Lq), q=mk(Lq), k=mk(Lk), v=mk(Lk), out=mk(Lq), lse=torch.zeros(B, H, Lq))


def test_dense_refusals():
    ok = dense_args()
    bad = [
        (ValueError, dict(q=ok["q"][0])), (ValueError, dict(k=ok["k"][:, :1])), (ValueError, dict(v=ok["v"][:, :, :3])),
        (ValueError, dict(k=ok["k"][..., :32], v=ok["v"][..., :32])), (TypeError, dict(q=ok["q"].float())), (TypeError, dict(k=ok["k"].half())),
        (ValueError, dict(dout=ok["dout"][:, :, :2])), (ValueError, dict(dout=ok["dout"].float())), (ValueError, dict(out=ok["out"].half())),
        (ValueError, dict(lse=ok["lse"].double())), (ValueError, dict(lse=ok["lse"][:, :1])), (RuntimeError, dict()),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            full_attention_backward(**{**ok, **kw})
    for D in (4, 68, 264):                                   # head dimensions that no kernel takes
        with pytest.raises(ValueError):
            full_attention_backward(**dense_args(D=D))
    for sizes in (dict(B=0), dict(H=0), dict(Lq=0), dict(Lk=0)):
        with pytest.raises(ValueError):
            full_attention_backward(**dense_args(**sizes))


def test_gather_refusals():
    B, S, H, D, K = 1, 300, 2, 64, 128
    mk = lambda: torch.zeros(B, S, H, D, dtype=torch.bfloat16)
    ok = dict(dout=mk(), q=mk(), k=mk(), v=mk(), out=mk(), lse=torch.zeros(B, H, S), gather_kv_indices=torch.zeros(B, H, 3, K, dtype=torch.int32))
    gi = ok["gather_kv_indices"]
    bad = [
        (TypeError, dict(q=mk().float())), (TypeError, dict(v=mk().half())), (ValueError, dict(k=mk()[:, :, :1])),
        (ValueError, dict(gather_kv_indices=gi[:, :, :2])), (ValueError, dict(gather_kv_indices=gi[..., :64])), (TypeError, dict(gather_kv_indices=gi.long())),
        (ValueError, dict(gather_kv_indices=torch.zeros(B, H, 3, 512, dtype=torch.int32))), (ValueError, dict(group_rows=0)), (ValueError, dict(group_rows=129)),
        (ValueError, dict(group_rows=64)), (TypeError, dict(gather_kv_lengths=torch.zeros(B, H, 3))),
        (ValueError, dict(gather_kv_lengths=torch.zeros(B, H, 2, dtype=torch.int32))), (TypeError, dict(perm=torch.zeros(B * H, S))),
        (ValueError, dict(perm=torch.zeros(B * H, S + 1, dtype=torch.int64))), (ValueError, dict(lse=torch.zeros(B, S, H))),
        (ValueError, dict(out=mk()[:, :5])), (ValueError, dict(dout=mk().float())), (RuntimeError, dict()),
    ]
    for err, kw in bad:
        with pytest.raises(err):
            flash_attn_gather_kv_backward_func(**{**ok, **kw})


def raw(**kw):
    a = _lib.AttnBwdArgs()
    for name in ("q", "k", "v", "out", "dout", "lse", "dq", "dk", "dv", "workspace", "status", "gi"):
        setattr(a, name, 0x10000)                            # never touched: every call below is refused on the host
    a.gi = None
    a.B, a.Sq, a.Sk, a.H, a.D, a.softmax_scale, a.gather_len, a.group_rows = 1, 256, 256, 2, 64, 0.125, 128, 128
    a.workspace_bytes = 1 << 40
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_entry_point_refusals():
    lib = _lib.lib()
    assert lib.mcs_dense_attn_bwd(None, None) == -1 and lib.mcs_dense_attn_bwd_workspace_bytes(None) == -1
    common = [(-2, dict(B=0)), (-2, dict(Sq=0)), (-2, dict(Sk=-1)), (-3, dict(D=4)), (-3, dict(D=260)), (-3, dict(D=257)), (-4, dict(dtype=2)),
              (-6, dict(softmax_scale=0.0)), (-6, dict(softmax_scale=float("inf"))), (-9, dict(flags=1)), (-10, dict(H=70000)),
              (-1, dict(q=None)), (-1, dict(dv=None)), (-1, dict(lse=None)), (-1, dict(workspace=None)), (-5, dict(dout=0x10008)),
              (-5, dict(workspace=0x10010)), (-7, dict(workspace_bytes=100))]
    for code, kw in common + [(-9, dict(perm=0x10000)), (-9, dict(gi=0x10000)), (-10, dict(Sq=2 ** 31 - 1))]:
        assert lib.mcs_dense_attn_bwd(raw(**kw), None) == code, kw
    for code, kw in common + [(-1, dict(gi=None)), (-2, dict(gather_len=64)), (-2, dict(gather_len=0)), (-2, dict(group_rows=0)), (-2, dict(group_rows=129)),
                              (-10, dict(Sq=1 << 20, group_rows=1, gather_len=4096))]:
        assert lib.mcs_gather_attn_bwd(raw(**{"gi": 0x10000, **kw}), None) == code, kw
    a = raw()
    a.dk_stride[1] = 4
    assert lib.mcs_dense_attn_bwd(a, None) == -5


def test_workspace_sizes():
    lib = _lib.lib()
    # the DiT layer: enough tiles for every SM, so only the rows' statistics (3 floats per row, 64 pairs of maxima per head)
    assert lib.mcs_dense_attn_bwd_workspace_bytes(raw(Sq=32760, Sk=32760, H=24, D=128)) == 24 * (3 * 32768 * 4 + 64 * 8)
    # few keys, many queries: partial sums of the split queries on top
    assert lib.mcs_dense_attn_bwd_workspace_bytes(raw(Sq=32760, Sk=512, H=1, D=128)) > 4 * 2 * 512 * 2 * 128
    # gather: the contributions of as many heads at a time as fit 4 GiB, at least one head's
    per_head = 256 * 2048 * 2 * 128 * 4
    one = lib.mcs_gather_attn_bwd_workspace_bytes(raw(Sq=32760, Sk=32760, H=1, D=128, gather_len=2048))
    many = lib.mcs_gather_attn_bwd_workspace_bytes(raw(Sq=32760, Sk=32760, H=24, D=128, gather_len=2048))
    assert per_head < one < 1.1 * per_head and 7 * per_head <= many < 1.1 * (4 << 30)
    long = lib.mcs_gather_attn_bwd_workspace_bytes(raw(Sq=98280, Sk=98280, H=5, D=128, gather_len=9856))
    assert 768 * 9856 * 1024 < long < 1.2 * 768 * 9856 * 1024


def test_layouts_that_the_kernels_read_in_place():
    x = torch.zeros(2, 6, 3, 64, dtype=torch.bfloat16)
    for t in (x, x.transpose(1, 2), x[:, 1:5], x[:, :, 1:], x.transpose(0, 2), torch.zeros(2, 6, 3, 3, 64, dtype=torch.bfloat16)[:, :, 1]):
        assert attn_bwd.readable(t) is t
    for t in (x[:1].expand(2, 6, 3, 64), x[:, :, :1].expand(2, 6, 3, 64), x.transpose(2, 3).contiguous().transpose(2, 3),
              torch.zeros(2 * 6 * 3 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 6, 3, 64), torch.zeros(2, 6, 3, 68, dtype=torch.bfloat16)[..., :64],
              x.as_strided((2, 6, 3, 64), (64, 64, 64, 1))):
        c = attn_bwd.readable(t)
        assert c is not t and c.is_contiguous() and torch.equal(c, t)
    assert attn_bwd.gradient_like(x.transpose(1, 2)).stride() == x.transpose(1, 2).stride()
    assert attn_bwd.gradient_like(x.transpose(2, 3)).is_contiguous()


def test_oracle_gradients_by_autograd():
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(n, 16, generator=g, dtype=torch.float64) for n in (5, 9, 9, 5))
    hide = torch.rand(5, 9, generator=g) < 0.3
    hide[:, 0] = False
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = torch.softmax((0.25 * leaves[0] @ leaves[1].t()).masked_fill(hide, float("-inf")), -1) @ leaves[2]
    want = torch.autograd.grad(out, leaves, dout)
    grads, bounds = head_grads(q, k, v, dout, out.detach(), 0.25, torch.bfloat16, hide)
    for a, b, t in zip(grads, want, bounds):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12) and bool((t > 0).any())


def test_gradients_have_contiguous_rows_whatever_the_input():
    x = torch.zeros(1000, dtype=torch.bfloat16)
    for shape, stride in [((1, 2, 4, 16), (0, 104, 1, 1)), ((2, 4, 2, 16), (304, 1, 64, 1)), ((2, 4, 2, 16), (304, 16, 16, 1))]:
        y = attn_bwd.gradient_like(x.as_strided(shape, stride))
        assert y.shape == shape and y.stride(3) == 1 and all(s % 8 == 0 for s in y.stride()[:3])
