"""GPU tests of the dense attention's backward pass against the gradients in 64 bits, with the bounds that oracle/attn_bwd.py
derives from the kernel's roundings."""

import math

import pytest
import torch

from oracle.attn_bwd import check_grads, dense_grads
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import (full_attention, full_attention_autograd, full_attention_backward,
                                                            full_attention_with_lse)

pytestmark = pytest.mark.gpu


def make(B, H, Lq, Lk, D, dtype, device, seed=0, sharp=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    mk = lambda L: torch.randn(B, L, H, D, generator=g, device=device).to(dtype).transpose(1, 2)
    q, k, v, dout = mk(Lq), mk(Lk), mk(Lk), mk(Lq)
    return q * sharp, k, v, dout


def run(q, k, v, dout, scale=None, what=""):
    out, lse = full_attention_with_lse(q, k, v, scale)
    got = full_attention_backward(dout, q, k, v, out, lse, scale)
    s = 1.0 / math.sqrt(q.shape[3]) if scale is None else scale
    check_grads(got, *dense_grads(q, k, v, dout, out, s, q.dtype), q.dtype, what)
    return out, lse, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 64, 96, 144, 256, 8, 72, 136, 192])
def test_head_dimensions(cuda_device, D, dtype):
    for i, (B, H, Lq, Lk) in enumerate([(1, 1, 128, 128), (1, 2, 130, 257), (2, 3, 300, 190)]):
        run(*make(B, H, Lq, Lk, D, dtype, cuda_device, seed=i), what=(B, H, Lq, Lk))


@pytest.mark.parametrize("D", [128, 144, 64])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 2), (2, 1), (1, 128), (1, 129), (127, 1), (129, 3), (64, 64), (65, 63), (3, 1000), (1000, 3), (513, 640)])
def test_lengths(cuda_device, Lq, Lk, D):
    _, _, (dq, dk, _) = run(*make(1, 3, Lq, Lk, D, torch.bfloat16, cuda_device, seed=Lq + Lk))
    if Lk == 1:
        assert not dq.any() and not dk.any()                 # softmax over one key does not depend on the scores


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (144, torch.bfloat16)])
def test_many_items_per_sm(cuda_device, D, dtype):
    """More tiles than SMs, so that a CTA walks several items of either kernel; and few keys or few queries, so that the summed axis is
    split."""
    run(*make(2, 24, 700, 900, D, dtype, cuda_device))
    run(*make(1, 2, 5000, 200, D, dtype, cuda_device))
    run(*make(1, 2, 200, 5000, D, dtype, cuda_device))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sharp_rows_scales_and_magnitudes(cuda_device, dtype):
    q, k, v, dout = make(1, 2, 400, 500, 128, dtype, cuda_device, sharp=6.0)
    run(q, k, v, dout, what="sharp")
    run(q, k, v, dout, scale=0.01, what="flat")
    # gradients far from 1 (a loss that is scaled, or not): fp16 operands have to hold them
    run(q / 6, k, v, dout * 2.0 ** 9, what="large gradients")
    run(q / 6, k, v * 2.0 ** 6, dout * 2.0 ** -8, what="small gradients")
    run(q / 6, k, v, dout * 0, what="no gradient")
    run(q, k * 0, v, dout, what="equal scores")


def test_long_rows_in_fp16(cuda_device):
    """Probabilities of 1 / 30,000 are far below fp16's normal range; they are taken times 2^14."""
    run(*make(1, 1, 130, 30000, 64, torch.float16, cuda_device))
    run(*make(1, 1, 30000, 130, 64, torch.float16, cuda_device))


def test_layouts(cuda_device):
    B, H, L, D = 2, 3, 200, 64
    g = torch.Generator(device=cuda_device).manual_seed(5)
    packed = torch.randn(B, L, 3, H, D, generator=g, device=cuda_device).bfloat16()
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))                        # slices of a packed projection
    dout = torch.randn(B, H, L, D, generator=g, device=cuda_device).bfloat16()           # heads first
    _, _, got = run(q, k, v, dout)
    for t, x in zip(got, (q, k, v)):
        assert t.shape == x.shape
    out, lse = full_attention_with_lse(q, k, v)
    ref = full_attention_backward(dout, q, k, v, out, lse)
    columns = dout.transpose(2, 3).contiguous().transpose(2, 3)                          # rows not contiguous
    shifted = torch.empty(dout.numel() + 1, dtype=dout.dtype, device=cuda_device)[1:].view(dout.shape).copy_(dout)   # 2-byte address
    for d in (columns, shifted):
        for a, b in zip(full_attention_backward(d, q, k, v, out, lse), ref):
            assert torch.equal(a, b)
    ones = torch.ones((), dtype=torch.bfloat16, device=cuda_device).expand(B, H, L, D)   # the gradient of a sum
    run(q, k, v, ones)
    one_head = q[:, :1].expand(B, H, L, D)                                               # q shared by the heads
    run(one_head, k, v, dout)


def test_same_bits_every_time(cuda_device):
    for shape in [(1, 4, 3000, 2000, 128), (1, 2, 4000, 100, 64), (1, 2, 100, 4000, 144)]:
        q, k, v, dout = make(*shape, torch.bfloat16, cuda_device)
        out, lse = full_attention_with_lse(q, k, v)
        first = full_attention_backward(dout, q, k, v, out, lse)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, full_attention_backward(dout, q, k, v, out, lse)))


def test_autograd(cuda_device):
    q, k, v, dout = (t.detach() for t in make(1, 2, 150, 170, 128, torch.bfloat16, cuda_device))
    out, lse = full_attention_with_lse(q, k, v)
    want = full_attention_backward(dout, q, k, v, out, lse)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y = full_attention_autograd(*leaves)
    assert torch.equal(y, out) and torch.equal(y, full_attention(q, k, v))
    got = torch.autograd.grad(y, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # only one input needs a gradient; an input that broadcasts sums its gradient over the copies
    kk = k[:, :1].clone().requires_grad_(True)
    (dk,) = torch.autograd.grad(full_attention_autograd(q, kk.expand(k.shape), v), kk, dout)
    full = full_attention_backward(dout, q, kk.detach().expand(k.shape), v, *full_attention_with_lse(q, kk.detach().expand(k.shape), v))
    assert torch.equal(dk, full[1].sum(1, keepdim=True))
    with pytest.raises(RuntimeError):                        # once differentiable
        (dq,) = torch.autograd.grad(full_attention_autograd(*leaves), leaves[0], dout.clone().requires_grad_(True), create_graph=True)
        torch.autograd.grad(dq.float().sum(), leaves[1])


def test_against_differences(cuda_device):
    """The gradient against central differences of the definition in 64 bits: step h, error h^2/6 of a third derivative that is far below
    10 here, so 1e-6 beside the bound of the kernel."""
    q, k, v, dout = make(1, 1, 5, 7, 64, torch.float16, cuda_device)
    out, lse, got = run(q, k, v, dout)
    grads, bounds = dense_grads(q, k, v, dout, out, 0.125, torch.float16)
    x = [t[0, 0].double() for t in (q, k, v)]
    f = lambda a, b, c: float((torch.softmax(0.125 * a @ b.t(), -1) @ c * dout[0, 0].double()).sum())
    for i in range(3):
        for r, c in [(0, 0), (4, 63), (2, 17)]:
            e = torch.zeros_like(x[i])
            e[r, c] = 1e-3
            diff = (f(*[t + e if j == i else t for j, t in enumerate(x)]) - f(*[t - e if j == i else t for j, t in enumerate(x)])) / 2e-3
            tol = 1e-5 + float(bounds[i][0, 0, r, c]) + 2.0 ** -11 * abs(diff)
            assert abs(diff - float(got[i][0, 0, r, c])) <= tol


def test_other_stream_and_capture(cuda_device, monkeypatch):
    monkeypatch.setenv("MCSPARSE_B200_CHECK", "0")
    q, k, v, dout = make(1, 4, 600, 500, 128, torch.float16, cuda_device)
    out, lse = full_attention_with_lse(q, k, v)
    ref = full_attention_backward(dout, q, k, v, out, lse)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = full_attention_backward(dout, q, k, v, out, lse)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = full_attention_backward(dout, q, k, v, out, lse)
    with torch.cuda.graph(other):
        second = full_attention_backward(dout * 2, q, k, v, out, lse)
    for _ in range(2):
        other.replay()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, ref))
    # twice the gradient is exactly twice everywhere (powers of two) but where fp16 results are subnormal
    for a, b in zip(second, ref):
        normal = b.abs() >= torch.finfo(torch.float16).smallest_normal
        assert torch.equal(a[normal], 2 * b[normal])


def test_neighbouring_memory_is_left_alone(cuda_device):
    """Gradients are written into exactly their rows: the C entry point on slices of larger buffers."""
    from mcsparse_b200.kernels.flash_mcsa.ops import attn_bwd
    for D, Lq, Lk in [(64, 130, 70), (96, 70, 130), (144, 65, 129)]:
        q, k, v, dout = (t.transpose(1, 2).contiguous() for t in make(1, 2, Lq, Lk, D, torch.bfloat16, cuda_device))
        out, lse = full_attention_with_lse(*(t.transpose(1, 2) for t in (q, k, v)))
        big = [torch.full((t.shape[0], t.shape[1] + 2, t.shape[2] + 2, D + 16), 7.0, dtype=t.dtype, device=cuda_device) for t in (q, k, v)]
        views = [b[:, 1:-1, 1:-1, 8:D + 8] for b in big]
        attn_bwd.launch_backward("mcs_dense_attn_bwd", dout, q, k, v, out.transpose(1, 2), lse, *views, D ** -0.5)
        ref = full_attention_backward(*(t.transpose(1, 2) for t in (dout, q, k, v)), out, lse)
        for b, w, r in zip(big, views, ref):
            assert torch.equal(w, r.transpose(1, 2))
            w.fill_(7.0)
            assert bool((b == 7.0).all())
