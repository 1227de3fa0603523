"""GPU tests of the gather-KV attention's backward pass against the gradients in 64 bits, with the bounds that oracle/attn_bwd.py
derives from the kernel's roundings."""

import math

import pytest
import torch

from oracle.attn_bwd import check_grads, gather_grads
from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import (PackedIndices, flash_attn_gather_kv_autograd_func,
                                                                         flash_attn_gather_kv_backward_func, flash_attn_gather_kv_func)
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_backward, full_attention_with_lse

pytestmark = pytest.mark.gpu


def make(B, H, Sq, Sk, D, K, dtype, device, rows=128, perm=False, lengths=False, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    mk = lambda L: torch.randn(B, L, H, D, generator=g, device=device).to(dtype)
    M = math.ceil(Sq / rows)
    # K different keys each, the first four in every list (K may exceed Sk by the tail of its last tile: those repeat)
    order = torch.rand(B, H, M, Sk, generator=g, device=device)
    order[..., :4] = -1.0
    gi = order.argsort(dim=-1)[..., :K].sort(dim=-1).values.int()
    gi = gi[..., torch.arange(K, device=device) % gi.shape[-1]]
    gl = torch.randint(0, K // 128 + 2, (B, H, M), generator=g, device=device, dtype=torch.int32) if lengths else None
    pm = torch.stack([torch.randperm(Sq, generator=g, device=device) for _ in range(B * H)]) if perm else None
    return dict(q=mk(Sq), k=mk(Sk), v=mk(Sk), dout=mk(Sq), gi=gi.contiguous(), gl=gl, perm=pm, rows=rows)


def run(c, scale=None, what=""):
    kw = dict(gather_kv_lengths=c["gl"], perm=c["perm"], group_rows=c["rows"])
    out, lse = flash_attn_gather_kv_func(c["q"], c["k"], c["v"], c["gi"], softmax_scale=scale, return_lse=True, **kw)
    got = flash_attn_gather_kv_backward_func(c["dout"], c["q"], c["k"], c["v"], out, lse, c["gi"], scale, **kw)
    s = c["q"].shape[3] ** -0.5 if scale is None else scale
    check_grads(got, *gather_grads(c["q"], c["k"], c["v"], c["dout"], out, c["gi"], c["gl"], c["perm"], c["rows"], s, c["q"].dtype), c["q"].dtype, what)
    return out, lse, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [128, 64, 96, 144, 256, 8, 72, 136, 192])
def test_head_dimensions(cuda_device, D, dtype):
    run(make(1, 1, 128, 256, D, 128, dtype, cuda_device), what="one tile")
    run(make(1, 2, 300, 500, D, 256, dtype, cuda_device, perm=True, seed=1), what="permuted")
    run(make(2, 2, 260, 700, D, 384, dtype, cuda_device, rows=64, perm=True, lengths=True, seed=2), what="lengths")


@pytest.mark.parametrize("Sq,Sk,K,rows", [(1, 1, 128, 128), (1, 300, 128, 128), (129, 127, 128, 128), (130, 130, 256, 128), (257, 128, 128, 128),
                                          (70, 200, 128, 1), (70, 200, 256, 33), (513, 1000, 640, 127)])
def test_sizes(cuda_device, Sq, Sk, K, rows):
    for D in (128, 144):
        run(make(1, 2, Sq, Sk, D, K, torch.bfloat16, cuda_device, rows=rows, perm=Sq > 100, seed=Sq))


def test_many_groups(cuda_device):
    run(make(2, 12, 1500, 900, 128, 256, torch.bfloat16, cuda_device, perm=True))
    run(make(1, 6, 4000, 600, 64, 256, torch.float16, cuda_device, rows=64, lengths=True))


def test_keys_that_every_group_or_none_selects(cuda_device):
    """One key in every list (more entries than one warp sums), lists that are all alike, keys in no list, lists of one key."""
    c = make(1, 2, 100 * 16, 500, 64, 128, torch.bfloat16, cuda_device, rows=16)
    run(c, what="sinks of 100 groups")
    c["gi"][:] = c["gi"][:, :, :1].clone()
    _, _, (_, dk, dv) = run(c, what="equal lists")
    unused = torch.ones(500, dtype=torch.bool, device=cuda_device)
    unused[c["gi"][0, 0, 0].long()] = False
    assert unused.any() and not dk[0, unused, 0].any() and not dv[0, unused, 0].any()
    c["gi"][:] = 7                                           # one key, 128 times in each list
    run(c, what="one key")
    c["gi"][0, :, ::2, :64] = 499
    run(c, what="two keys")


def test_indices_outside_are_clamped_as_in_the_forward_pass(cuda_device):
    c = make(1, 2, 200, 300, 128, 256, torch.bfloat16, cuda_device)
    c["gi"][0, 0, 0, :3] = -5
    c["gi"][0, 1, 1, 250:] = 1 << 30
    run(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_magnitudes(cuda_device, dtype):
    c = make(1, 2, 300, 500, 128, 256, dtype, cuda_device, perm=True)
    run(dict(c, q=c["q"] * 6), what="sharp")
    run(c, scale=0.01, what="flat")
    run(dict(c, dout=c["dout"] * 2.0 ** 9), what="large gradients")
    run(dict(c, v=c["v"] * 2.0 ** 6, dout=c["dout"] * 2.0 ** -8), what="small gradients")
    run(dict(c, dout=c["dout"] * 0), what="no gradient")


def test_all_keys_selected_is_the_dense_gradient(cuda_device):
    """Every group lists every key in order: dq has the dense call's bits (the same products in the same order); dk and dv agree within the
    roundings that oracle/attn_bwd.py bounds."""
    c = make(1, 2, 256, 256, 128, 256, torch.bfloat16, cuda_device)
    c["gi"][:] = torch.arange(256, device=cuda_device, dtype=torch.int32)
    out, lse, got = run(c)
    t = lambda x: x.transpose(1, 2)
    dense = full_attention_backward(t(c["dout"]), t(c["q"]), t(c["k"]), t(c["v"]), t(out), lse)
    grads, bounds = gather_grads(c["q"], c["k"], c["v"], c["dout"], out, c["gi"], None, None, 128, 128 ** -0.5, torch.bfloat16)
    check_grads([t(x) for x in dense], grads, bounds, torch.bfloat16)


def test_layouts_and_packed_indices(cuda_device):
    c = make(1, 3, 260, 300, 64, 256, torch.bfloat16, cuda_device, perm=True)
    out, lse, ref = run(c)
    kw = dict(perm=c["perm"])
    heads_first = {n: c[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v", "dout")}
    got = flash_attn_gather_kv_backward_func(heads_first["dout"], heads_first["q"], heads_first["k"], heads_first["v"], out, lse, c["gi"], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    got = flash_attn_gather_kv_backward_func(c["dout"], c["q"], c["k"], c["v"], out, lse, PackedIndices.pack(c["gi"]), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    spread = torch.empty(1, 3, 3, 512, dtype=torch.int32, device=cuda_device)[..., :256].copy_(c["gi"])
    columns = c["dout"].transpose(2, 3).contiguous().transpose(2, 3)
    got = flash_attn_gather_kv_backward_func(columns, c["q"], c["k"], c["v"], out, lse, spread, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    run(dict(c, dout=torch.ones((), dtype=torch.bfloat16, device=cuda_device).expand(c["q"].shape)))


def test_same_bits_every_time(cuda_device):
    for D in (64, 144):
        c = make(1, 4, 3000, 1000, D, 384, torch.bfloat16, cuda_device, perm=True, rows=64)
        out, lse, first = run(c)
        for _ in range(3):
            again = flash_attn_gather_kv_backward_func(c["dout"], c["q"], c["k"], c["v"], out, lse, c["gi"], perm=c["perm"], group_rows=64)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_autograd(cuda_device):
    c = make(1, 2, 260, 300, 128, 256, torch.bfloat16, cuda_device, perm=True, lengths=True)
    out, lse, want = run(c)
    for gi in (c["gi"], PackedIndices.pack(c["gi"])):
        leaves = [c[n].clone().requires_grad_(True) for n in ("q", "k", "v")]
        y = flash_attn_gather_kv_autograd_func(*leaves, gi, gather_kv_lengths=c["gl"], perm=c["perm"])
        assert torch.equal(y, out)
        got = torch.autograd.grad(y, leaves, c["dout"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    y = flash_attn_gather_kv_autograd_func(*leaves, c["gi"], gather_kv_lengths=c["gl"], perm=c["perm"])
    c["gi"].add_(0)                                          # overwritten before the backward pass
    with pytest.raises(RuntimeError):
        y.backward(c["dout"])


def test_other_stream_and_capture(cuda_device, monkeypatch):
    monkeypatch.setenv("MCSPARSE_B200_CHECK", "0")
    c = make(1, 4, 700, 900, 128, 256, torch.float16, cuda_device, perm=True)
    out, lse = flash_attn_gather_kv_func(c["q"], c["k"], c["v"], c["gi"], return_lse=True, perm=c["perm"])
    call = lambda d: flash_attn_gather_kv_backward_func(d, c["q"], c["k"], c["v"], out, lse, c["gi"], perm=c["perm"])
    ref = call(c["dout"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(c["dout"])
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    captured = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            captured.append(call(c["dout"]))
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got in captured:
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    # new selections in the captured call's own tensor
    c["gi"].copy_(c["gi"].flip(2))
    graphs[0].replay()
    torch.cuda.synchronize()
    # (out and lse stay those of the old lists: only the launch is checked)
    assert all(torch.equal(a, b) for a, b in zip(captured[0], call(c["dout"])))


def test_neighbouring_memory_is_left_alone(cuda_device):
    from mcsparse_b200.kernels.flash_mcsa.ops import attn_bwd
    for D in (64, 96, 144):
        c = make(1, 2, 200, 300, D, 256, torch.bfloat16, cuda_device, perm=True)
        out, lse, ref = run(c)
        big = [torch.full((t.shape[0], t.shape[1] + 2, t.shape[2] + 2, D + 16), 7.0, dtype=t.dtype, device=cuda_device) for t in (c["q"], c["k"], c["v"])]
        views = [b[:, 1:-1, 1:-1, 8:D + 8] for b in big]
        attn_bwd.launch_backward("mcs_gather_attn_bwd", c["dout"], c["q"], c["k"], c["v"], out, lse, *views, D ** -0.5, c["gi"], None, c["perm"])
        for b, w, r in zip(big, views, ref):
            assert torch.equal(w, r)
            w.fill_(7.0)
            assert bool((b == 7.0).all())


def test_entries_of_perm_out_of_range_take_no_part(cuda_device):
    """Bounds-checked in every kernel that follows perm: nothing outside the tensors is read or written."""
    c = make(1, 2, 300, 400, 64, 128, torch.bfloat16, cuda_device, perm=True)
    kw = dict(gather_kv_lengths=c["gl"], group_rows=c["rows"])
    out, lse = flash_attn_gather_kv_func(c["q"], c["k"], c["v"], c["gi"], return_lse=True, perm=c["perm"], **kw)
    gone, bad = c["perm"][:, 5].clone(), c["perm"].clone()
    bad[0, 5], bad[1, 5] = 300, -1
    dout = c["dout"].clone()
    for h in range(2):
        dout[0, gone[h], h] = 0                              # a row without gradient from above adds nothing to dk and dv
    want = flash_attn_gather_kv_backward_func(dout, c["q"], c["k"], c["v"], out, lse, c["gi"], perm=c["perm"], **kw)
    got = flash_attn_gather_kv_backward_func(c["dout"], c["q"], c["k"], c["v"], out, lse, c["gi"], perm=bad, **kw)
    for h in range(2):
        others = torch.arange(300, device=cuda_device) != gone[h]
        assert torch.equal(got[0][0, others, h], want[0][0, others, h])
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
