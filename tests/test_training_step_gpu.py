"""The training-side operators together, as an attention layer uses them: q and k are rotated on the video grid, the sparse call attends
on selected keys, a dense call on the text, both outputs are added, and the gradients run back through all of it."""

import math

import pytest
import torch

from mcsparse_b200.h3.ulysses_layer import rope_pairs
from mcsparse_b200.kernels.flash_mcsa.ops.flash_sparse_attn.cute import flash_attn_gather_kv_autograd_func
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_autograd
from mcsparse_b200.kernels.flash_mcsa.ops.rotary import RotaryEmbedding
from mcsparse_b200.kernels.flash_mcsa.pca_group import pca_group_perm
from mcsparse_b200.kernels.flash_mcsa.token_sparse import group_mass, select_topk_with_sinks
from mcsparse_b200.kernels.flash_mcsa.ops.full_attn import full_attention_with_lse

pytestmark = pytest.mark.gpu


def _inputs(device, dtype=torch.bfloat16):
    g = torch.Generator(device=device).manual_seed(3)
    F, Y, X, H, D, T = 4, 12, 14, 3, 128, 77
    L = F * Y * X
    mk = lambda n: torch.randn(1, n, H, D, generator=g, device=device).to(dtype)
    t = torch.arange(L, device=device)
    pos = torch.stack([t // (Y * X), t // X % Y, t % X], dim=-1)
    return dict(q=mk(L), k=mk(L), v=mk(L), tk=mk(T), tv=mk(T), dout=mk(L), pos=pos, L=L, H=H, D=D)


def test_layer_gradients(cuda_device):
    c = _inputs(cuda_device)
    rope = RotaryEmbedding(c["D"], axis_pairs=rope_pairs(c["D"]))
    leaves = {n: c[n].clone().requires_grad_(True) for n in ("q", "k", "v", "tk", "tv")}

    # the selection of this step: grouping, masses and token selection on detached tensors, as in an anchor step
    with torch.no_grad():
        rq, rk = (x.transpose(1, 2).contiguous() for x in rope(c["q"], c["k"], positions=c["pos"]))
        perm = pca_group_perm(rq[0], C=128).view(c["H"], c["L"])
        _, lse = full_attention_with_lse(rq, rk, c["v"].transpose(1, 2), perm=perm, group_order=True)
        mass = group_mass(rq, rk, lse, perm=perm)
        gi = select_topk_with_sinks(mass, 256, [(0, 4)])
    q, k = rope(leaves["q"], leaves["k"], positions=c["pos"])
    sparse = flash_attn_gather_kv_autograd_func(q, k, leaves["v"], gi, perm=perm)
    text = full_attention_autograd(q.transpose(1, 2), leaves["tk"].transpose(1, 2), leaves["tv"].transpose(1, 2)).transpose(1, 2)
    y = sparse + text
    got = torch.autograd.grad(y, list(leaves.values()), c["dout"])

    # the same in 64 bits
    ref = {n: c[n].double().requires_grad_(True) for n in leaves}
    n = len(rope.frequencies)
    ang = c["pos"].double()[:, list(rope.pair_axis)] * torch.tensor(rope.frequencies, dtype=torch.float64, device=cuda_device)
    cos, sin = torch.cos(ang)[None, :, None], torch.sin(ang)[None, :, None]

    def turn(x):
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    rq, rk = turn(ref["q"]), turn(ref["k"])
    outs = []
    for h in range(c["H"]):
        s = rq[0, :, h] @ rk[0, :, h].t() / math.sqrt(c["D"])
        member = torch.empty(c["L"], dtype=torch.int64, device=cuda_device)
        member[perm[h]] = torch.arange(c["L"], device=cuda_device) // 128
        seen = torch.zeros(gi.shape[2], c["L"], dtype=torch.bool, device=cuda_device).scatter_(1, gi[0, h].long(), True)
        o = torch.softmax(s.masked_fill(~seen[member], -math.inf), -1) @ ref["v"][0, :, h]
        o = o + torch.softmax(rq[0, :, h] @ ref["tk"][0, :, h].t() / math.sqrt(c["D"]), -1) @ ref["tv"][0, :, h]
        outs.append(o)
    want = torch.autograd.grad(torch.stack(outs, dim=1)[None], list(ref.values()), c["dout"].double())
    # Relative 2-norms.  Along the longest path a gradient is rounded to bf16 five times (operands P or dS, the attention's gradient, their sum over
    # both calls, the rotation, and the rotated inputs' rounding, which moves scores): each by at most 2^-8 of its values, so the
    # whole by at most 5 * 2^-8 of sums of magnitudes; those exceed the norm of a sum of n random terms by up to sqrt(n), but then the
    # roundings' own signs average the same way: 5 * 2^-8 of the norm with a factor 2 for scores (|s| < 8 here: e^(8 * 2^-8) - 1 < 2^-4.9).
    for name, a, b in zip(leaves, got, want):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 5 * 2.0 ** -8 * 2, (name, rel)
        assert a.dtype == torch.bfloat16 and a.shape == c[name].shape


def test_two_steps_at_once(cuda_device, monkeypatch):
    """The same step on two streams at the same time: workspaces are each call's own."""
    monkeypatch.setenv("MCSPARSE_B200_CHECK", "0")
    c = _inputs(cuda_device)
    gi = torch.stack([torch.randperm(c["L"], device=cuda_device)[:256].sort().values for _ in range(c["H"] * 6)]).view(1, c["H"], 6, 256).int()
    rope = RotaryEmbedding(c["D"], axis_pairs=rope_pairs(c["D"]))

    def step():
        q, k, v = (c[n].clone().requires_grad_(True) for n in ("q", "k", "v"))
        rq, rk = rope(q, k, positions=c["pos"])
        y = flash_attn_gather_kv_autograd_func(rq, rk, v, gi) + full_attention_autograd(rq.transpose(1, 2), rk.transpose(1, 2), v.transpose(1, 2)).transpose(1, 2)
        return torch.autograd.grad(y, [q, k, v], c["dout"])
    ref = step()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(step())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_in_place_rotation_is_seen_by_autograd(cuda_device):
    rope = RotaryEmbedding(64)
    x = torch.randn(1, 8, 2, 64, device=cuda_device)
    w = torch.randn(64, device=cuda_device, requires_grad=True)
    y = (x * w).sum()                                        # saves x
    rope.rotate(x, positions=torch.arange(8, device=cuda_device), inplace=True)
    with pytest.raises(RuntimeError):
        y.backward()
