"""GPU tests of rotary positions against the definition in 64 bits.

Tolerance.  A coefficient m cos w, m sin w of the kernel is off by at most: the angle, pi * (2^-25 + 2^-31) from its conversion to
32 bits; sincospif, 2 units in the last place of values up to 1, 2^-23; the product with the magnitude, 2^-24: together below
2^-21.6 m.  The product d s and the sum add 2^-24 of their values.  So an output is within 2^-21 m (|x_a| + |x_b|) of the
definition before its one rounding, which adds eps / 2 of the value (for subnormal results half their spacing).
"""

import math

import pytest
import torch

from mcsparse_b200.h3.ulysses_layer import qkv_norm_rope_scatter, rope_pairs, rope_table
from mcsparse_b200.kernels.flash_mcsa.ops.rotary import RotaryEmbedding

pytestmark = pytest.mark.gpu


def reference(plan, x, positions, inverse=False):
    """(value, bound of |x_a| + |x_b|) in 64 bits on the CPU."""
    x, positions = x.detach().cpu().double(), positions.cpu()
    n, axes = len(plan.frequencies), len(plan.axis_pairs)
    p = positions.unsqueeze(-1) if axes == 1 else positions
    if p.dim() == 2:
        p = p.unsqueeze(0)
    # the angle modulo one turn from integers: a 64-bit float product loses it at the farthest positions
    turns = [int(t) for t in plan._turns]
    ang = torch.tensor([[[2 * math.pi * ((int(v[plan.pair_axis[i]]) * turns[i]) % 2 ** 64) / 2 ** 64 for i in range(n)] for v in row]
                        for row in p.tolist()], dtype=torch.float64).view(p.shape[0], p.shape[1], 1, n)
    c, s = plan.magnitude * torch.cos(ang), plan.magnitude * torch.sin(ang)
    if inverse:
        s = -s
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if plan.layout == "interleaved" else (slice(0, n), slice(n, 2 * n))
    y, mass = x.clone(), torch.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    mass[..., a] = mass[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, mass * plan.magnitude


def check(plan, got, x, positions, inverse=False):
    ref, mass = reference(plan, x, positions, inverse)
    fi = torch.finfo(x.dtype)
    tol = 2.0 ** -21 * mass + fi.eps / 2 * (ref.abs() + 2.0 ** -21 * mass) + fi.smallest_normal * fi.eps / 2
    assert got.shape == x.shape and got.dtype == x.dtype
    d = (got.detach().cpu().double() - ref).abs()
    assert bool((d <= tol).all()), float((d / tol.clamp_min(1e-300)).max())
    n = 2 * len(plan.frequencies)
    assert torch.equal(got[..., n:].cpu(), x[..., n:].cpu())           # the rest of the head passes through


PLANS = {
    "whole": dict(head_dim=64),
    "half": dict(head_dim=64, layout="half"),
    "part": dict(head_dim=128, rotary_dim=64, layout="half"),
    "part_interleaved": dict(head_dim=144, rotary_dim=96),
    "odd_part": dict(head_dim=72, rotary_dim=20, layout="half"),       # single-element accesses
    "odd_interleaved": dict(head_dim=70, rotary_dim=34),
    "one_pair": dict(head_dim=8, rotary_dim=2),
    "grid": dict(head_dim=128, axis_pairs=rope_pairs(128)),
    "grid_half": dict(head_dim=96, axis_pairs=rope_pairs(96), layout="half"),
    "empty_axis": dict(head_dim=64, axis_pairs=(0, 32)),
    "linear": dict(head_dim=64, scaling="linear", factor=8.0),
    "ntk": dict(head_dim=64, scaling="ntk", factor=8.0, layout="half"),
    "yarn": dict(head_dim=128, scaling="yarn", factor=8.0, original_length=4096),
    "widest": dict(head_dim=256, layout="half"),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("name", sorted(PLANS))
def test_against_the_definition(cuda_device, name, dtype):
    plan = RotaryEmbedding(**PLANS[name])
    g = torch.Generator().manual_seed(len(name))
    axes = len(plan.axis_pairs)
    for B, L, Hq, Hk in [(1, 1, 1, 1), (2, 7, 3, 1), (1, 130, 20, 5)]:
        q = torch.randn(B, L, Hq, plan.head_dim, generator=g).to(dtype).to(cuda_device)
        k = torch.randn(B, L, Hk, plan.head_dim, generator=g).to(dtype).to(cuda_device)
        shape = (B, L) if axes == 1 else (B, L, axes)
        pos = torch.randint(-50, 1 << 20, shape, generator=g).to(cuda_device)
        y, z = plan.rotate(q, k, positions=pos)
        check(plan, y, q, pos)
        check(plan, z, k, pos)
        y, z = plan.rotate_backward(q, k, positions=pos.int())
        check(plan, y, q, pos, inverse=True)
        check(plan, z, k, pos, inverse=True)


def test_far_positions_and_position_layouts(cuda_device):
    plan = RotaryEmbedding(64)
    x = torch.randn(2, 6, 4, 64, device=cuda_device)
    far = torch.tensor([0, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31), 2 ** 40 + 3, -7], device=cuda_device)
    check(plan, plan.rotate(x, positions=far), x, far)                                  # (L,): shared by the batch
    check(plan, plan.rotate(x, positions=far.expand(2, 6)), x, far)                     # stride 0
    wide = torch.stack([far, far + 1, far * 0], dim=1).t().contiguous()                 # (3, L)
    grid = RotaryEmbedding(64, axis_pairs=(12, 10, 10))
    check(grid, grid.rotate(x, positions=wide.t()), x, wide.t())                        # axes not innermost
    near = torch.arange(12, device=cuda_device, dtype=torch.int32)[::2]
    check(plan, plan.rotate(x, positions=near), x, near)                                # every second element


def test_strides_and_alignment(cuda_device):
    plan = RotaryEmbedding(64, rotary_dim=32, layout="half")
    pos = torch.arange(33, device=cuda_device)
    packed = torch.randn(2, 33, 3, 4, 64, device=cuda_device).bfloat16()
    q, k = packed[:, :, 0], packed[:, :, 1]                                             # slices of a packed projection
    y, z = plan.rotate(q, k, positions=pos)
    check(plan, y, q, pos)
    check(plan, z, k, pos)
    heads_first = torch.randn(2, 4, 33, 64, device=cuda_device).bfloat16().transpose(1, 2)
    check(plan, plan.rotate(heads_first, positions=pos), heads_first, pos)
    base = torch.randn(2 * 33 * 4 * 64 + 1, device=cuda_device).bfloat16()
    odd = base[1:].view(2, 33, 4, 64)                                                   # 2-byte alignment
    check(plan, plan.rotate(odd, positions=pos), odd, pos)
    gaps = torch.randn(2, 33, 4, 67, device=cuda_device).bfloat16()[..., :64]           # odd strides
    check(plan, plan.rotate(gaps, positions=pos), gaps, pos)
    columns = torch.randn(2, 33, 64, 4, device=cuda_device).bfloat16().transpose(2, 3)  # rows not contiguous
    check(plan, plan.rotate(columns, positions=pos), columns, pos)
    same = torch.randn(1, 33, 1, 64, device=cuda_device).bfloat16().expand(2, 33, 4, 64)
    check(plan, plan.rotate(same, positions=pos), same, pos)


@pytest.mark.parametrize("name", ["whole", "part", "odd_part"])
def test_in_place(cuda_device, name):
    plan = RotaryEmbedding(**PLANS[name])
    pos = torch.arange(50, device=cuda_device)
    around = torch.randn(2, 52, 3, plan.head_dim, device=cuda_device)
    before = around.clone()
    x = around[:, 1:51]
    y = plan.rotate(x, positions=pos, inplace=True)
    assert y.data_ptr() == x.data_ptr()
    check(plan, x, before[:, 1:51], pos)
    assert torch.equal(around[:, 0], before[:, 0]) and torch.equal(around[:, 51], before[:, 51])
    assert torch.equal(x, plan.rotate(before[:, 1:51], positions=pos))
    with pytest.raises(ValueError):
        plan.rotate(before[:1].expand(2, 52, 3, plan.head_dim)[:, :50], positions=pos, inplace=True)
    with pytest.raises(ValueError):
        plan.rotate(x, x, positions=pos, inplace=True)


def test_gradient(cuda_device):
    """The gradient is the transposed rotation (checked against the definition above); here through autograd, for q alone, for
    both, and against differences of the forward pass in 32 bits."""
    plan = RotaryEmbedding(32, rotary_dim=24, layout="half", scaling="yarn", factor=4.0, original_length=128)
    pos = torch.tensor([3, 1000, 5], device=cuda_device)
    q = torch.randn(2, 3, 4, 32, device=cuda_device, requires_grad=True)
    k = torch.randn(2, 3, 2, 32, device=cuda_device, requires_grad=True)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    y, z = plan(q, k, positions=pos)
    dq, dk = torch.autograd.grad([y, z], [q, k], [gq, gk])
    check(plan, dq, gq, pos, inverse=True)
    check(plan, dk, gk, pos, inverse=True)
    (only,) = torch.autograd.grad(plan(q, k.detach(), positions=pos)[0].sum(), q)       # an expanded gradient from above
    check(plan, only, torch.ones_like(q), pos, inverse=True)
    # the map is linear: a central difference with step 1 is exact but for the roundings of its two sides, each within 2^-21 m
    # of 2 * 32 elements of size below 8 times a gradient below 6
    e = torch.zeros_like(q)
    e[1, 2, 3, 5] = 1.0
    with torch.no_grad():
        diff = ((plan(q + e, positions=pos) - plan(q - e, positions=pos)).double() * gq.double()).sum() / 2
    assert abs(float(diff) - float(dq[1, 2, 3, 5])) <= 2.0 ** -20 * plan.magnitude * 2 * 8 * 6 * 2


def test_empty_and_other_stream(cuda_device):
    plan = RotaryEmbedding(64)
    for shape in [(0, 4, 2, 64), (2, 0, 2, 64), (2, 4, 0, 64)]:
        x = torch.zeros(shape, device=cuda_device)
        assert plan.rotate(x, positions=torch.arange(shape[1], device=cuda_device)).shape == shape
    x, pos = torch.randn(1, 4000, 8, 64, device=cuda_device), torch.arange(4000, device=cuda_device)
    ref = plan.rotate(x, positions=pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = plan.rotate(x, positions=pos)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ref)


def test_captured(cuda_device, monkeypatch):
    monkeypatch.setenv("MCSPARSE_B200_CHECK", "0")          # the check synchronises, which a capture does not allow
    plan = RotaryEmbedding(128, axis_pairs=rope_pairs(128))
    q, k = (torch.randn(1, 60, 3, 128, device=cuda_device).bfloat16() for _ in range(2))
    pos = torch.randint(0, 50, (60, 3), device=cuda_device)
    plan.rotate(q, k, positions=pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = plan.rotate(q, k, positions=pos)
    q.normal_()
    pos.add_(7)
    graph.replay()
    torch.cuda.synchronize()
    check(plan, y, q, pos)
    check(plan, z, k, pos)


def test_same_rotation_as_the_projection_epilogue(cuda_device):
    """A grid plan turns a head as the fused epilogue of the context-parallel layer does: both round one fp32 value, whose tables
    (there) and angles (here) differ by at most 2^-21 of |x_a| + |x_b|; RMSNorm is made the identity up to its own rounding."""
    F, Hh, W, D = 3, 5, 4, 128
    L = F * Hh * W
    x = torch.randn(L, 2 * D, device=cuda_device)
    x = x.view(L, 2, D)
    x = (x / x.pow(2).mean(-1, keepdim=True).sqrt()).bfloat16().view(L, 2 * D)
    out = torch.empty(L, 2, D, dtype=torch.bfloat16, device=cuda_device)
    one = torch.ones(D, device=cuda_device)
    qkv_norm_rope_scatter(x, [out.data_ptr(), out.data_ptr() + 2 * D], [2 * D, 2 * D], [0, 1], one, one,
                          rope_table((F, Hh, W), D).to(cuda_device), (F, Hh, W), D, 0, 0, eps=0.0)
    t = torch.arange(L, device=cuda_device)
    pos = torch.stack([t // (Hh * W), t // W % Hh, t % W], dim=-1)
    mine = RotaryEmbedding(D, axis_pairs=rope_pairs(D)).rotate(x.view(1, L, 2, D), positions=pos)[0]
    # the row was scaled to a mean square of 1 before rounding to bf16, which moves it by at most 2^-8: the norm divides by a value
    # within 2^-8 of 1, and either side rounds to bf16 (2^-8 of a value of at most |x_a| + |x_b|)
    pairs = x.view(L, 2, D // 2, 2).float().abs().sum(-1).repeat_interleave(2, dim=-1)
    assert bool(((mine.float() - out.float()).abs() <= 3 * 2.0 ** -8 * pairs * 1.01).all())
