"""CPU tests of the rotary plan: frequencies, fixed-point turns, refusals of the wrapper and of the C entry point."""

import ctypes as C
import math

import pytest
import torch

from mcsparse_b200 import _lib
from mcsparse_b200.kernels.flash_mcsa.ops import rotary as rotary_module
from mcsparse_b200.h3.ulysses_layer import rope_pairs
from mcsparse_b200.kernels.flash_mcsa.ops.rotary import RotaryEmbedding


def test_turns_are_frequencies_in_fixed_point():
    plan = RotaryEmbedding(128, axis_pairs=rope_pairs(128))
    assert plan.axis_pairs == (22, 21, 21) and len(plan._turns) == 64 and max(plan.pair_axis) == 2
    for t, f in zip(plan._turns, plan.frequencies):
        # both sides rounded once to 53 bits
        assert abs(t / 2 ** 64 - f / (2 * math.pi)) <= 2 ** -52 * f
    # a frequency of several turns per position keeps its part of a turn
    from mcsparse_b200.kernels.flash_mcsa.ops.rotary import _turns
    assert abs(_turns(10.0) / 2 ** 64 - (10.0 / (2 * math.pi)) % 1.0) < 1e-15
    # the integer product is the angle modulo one turn, far positions and negative ones included
    for pos in (1, 77, 10 ** 6, 2 ** 31 - 1, -5, -(2 ** 31)):
        turn = (pos * plan._turns[0]) % 2 ** 64 / 2 ** 64
        assert abs(math.cos(2 * math.pi * turn) - math.cos(float(pos))) < 1e-8


def test_scalings():
    base = RotaryEmbedding(64).frequencies
    n = 32
    assert base[0] == 1.0 and base[-1] == pytest.approx(10000.0 ** (-(n - 1) / n), rel=1e-14)
    linear = RotaryEmbedding(64, scaling="linear", factor=4.0).frequencies
    assert all(a == pytest.approx(b / 4.0, rel=1e-14) for a, b in zip(linear, base))
    ntk = RotaryEmbedding(64, scaling="ntk", factor=4.0).frequencies
    assert ntk[0] == 1.0
    # the lowest frequency, i = n - 1: theta'^-(n-1)/n = theta^-(n-1)/n * factor^-1
    assert ntk[-1] == pytest.approx(base[-1] / 4.0, rel=1e-12)
    yarn = RotaryEmbedding(64, scaling="yarn", factor=4.0, original_length=4096)
    turns = [4096 * f / (2 * math.pi) for f in base]
    for f, b, r in zip(yarn.frequencies, base, turns):
        if r >= 32:
            assert f == b
        elif r <= 1:
            assert f == pytest.approx(b / 4.0, rel=1e-14)
        else:
            assert b / 4.0 < f < b
    assert yarn.magnitude == pytest.approx(0.1 * math.log(4.0) + 1.0)
    assert RotaryEmbedding(64, scaling="yarn", factor=0.5, original_length=4096).magnitude == 1.0
    per_axis = RotaryEmbedding(128, axis_pairs=(22, 21, 21), scaling="linear", factor=(2.0, 1.0, 1.0))
    plain = RotaryEmbedding(128, axis_pairs=(22, 21, 21))
    assert per_axis.frequencies[0] == 0.5 and per_axis.frequencies[22:] == plain.frequencies[22:]


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=66), dict(rotary_dim=0), dict(axis_pairs=(10, 10)), dict(axis_pairs=(8, 8, 8, 8)),
                                dict(axis_pairs=(33, -1)), dict(layout="rows"), dict(scaling="other"), dict(theta=0.0), dict(theta=float("nan")),
                                dict(scaling="linear", factor=0.0), dict(scaling="linear", factor=(1.0, 2.0)),
                                dict(scaling="yarn", factor=2.0), dict(scaling="yarn", original_length=10, beta_fast=1.0),
                                dict(magnitude=float("inf"))])
def test_plan_refusals(kw):
    with pytest.raises(ValueError):
        RotaryEmbedding(64, **kw)


def test_call_refusals():
    plan, grid = RotaryEmbedding(64), RotaryEmbedding(64, axis_pairs=(12, 10, 10))
    x, pos = torch.zeros(2, 5, 3, 64), torch.arange(5)
    bad = [
        (ValueError, plan, (x[0],), pos), (ValueError, plan, (x[..., :32],), pos), (ValueError, plan, (x, x, x), pos),
        (ValueError, plan, (), pos), (ValueError, plan, (x, x[:, :4]), pos), (TypeError, plan, (x.double(),), pos),
        (TypeError, plan, (x, x.half()), pos), (TypeError, plan, (x,), pos.float()), (ValueError, plan, (x,), pos[:4]),
        (ValueError, plan, (x,), pos.view(1, 1, 5)), (ValueError, plan, (x,), torch.zeros(3, 5, dtype=torch.int64)),
        (ValueError, grid, (x,), pos), (ValueError, grid, (x,), torch.zeros(5, 2, dtype=torch.int64)),
        (RuntimeError, plan, (x,), pos), (RuntimeError, grid, (x,), torch.zeros(2, 5, 3, dtype=torch.int32)),
    ]
    for err, p, tensors, positions in bad:
        with pytest.raises(err):
            p.rotate(*tensors, positions=positions)
        with pytest.raises(err):
            p.rotate_backward(*tensors, positions=positions)
    with pytest.raises(RuntimeError):                       # in place is forward-only
        plan.rotate(x.clone().requires_grad_(True), positions=pos, inplace=True)


def test_entry_point_refusals():
    """Validation happens before any CUDA call: the addresses below are never touched."""
    lib = _lib.lib()
    assert lib.mcs_rotary(None, None) == -1
    turns, axis = (C.c_uint64 * 32)(), (C.c_uint8 * 32)()

    def args(**kw):
        a = _lib.RotaryArgs()
        a.x[0] = a.y[0] = 0x1000
        a.positions, a.turns, a.axis = 0x1000, turns, axis
        a.H[0], a.B, a.L, a.D, a.n_pairs, a.n_axes, a.magnitude, a.pos64 = 4, 1, 8, 64, 32, 1, 1.0, 1
        for k, v in kw.items():
            setattr(a, k, v)
        return a
    for code, kw in [(-2, dict(B=-1)), (-2, dict(n_axes=0)), (-2, dict(n_axes=4)), (-3, dict(n_pairs=0)), (-3, dict(n_pairs=33)), (-3, dict(D=0)),
                     (-3, dict(n_pairs=129, D=300)), (-9, dict(layout=2)), (-4, dict(dtype=2)), (-6, dict(magnitude=float("nan"))),
                     (-1, dict(positions=None)), (-5, dict(positions=0x1004)), (0, dict(L=0)), (0, dict(B=0))]:
        assert lib.mcs_rotary(args(**kw), None) == code, kw
    a = args()
    a.x[0] = None
    assert lib.mcs_rotary(a, None) == -1
    a = args()
    a.x[0] = 0x1001
    assert lib.mcs_rotary(a, None) == -5
    a = args()
    axis[3] = 1
    assert lib.mcs_rotary(a, None) == -2                    # a pair on an axis that does not exist
    axis[3] = 0
    a = args()
    a.H[0] = 0
    assert lib.mcs_rotary(a, None) == 0


def test_results_have_contiguous_rows_whatever_the_input():
    """Windows of a sequence (a stride of one twice): memory in the input's order of strides would put the window, not the head, last."""
    x = torch.zeros(1000)
    for shape, stride in [((1, 2, 4, 16), (0, 100, 1, 1)), ((2, 4, 2, 16), (300, 1, 64, 1)), ((2, 4, 2, 16), (300, 64, 16, 1))]:
        t = x.as_strided(shape, stride)
        y = rotary_module._memory_like(t)
        assert y.shape == t.shape and y.stride(3) == 1 and not rotary_module._overlaps_itself(y)
    t = torch.zeros(2, 3, 5, 16).transpose(1, 2)
    assert rotary_module._memory_like(t).stride() == t.stride()


def test_tensors_that_share_elements_are_told_from_slices_of_one_projection():
    """Against sets of element offsets, over slices of packed projections and shifted views."""
    base = torch.zeros(4000)

    def offsets(t):
        at = t.storage_offset() + sum(torch.arange(n).view([-1 if i == d else 1 for i in range(4)]) * s for d, (n, s) in enumerate(zip(t.shape, t.stride())))
        return set(at.flatten().tolist())
    packed, heads = base[:2 * 5 * 7 * 8].view(2, 5, 7, 8), base[:2 * 6 * 5 * 8].view(2, 6, 5, 8).transpose(1, 2)
    three = base[:2 * 5 * 3 * 2 * 8].view(2, 5, 3, 2, 8)
    apart = [(packed[:, :, :4], packed[:, :, 4:6]), (packed[:, :, 5:], packed[:, :, :3]), (heads[:, :, :3], heads[:, :, 3:]), (packed[:1], packed[1:]),
             (three[:, :, 0], three[:, :, 1]), (three[:, :, 2], three[:, :, 0]), (packed[:, :, :, :4], packed[:, :, :, 4:]),
             (packed[:, :4, :4], packed[:, 1:, 4:]), (packed[:, :, :1], packed[:, :, 1:]), (packed[:, :, :0], packed), (base[:320].view(2, 5, 4, 8), base[320:640].view(2, 5, 4, 8))]
    share = [(packed, packed), (packed[:, :, :4], packed[:, :, 3:]), (packed[:, :4], packed[:, 1:]), (packed[:, :, :4], packed[:, :, 2:6]),
             (heads[:, :, :3], heads[:, :, 2:5]), (packed[..., :5], packed[..., 3:]), (base[:320].view(2, 5, 4, 8), base[8:328].view(2, 5, 4, 8)),
             (base[:320].view(2, 5, 4, 8), base[:320].view(2, 4, 5, 8).transpose(1, 2))]
    for a, b in apart:
        assert not offsets(a) & offsets(b)
        assert not rotary_module._may_share(a, b) and not rotary_module._may_share(b, a)
    for a, b in share:
        assert offsets(a) & offsets(b)
        assert rotary_module._may_share(a, b) and rotary_module._may_share(b, a)
    # never missed, whatever the strides
    g = torch.Generator().manual_seed(0)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=g))
    for _ in range(600):
        shape = [(1 + pick(3), 1 + pick(4), 1 + pick(3), 4) for _ in range(2)]
        strides = (pick(60), pick(30), pick(16), 1)
        a, b = (base.as_strided(s, strides, pick(80)) for s in shape)
        if rotary_module._overlaps_itself(a) or rotary_module._overlaps_itself(b):
            continue
        if offsets(a) & offsets(b):
            assert rotary_module._may_share(a, b), (a.shape, b.shape, strides, a.storage_offset(), b.storage_offset())


def test_plan_is_copied_and_stored_with_a_module():
    import copy
    import pickle
    plan = RotaryEmbedding(32, rotary_dim=16, axis_pairs=(4, 4), layout="half", scaling="linear", factor=2.0)
    for other in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert list(other._turns) == list(plan._turns) and list(other._axis) == list(plan._axis)
        assert C.addressof(other._turns) != C.addressof(plan._turns)
        assert other.frequencies == plan.frequencies and other.layout == plan.layout and other.magnitude == plan.magnitude
