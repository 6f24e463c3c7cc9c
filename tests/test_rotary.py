"""Rotary positions on the CPU: frequencies, the torch path against the
definition in 64 bits, gradients, refusals."""
import math

import pytest
import torch

from kotflash_amd.rotary import Rotary, rotary_frequencies
from tests.rotary_oracle import assert_turned, turned64


def _randn(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def test_frequencies():
    f = rotary_frequencies(8, base=100.0)
    assert f == pytest.approx([1, 100 ** -0.25, 0.1, 100 ** -0.75])
    assert rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0) == pytest.approx([x / 4 for x in f])
    stretched = rotary_frequencies(8, base=100.0, scaling="base", factor=4.0)
    assert stretched[0] == 1 and stretched[-1] == pytest.approx(f[-1] / 4)
    # 2 pi 16 positions: the pairs turn 16, 16 * 100^-0.25, 1.6 and 0.506 times.
    n = round(2 * math.pi * 16)
    ramp = rotary_frequencies(8, base=100.0, scaling="ramp", factor=4.0, original_length=n)
    w = (n * f[2] / (2 * math.pi) - 1) / 3
    assert ramp == pytest.approx([f[0], f[1], f[2] * w + f[2] / 4 * (1 - w), f[3] / 4])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(64, 64), (72, 40), (6, 2)])
def test_against_definition(dtype, interleaved, d, r):
    rot = Rotary(d, rotary_dim=r, interleaved=interleaved, amplitude=1.25, device="cpu")
    q, k = _randn(2, 4, 5, d, dtype=dtype), _randn(2, 2, 5, d, dtype=dtype, seed=1)
    for positions in (0, 3, 10 ** 6, torch.tensor([7, 123456]), torch.tensor([[0, 9, 2, 5, 5]], dtype=torch.int32)):
        for x, y in zip((q, k), rot(q, k, positions=positions)):
            assert y.dtype == dtype and y.is_contiguous()
            assert_turned(y, x, rot, positions)
    assert torch.equal(rot(q, positions=3), rot(q, k, positions=3)[0])


def test_far_and_negative_positions():
    """Angles by exact integers: positions beyond 2^31 and before the origin."""
    rot = Rotary(32, device="cpu")
    q = _randn(1, 1, 3, 32, dtype=torch.float64)
    for n in (2 ** 31 + 5, 2 ** 40 + 1, -1, -70000):
        assert_turned(rot(q, positions=n), q, rot, n)
    there = rot(q, positions=12345)
    back = rot(there, positions=torch.tensor([[-12345, -12346, -12347]]))
    assert (back - q).abs().max() < 1e-12


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(interleaved):
    rot = Rotary(8, rotary_dim=4, interleaved=interleaved, amplitude=0.5, device="cpu")
    q, k = (_randn(1, h, 3, 8, dtype=torch.float64).requires_grad_() for h in (2, 1))
    assert torch.autograd.gradcheck(lambda a, b: rot(a, b, positions=5), (q, k))
    # Heads that share their keys: the gradient of an expanded input is the sum.
    shared = _randn(1, 1, 3, 8, dtype=torch.float64).requires_grad_()
    g = _randn(1, 4, 3, 8, dtype=torch.float64, seed=2)
    got, = torch.autograd.grad(rot(shared.expand(1, 4, 3, 8)), shared, g)
    back = turned64(g.sum(1, keepdim=True), rot, 0, inverse=True)
    assert (got - back).abs().max() < 1e-12


@pytest.mark.parametrize("kw,error,match", [
    (dict(head_dim=0), ValueError, "head_dim"), (dict(rotary_dim=3), ValueError, "even"),
    (dict(rotary_dim=0), ValueError, "even"), (dict(rotary_dim=66), ValueError, "exceed"),
    (dict(base=1.0), ValueError, "base"), (dict(base=math.inf), ValueError, "base"),
    (dict(scaling="log"), ValueError, "one of"), (dict(factor=2.0), ValueError, "factor"),
    (dict(scaling="linear", factor=0.5), ValueError, "factor"),
    (dict(scaling="linear", factor=math.nan), ValueError, "factor"),
    (dict(scaling="base", factor=2.0, rotary_dim=2), ValueError, "more than one pair"),
    (dict(scaling="ramp", factor=2.0), ValueError, "original_length"),
    (dict(scaling="ramp", factor=2.0, original_length=100, slow_turns=4.0), ValueError, "slow_turns"),
    (dict(interleaved=1), TypeError, "interleaved"), (dict(amplitude=math.inf), ValueError, "amplitude"),
    (dict(frequencies=[1.0]), ValueError, "rotary_dim / 2"), (dict(frequencies=[4.0] * 32), ValueError, "below pi"),
])
def test_constructor_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        Rotary(**{"head_dim": 64, "device": "cpu", **kw})


def test_call_refusals():
    rot = Rotary(64, device="cpu")
    q, k = _randn(2, 4, 3, 64), _randn(2, 2, 3, 64)
    for args, kw, error, match in [
        (([1], k), {}, TypeError, "q must be a torch.Tensor"), ((q, "k"), {}, TypeError, "k must be a torch.Tensor"),
        ((q[0], k), {}, ValueError, "layout"), ((q.long(), None), {}, TypeError, "floating"),
        ((q[:, :0], k), {}, ValueError, "non-empty"), ((q, k[:, :0]), {}, ValueError, "k must have"),
        ((q[..., :32], k), {}, ValueError, "head_dim 64"), ((q, k[:, :, :2]), {}, ValueError, "k must have"),
        ((q, k.half()), {}, ValueError, "same dtype"), ((q, k), dict(positions=1.5), TypeError, "positions"),
        ((q, k), dict(positions=True), TypeError, "positions"), ((q, k), dict(positions=2 ** 62), ValueError, "2\\*\\*62"),
        ((q, k), dict(positions=torch.zeros(2)), ValueError, "int32 or int64"),
        ((q, k), dict(positions=torch.zeros(3, dtype=torch.int64)), ValueError, "shape"),
        ((q, k), dict(positions=torch.zeros(3, 3, dtype=torch.int64)), ValueError, "shape"),
        ((q, k), dict(backend="cuda"), ValueError, "backend"), ((q, k), dict(backend="hip"), RuntimeError, "gfx950"),
    ]:
        with pytest.raises(error, match=match):
            rot(*args, **kw)


def test_compiles_to_one_graph():
    rot = Rotary(16, device="cpu")
    f = torch.compile(lambda q, k: rot(q, k, positions=4), fullgraph=True, backend="eager")
    q, k = _randn(1, 2, 3, 16), _randn(1, 1, 3, 16)
    assert all(torch.equal(a, b) for a, b in zip(f(q, k), rot(q, k, positions=4)))


def test_op_registration():
    """Shapes and types of the op's outputs without running it."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import kotflash_amd.ops  # noqa: F401

    with FakeTensorMode():
        q, k = torch.empty(2, 4, 3, 64, dtype=torch.float16).transpose(1, 2), torch.empty(2, 3, 2, 64).half()
        turns = torch.empty(32, dtype=torch.int64)
        a, b = torch.ops.kotflash_amd.rotary(q, k, turns, None, 5, False, False, 1.0)
    assert a.shape == q.shape and b.shape == k.shape and a.is_contiguous() and a.dtype == torch.float16
