"""Rotary positions under torch.func and forward-mode gradients: what the kernel
does not take, ``auto`` runs in torch operations, and ``hip`` refuses."""
import pytest
import torch
from torch.autograd import forward_ad

from kotflash_amd.rotary import Rotary

pytestmark = pytest.mark.gpu


def _randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half().cuda()


@pytest.fixture
def rot():
    return Rotary(64, device="cuda")


def test_vmap(rot):
    q, k = _randn(3, 2, 4, 5, 64), _randn(3, 2, 2, 5, 64, seed=1)
    got = torch.vmap(lambda a, b: rot(a, b, positions=9))(q, k)
    for i in range(3):
        want = rot(q[i], k[i], positions=9, backend="torch")
        assert all(torch.equal(g[i], w) for g, w in zip(got, want))
    # Positions alone are mapped.
    n = torch.tensor([[1, 5], [70, 9]], device="cuda")
    got = torch.vmap(lambda p: rot(q[0], positions=p))(n)
    assert all(torch.equal(got[i], rot(q[0], positions=n[i], backend="torch")) for i in range(2))


def test_grad(rot):
    q, g = _randn(2, 4, 5, 64), _randn(2, 4, 5, 64, seed=1)
    got = torch.func.grad(lambda x: (rot(x, positions=9) * g).sum())(q)
    leaf = q.clone().requires_grad_()
    want, = torch.autograd.grad(rot(leaf, positions=9, backend="torch"), leaf, g)
    assert torch.equal(got, want)


def test_forward_mode(rot):
    """Linear: the tangent is turned as the value is."""
    q, t = _randn(2, 4, 5, 64), _randn(2, 4, 5, 64, seed=1)
    want = rot(q, positions=9, backend="torch"), rot(t, positions=9, backend="torch")
    got = torch.func.jvp(lambda x: rot(x, positions=9), (q,), (t,))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with forward_ad.dual_level():
        out = forward_ad.unpack_dual(rot(forward_ad.make_dual(q, t), positions=9))
        assert torch.equal(out.primal, want[0]) and torch.equal(out.tangent, want[1])
        k = forward_ad.make_dual(q, t)
        assert torch.equal(forward_ad.unpack_dual(rot(q, k, positions=9)[1]).tangent, want[1])


def test_hip_refuses(rot):
    q, t = _randn(2, 4, 5, 64), _randn(2, 4, 5, 64, seed=1)
    with pytest.raises(RuntimeError, match="backend='torch'"):
        torch.vmap(lambda x: rot(x, backend="hip"))(q[None])
    with pytest.raises(RuntimeError, match="backend='torch'"):
        torch.func.jvp(lambda x: rot(x, backend="hip"), (q,), (t,))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="backend='torch'"):
        rot(forward_ad.make_dual(q, t), backend="hip")


def test_made_in_inference_mode():
    with torch.inference_mode():
        made = Rotary(64, device="cuda")
    q, g = _randn(2, 4, 5, 64).requires_grad_(), _randn(2, 4, 5, 64, seed=1)
    dq, = torch.autograd.grad(made(q, positions=9), q, g)
    assert torch.equal(dq, torch.autograd.grad(Rotary(64, device="cuda")(q, positions=9), q, g)[0])
