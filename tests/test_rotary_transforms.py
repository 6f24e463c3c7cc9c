"""Rotary positions under torch.func on the CPU."""
import torch

from kotflash_amd.rotary import Rotary


def test_transforms():
    rot = Rotary(16, device="cpu")
    q, t = (torch.randn(3, 2, 4, 5, 16, dtype=torch.float64, generator=torch.Generator().manual_seed(s)) for s in (0, 1))
    got = torch.vmap(lambda x: rot(x, positions=9))(q)
    assert all(torch.equal(got[i], rot(q[i], positions=9)) for i in range(3))
    out, tangent = torch.func.jvp(lambda x: rot(x, positions=9), (q[0],), (t[0],))
    assert torch.equal(out, rot(q[0], positions=9)) and torch.equal(tangent, rot(t[0], positions=9))
    back = torch.func.grad(lambda x: (rot(x, positions=9) * t[0]).sum())(q[0])
    leaf = q[0].clone().requires_grad_()
    want, = torch.autograd.grad(rot(leaf, positions=9), leaf, t[0])
    assert torch.equal(back, want)


def test_made_in_inference_mode():
    with torch.inference_mode():
        rot = Rotary(16, device="cpu")
    assert not rot.turns.is_inference()
    q = torch.randn(1, 2, 3, 16).requires_grad_()
    assert torch.autograd.grad(rot(q).sum(), q)[0].shape == q.shape
