"""The rotary kernel on the GPU, against the definition in 64 bits."""
import pytest
import torch

import kotflash_amd.ops  # noqa: F401
from kotflash_amd import attention
from kotflash_amd.rotary import Rotary, _HipRotary
from tests.rotary_oracle import assert_turned, turned64

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _randn(*shape, dtype=F16, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _check(rot, q, k, positions=0, **kw):
    out = rot(q, k, positions=positions, backend="hip", **kw)
    where = positions.cpu() if isinstance(positions, torch.Tensor) else positions
    for x, y in zip((q, k), out):
        assert y.is_contiguous()
        assert_turned(y, x, rot, where)
    return out


# head_dim, rotary_dim: whole 16-byte pieces (16 | rotary_dim, 8 | head_dim),
# odd pieces behind, and what the plain kernel takes.
DIMS = [(128, 128), (64, 64), (96, 96), (128, 64), (72, 16), (72, 64), (80, 32), (16, 16), (256, 256), (1024, 1024),
        (128, 8), (64, 6), (7, 2), (100, 100), (72, 72), (2048, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", DIMS)
def test_dims(dtype, interleaved, d, r):
    rot = Rotary(d, rotary_dim=r, interleaved=interleaved, amplitude=1.25)
    _check(rot, _randn(2, 4, 5, d, dtype=dtype), _randn(2, 2, 5, d, dtype=dtype, seed=1), positions=1000)


@pytest.mark.parametrize("b,hq,hk,s", [(1, 1, 1, 1), (1, 1, 3, 1), (3, 32, 8, 1), (2, 7, 1, 33), (64, 8, 2, 1),
                                       (1, 40, 8, 900), (2, 71, 5, 100), (1, 16, 4, 2500)])
@pytest.mark.parametrize("d", [64, 96])
def test_shapes(b, hq, hk, s, d):
    """One wave per token and few heads, up to four times as many heads."""
    rot = Rotary(d)
    _check(rot, _randn(b, hq, s, d), _randn(b, hk, s, d, seed=1), positions=7)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_positions(wide):
    rot = Rotary(64, base=500000.0)
    q, k = _randn(3, 4, 6, 64), _randn(3, 2, 6, 64, seed=1)
    g = torch.Generator().manual_seed(3)
    top = 2 ** 31 - 7 if wide == torch.int32 else 2 ** 45
    first = torch.randint(-1000, top, (3,), generator=g).to(wide).cuda()
    _check(rot, q, k, first)
    each = torch.randint(0, top, (3, 6), generator=g).to(wide).cuda()
    _check(rot, q, k, each)
    _check(rot, q, k, each[:1])
    # Views: every other entry, a column, one value for all.
    _check(rot, q, k, torch.stack((first, first + 5), 1)[:, 1])
    _check(rot, q, k, each.t().contiguous().t())
    _check(rot, q, k, first[:1].expand(3))
    for n in (0, -3, 2 ** 31 + 11, 10 ** 15):
        _check(rot, q, k, n)
    _check(rot, q[:1], k[:1], first[:1])


@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(interleaved):
    """Projections' transposed views, rows off 16-byte borders, expanded heads,
    a stride of two, an offset base."""
    rot = Rotary(64, interleaved=interleaved)
    q, k = _randn(2, 9, 4, 64).transpose(1, 2), _randn(2, 9, 2, 64, seed=1).transpose(1, 2)
    want = _check(rot, q, k)
    assert torch.equal(rot(q.contiguous(), k.contiguous(), backend="hip")[0], want[0])
    _check(rot, _randn(2, 4, 9, 68)[..., :64], k)
    _check(rot, q, _randn(2, 1, 9, 64).expand(2, 3, 9, 64))
    _check(rot, _randn(2, 4, 9, 128)[..., ::2], k)
    _check(rot, _randn(2 * 4 * 9 * 64 + 3)[3:].view(2, 4, 9, 64), k)
    _check(rot, q.flip(3).flip(3)[:, ::2], k[:, :1])
    _check(rot, _randn(2, 4, 64, 9).transpose(2, 3), k)


def test_query_alone_and_paths_agree():
    """The native call, the ctypes one and the op give the same bits."""
    rot = Rotary(128, rotary_dim=64, interleaved=True, scaling="linear", factor=2.0)
    q, k = _randn(2, 8, 17, 128, dtype=BF16), _randn(2, 2, 17, 128, dtype=BF16, seed=1)
    n = torch.tensor([5, 99], dtype=torch.int32, device="cuda")
    want = _check(rot, q, k, n)
    assert torch.equal(rot(q, positions=n), want[0])
    args = (rot.turns, n, True, False, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(_HipRotary.apply(q, k, *args), want))
    assert torch.equal(_HipRotary.apply(q, None, *args), want[0])
    got = torch.ops.kotflash_amd.rotary(q, k, rot.turns, n, 0, True, False, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    compiled = torch.compile(lambda a, b: rot(a, b, positions=n), fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(compiled(q, k), want))


def test_special_values():
    """NaN and infinity stay in their pair; the type's largest value overflows
    as its rounding does."""
    rot = Rotary(32)
    q = _randn(1, 1, 4, 32)
    q[0, 0, 0, 3], q[0, 0, 1, 20], q[0, 0, 2, 5] = float("nan"), float("inf"), 65504.0
    out = rot(q, positions=1, backend="hip").cpu()
    assert out[0, 0, 0, [3, 19]].isnan().all() and out[0, 0, 1, [4, 20]].isinf().all()
    rest = torch.ones(4, 32, dtype=torch.bool)
    rest[0, [3, 19]] = rest[1, [4, 20]] = False
    assert out[0, 0][rest].isfinite().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved,layout", [(False, "bhsd"), (True, "bshd")])
def test_gradients(dtype, interleaved, layout):
    """The gradient turns back; missing and expanded ones; twice."""
    rot = Rotary(96, rotary_dim=48, interleaved=interleaved, amplitude=0.75)

    def new(h, seed):
        if layout == "bshd":
            return _randn(2, 11, h, 96, dtype=dtype, seed=seed).transpose(1, 2)
        return _randn(2, h, 11, 96, dtype=dtype, seed=seed)

    n = torch.tensor([3, 4000], device="cuda")
    q, k = new(6, 0).requires_grad_(), new(2, 1).requires_grad_()
    gq, gk = new(6, 2), new(2, 3)
    out = rot(q, k, positions=n, backend="hip")
    dq, dk = torch.autograd.grad(out, (q, k), (gq, gk), retain_graph=True)
    assert_turned(dq, gq, rot, n.cpu(), inverse=True)
    assert_turned(dk, gk, rot, n.cpu(), inverse=True)
    only, = torch.autograd.grad(out[1], k, gk, retain_graph=True)
    assert torch.equal(only, dk)
    none = torch.autograd.grad(out[1], (q, k), gk, allow_unused=True, retain_graph=True)
    assert none[0] is None and torch.equal(none[1], dk)
    one, = torch.autograd.grad(out[0].sum(), q, retain_graph=True)
    assert_turned(one, torch.ones_like(gq), rot, n.cpu(), inverse=True)
    # The gradient's gradient, which the function gives too.
    g2 = gq.clone().requires_grad_()
    d, = torch.autograd.grad(out[0], q, g2, create_graph=True)
    dd, = torch.autograd.grad(d, g2, q.detach())
    assert torch.equal(dd, out[0].detach())
    # The same through the ctypes path and through the op.
    args = (rot.turns, n, interleaved, False, 0.75)
    for f in (lambda a, b: _HipRotary.apply(a, b, *args),
              lambda a, b: torch.ops.kotflash_amd.rotary(a, b, rot.turns, n, 0, interleaved, False, 0.75)):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(f(q, k), (q, k), (gq, gk)), (dq, dk)))
    both = torch.ops.kotflash_amd.rotary(q, k, rot.turns, n, 0, interleaved, False, 0.75)
    assert torch.equal(torch.autograd.grad(both[1], k, gk)[0], dk)
    compiled = torch.compile(lambda a, b: rot(a, b, positions=n), fullgraph=True, backend="aot_eager")
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(compiled(q, k), (q, k), (gq, gk)), (dq, dk)))
    alone = torch.compile(lambda a: rot(a, positions=n), fullgraph=True, backend="aot_eager")
    assert torch.equal(torch.autograd.grad(alone(q), q, gq)[0], dq)
    a, b = torch.autograd.grad(_HipRotary.apply(q, k, *args)[1], (q, k), gk, allow_unused=True)
    assert a is None and torch.equal(b, dk)
    # Queries alone, from an int position on.
    d1, = torch.autograd.grad(rot(q, positions=12, backend="hip"), q, gq)
    assert_turned(d1, gq, rot, 12, inverse=True)
    # A leaf that needs none.
    dk2, = torch.autograd.grad(rot(q.detach(), k, positions=n, backend="hip")[1], k, gk)
    assert torch.equal(dk2, dk)


def test_gradient_differences():
    """Directional differences of a step, in fp16: the kernel is linear, so the
    difference is the derivative but for roundings of eps / 2 in both ends."""
    rot = Rotary(64)
    q, v, g = (_randn(1, 2, 8, 64, seed=s) for s in range(3))
    leaf = q.clone().requires_grad_()
    d, = torch.autograd.grad(rot(leaf, positions=50, backend="hip"), leaf, g)
    ends = [rot(q + s * v, positions=50, backend="hip").double() for s in (1, -1)]
    step = ((q + v).double() - (q - v).double())
    want = ((ends[0] - ends[1]) * g.double()).sum()
    got = (d.double() * step).sum()
    eps = torch.finfo(F16).eps / 2
    tol = eps * ((ends[0].abs() + ends[1].abs()) * g.double().abs()).sum() + eps * (d.double().abs() * step.abs()).sum()
    assert abs(got - want) <= tol + 1e-3


def test_positions_changed_before_backward_are_refused():
    rot = Rotary(64)
    n = torch.tensor([3], dtype=torch.int32, device="cuda")
    q = _randn(1, 2, 4, 64).requires_grad_()
    out = rot(q, positions=n)
    n.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_graph_replays_follow_positions():
    """A captured call turns by what the positions hold at each replay; the
    backward pass is captured with it."""
    rot = Rotary(128)
    q, k = _randn(4, 8, 1, 128).requires_grad_(), _randn(4, 2, 1, 128, seed=1).requires_grad_()
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    g = _randn(4, 8, 1, 128, seed=2), _randn(4, 2, 1, 128, seed=3)

    def call():
        out = rot(q, k, positions=n)
        return (*out, *torch.autograd.grad(out, (q, k), g))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for start in (0, 17, 100000):
        n.copy_(torch.arange(4, dtype=torch.int32, device="cuda") * 5 + start)
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert_turned(held[0], q, rot, n.cpu())


def test_other_stream():
    rot = Rotary(128)
    q = _randn(2, 8, 500, 128)
    want = rot(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = rot(q)
    stream.synchronize()
    assert torch.equal(got, want)


def test_other_types_and_refusals():
    rot = Rotary(64)
    q = _randn(1, 2, 3, 64, dtype=torch.float32)
    assert_turned(rot(q, positions=4), q, rot, 4)
    with pytest.raises(TypeError, match="float16 and bfloat16"):
        rot(q, backend="hip")
    half = q.half()
    with pytest.raises(ValueError, match="positions"):
        rot(half, positions=torch.zeros(5, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="q's device"):
        rot(half, positions=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="device"):
        rot(half.cpu())
    with pytest.raises(ValueError, match="same dtype"):
        rot(half, q)


def test_with_attention():
    """Scores depend on the distance alone: a common shift of all positions
    leaves the attention as it was, but for the roundings of the turned
    queries and keys: each score's error is at most 2 eps |q| |k| / sqrt(D)."""
    rot = Rotary(64)
    q, k, v = _randn(1, 4, 40, 64), _randn(1, 2, 40, 64, seed=1), _randn(1, 2, 40, 64, seed=2)
    a, b = (attention(*rot(q, k, positions=n), v, causal=True).double() for n in (0, 1234))
    eps = torch.finfo(F16).eps / 2
    ds = 4 * eps * float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) / 8
    assert (a - b).abs().max() <= 2 * (2 * ds + 4 * eps) * float(v.abs().max())


def test_large_tensor():
    """Elements beyond 2^31: 17 heads of 4 GB."""
    s, h = 1_000_003, 17
    rot = Rotary(128)
    q = torch.zeros(1, h, s, 128, dtype=F16, device="cuda")
    tail = _randn(1, h, 5, 128)
    q[:, :, -5:] = tail
    out = rot(q, positions=3)
    assert_turned(out[:, :, -5:].contiguous(), tail, rot, 3 + s - 5)
    assert int(out[:, :, :-5].count_nonzero()) == 0
