"""The rotary kernels against the formulas themselves (``rotary_definition``)."""
import pytest
import torch

from kotflash_amd.rotary import Rotary
from tests.rotary_definition import assert_definition, frequencies
from tests.test_rotary_angles import SCALINGS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", SCALINGS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (72, 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_outputs(kw, interleaved, d, r, dtype):
    """16 | rotary_dim, and the kernel for any other."""
    rot = Rotary(d, rotary_dim=r, interleaved=interleaved, amplitude=0.75, device="cuda", **kw)
    f = frequencies(r, **kw)
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, h, 5, d, generator=g).to(dtype).cuda() for h in (4, 2))
    first = torch.tensor([3, 100000], device="cuda")
    where = first.cpu()[:, None] + torch.arange(5)
    for x, y in zip((q, k), rot(q, k, positions=first, backend="hip")):
        assert_definition(y, x, f, where, interleaved=interleaved, amplitude=0.75)
