"""Norm + rotation + append with activations and rotation table of different
types: the same as the table's values in the activations' own type."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from paged_util import ints, make_cache, starts  # noqa: E402


@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 96), (256, 128)])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("x_type", [torch.float32, torch.bfloat16])
def test_mixed_types(hd, rot, norm, x_type):
    g = torch.Generator().manual_seed(hd)
    x = torch.randn(30, 10 * hd, generator=g).bfloat16()            # exact in both types
    table = (2 * torch.rand(64, 2 * rot, generator=g) - 1).bfloat16()
    w = (torch.rand(hd, generator=g) + 0.5).cuda() if norm else None
    got = []
    for t_type in (torch.float32, torch.bfloat16):
        k, v, pages, _ = make_cache([50, 9], 2, hd, 16, fill=0.0)
        out = torch.zeros(30, 6, hd, dtype=torch.bfloat16, device="cuda")
        ab.qk_norm_rope(x.to(x_type).cuda(), out, k, v, pages, starts([25, 5]), ints([50, 9]), table.to(t_type).cuda(),
                        q_weight=w, k_weight=w)
        got.append((out, k, v))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][0].any()
