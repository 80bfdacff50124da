"""Borders of sampling that a rounding could move."""

import pytest
import torch

from test_gpu_sampling import _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_just_below_zero(dtype):
    """Zero is an edge of the bins; logits down to -2^-29 are so near it that their place in the bin below rounds to its end."""
    g = torch.Generator(device=DEV).manual_seed(61)
    l = -3.0 + torch.randn(4, 3000, device=DEV, generator=g)
    l[0, ::7] = -1e-9  # 429 equal ones at the top
    l[1, ::5] = -2.0 ** -29 * torch.rand(600, device=DEV, generator=g)
    l[2, ::5] = -2.0 ** -28 * torch.rand(600, device=DEV, generator=g)
    l[2, 3::11] = -0.06 * torch.rand(273, device=DEV, generator=g)
    l[3, ::3] = -1e-9
    l[3, 1::30] = 0.4 * torch.rand(100, device=DEV, generator=g)
    l, u = l.to(dtype), torch.rand(4, device=DEV, generator=g)
    for kw in (dict(k=50), dict(k=300), dict(k=400, p=0.5), dict(p=0.3), dict(p=0.6), dict(k=700, m=0.9), dict(t=3.0, p=0.4)):
        print("case:", dtype, kw, flush=True)
        _check(l, u, **kw)


@pytest.mark.parametrize("light,p", [(-1.54, 1 - 1e-6), (-1.54, 1 - 2e-6), (-1.6, 1 - 1e-6)])
def test_top_p_over_hundreds_of_chunks(light, p):
    """598 chunks with the same masses, whose float32 sums over the chunks would all be rounded to one side."""
    V = 598 * 4096
    l = torch.full((1, V), light, device=DEV)
    l[0, ::4096] = 0.0
    print("case:", light, p, flush=True)
    probs, _ = _check(l, torch.full((1,), 0.999999, device=DEV), p=p)
    assert int((probs > 0).sum()) < V
