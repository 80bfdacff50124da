"""Borders of sampling that a rounding could move: where what is kept or drawn ends within 2^-30 of the total beside a token's edge.

Rows of a few levels, each of many equal logits, so that every sum is a product: a level's tokens times their weight, off by a
few 2^-53 of itself.  Borders are set on either side of an edge, further from it than 2^-40 of the total: the weights'
series is off by 3e-13 (2^-41.6), sums by less."""

import math

import pytest
import torch

from test_gpu_sampling import _check
from turboquant_pytorch import filter_probs, sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _near_edges(first, last, weight, total, least, most, count):
    """(uniforms, tokens): u total lies `least` to `most` beside the edge between tokens j - 1 and j of a row that begins with
    equal tokens; the draw is j where it lies behind the edge, else j - 1."""
    j = torch.arange(first, last, dtype=torch.float64)
    u = (j * weight / total).float()
    off = u.double() * total - j * weight
    take = torch.nonzero((off.abs() >= least) & (off.abs() <= most))[:, 0]
    take = take[torch.randperm(len(take), generator=torch.Generator().manual_seed(1))[:count]]
    assert len(take) == count and (off[take] > 0).any() and (off[take] < 0).any()
    return u[take].to(DEV), (j[take].long() - (off[take] < 0).long()).to(DEV)


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


def test_draws_between_light_tokens_under_min_p():
    n, at = 150000, -16.4716796875
    w = math.exp(at)
    u, want = _near_edges(60000, n, w, 1 + n * w, 4e-12, 1e-10, 48)
    l = torch.full((1, n + 1), at, device=DEV)
    l[0, n] = 0.0
    assert torch.equal(sample_tokens(l.expand(48, -1), u, min_p=1e-8), want)
    for i in range(4):  # a row by itself is cut into other chunks
        assert torch.equal(sample_tokens(l, u[i:i + 1], min_p=1e-8), want[i:i + 1])


@pytest.mark.parametrize("off", [2e-11, -2e-11])
def test_top_p_ends_among_light_tokens_below_light_ones(off):
    """60000 tokens that are kept for certain above the level in which the border lies."""
    n, a, b = 60000, -11.0439453125, -11.2939453125
    wa, wb = math.exp(a), math.exp(b)
    l = torch.full((1, 2 * n + 1), a, device=DEV)
    l[0, 1::2] = b
    l[0, 7000] = 0.0  # in place of one of the upper level, which has n + 1 places
    for j in (20000, 47000):
        p = (1 + n * wa + j * wb + off) / (1 + n * wa + n * wb)
        print("case:", j, p, flush=True)
        probs = filter_probs(l, top_p=p)
        assert int((probs > 0).sum()) == 1 + n + j + (off > 0)


@pytest.mark.parametrize("off", [3e-10, -3e-10])
def test_top_p_counts_tokens_that_weigh_almost_nothing(off):
    """A million tokens of 2^-49.1 each weigh 1.7e-9 together, beside 256 of weight 1 (2^-40 of the total is 2.3e-10)."""
    V, at = 1 << 20, -34.0625
    l = torch.full((1, V), at, device=DEV)
    l[0, ::4096] = 0.0
    for j in (150, 220):
        p = (j + off) / (256 + (V - 256) * math.exp(at))
        print("case:", j, p, flush=True)
        assert int((filter_probs(l, top_p=p) > 0).sum()) == j + (off > 0)


@pytest.mark.parametrize("off", [1e-10, -1e-10])
def test_top_p_of_many_ranked_tokens(off):
    n, at = 100000, -11.494140625
    w = math.exp(at)
    l = torch.full((1, 150001), at, device=DEV)
    l[0, 140000] = 0.0
    for j in (30000, 50000):
        p = (1 + j * w + off) / (1 + n * w)
        probs = filter_probs(l, top_k=n + 1, top_p=p)
        assert int((probs > 0).sum()) == 1 + j + (off > 0)


def test_draws_between_many_ranked_tokens():
    n, at = 100000, -11.494140625
    w = math.exp(at)
    u, want = _near_edges(20000, 90000, w, 1 + n * w, 2e-11, 4e-10, 16)
    l = torch.full((1, 150001), at, device=DEV)
    l[0, 150000] = 0.0
    assert torch.equal(sample_tokens(l.expand(16, -1), u, top_k=n + 1), want)
