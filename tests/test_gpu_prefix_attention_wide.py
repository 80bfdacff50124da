"""The tests of tests/test_gpu_prefix_attention.py over tables wide enough that shared rows are read once for a group.

Over a table that holds little, prefix_attention works each sequence by itself; the same cases here have tables with
unused entries behind, for 2^16 positions and more."""

import pytest
import torch

import test_gpu_prefix_attention as narrow
from test_gpu_prefix_attention import *  # noqa: F401,F403  (the tests)
from turboquant_pytorch import prefix_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def wide_tables(monkeypatch):
    setup = narrow._setup

    def wide(D, bits, Hq, Hkv, T, sizes, shared, own, page, seed=0):
        kc, vc, pool, table, *rest = setup(D, bits, Hq, Hkv, T, sizes, shared, own, page, seed)
        behind = torch.full((len(table), (1 << 16) // page + 1), -1, dtype=torch.int32, device=table.device)
        return kc, vc, pool, torch.cat([table, behind], 1), *rest

    monkeypatch.setattr(narrow, "_setup", wide)


def test_both_ways_agree_where_the_rule_changes():
    """The widest table for which sequences are worked apart and the next one, and a sequence shorter than its share."""
    T = 3
    kc, vc, pool, table, lengths, groups, q = narrow._setup(128, 3, 8, 2, T, [4, 2], [256, 96], [30, 100, 5, 64, 13, 50], 32, seed=19)
    lengths[2] = 255
    outs = []
    for positions in range(4096, 8192 + 1, 128):  # 6 x 2 x 33 to 64 rounds, on both sides of 512
        part = table[:, :positions // 32].contiguous()
        out = prefix_attention(q, kc, vc, pool, 1, part, lengths, groups, out_dtype=torch.float32)
        assert (out[2] == 0).all()
        outs.append(out)
    seen = lengths.clone()
    seen[2] = -1
    for out in (outs[0], outs[-1]):
        narrow._check(out, kc, vc, pool, table, seen, q, None)
    # in between only the two results appear, the one behind the other: 2^-10 a column, as rounding differs
    change = [i for i in range(1, len(outs)) if not torch.equal(outs[i], outs[i - 1])]
    assert change and (outs[0] - outs[-1]).norm() <= 16 * 2.0 ** -10 * outs[0].norm()


def test_a_pool_past_4_gib():
    """Shared and own pages whose rows lie beyond 2^32 bytes of a plane."""
    N, P, H, D, T = 46000, 256, 8, 128, 2
    kc, vc = narrow._compressors(D, 3)
    pool = narrow.PagePool(N, P, H, D, 3, layers=2, device="cuda")
    assert pool.planes(1)["vcodes"].numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(23)
    table = torch.full((3, 64), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = torch.tensor([N - 1, N - 2], dtype=torch.int32)
    table[:, 2] = torch.tensor([N - 5, N - 4, N - 3], dtype=torch.int32)
    shared = [torch.randn(1, H, 2 * P, D, device="cuda", generator=g).expand(3, -1, -1, -1) for _ in range(2)]
    k, v = (torch.cat([t, torch.randn(3, H, 100, D, device="cuda", generator=g)], 2) for t in shared)
    pool.write(1, kc.compress(k), vc.compress(v), table, torch.zeros(3, dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([2 * P + 98, 2 * P + 50, 2 * P], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 32, T, D, device="cuda", generator=g)
    groups = narrow.prefix_groups([3], [2 * P])
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, out_dtype=torch.float32)
    narrow._check(out, kc, vc, pool, table, lengths, q, None)
