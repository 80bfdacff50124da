"""The fused step of a layer over pages: the rows it writes, and its attention, are bit for bit those of the
operators it joins (compression, page writes, tree attention)."""

import pytest
import torch

from turboquant_pytorch import PagePool, tree_attention
from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2
from turboquant_pytorch.drafts import append_tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(D, bits, B, Hkv, T, lens, page, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kc = TurboQuantCompressorV2(D, bits, seed=42, device=DEV)
    vc = TurboQuantCompressorMSE(D, bits, seed=10042, device=DEV)
    need = [max(0, -(-(n + T) // page)) for n in lens]
    pools = []
    pool = PagePool(sum(need) + 2, page, Hkv, D, bits, layers=2, device=DEV)
    for t in pool._planes:  # rows that belong to nobody hold random bytes
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, device=DEV, generator=g, dtype=torch.uint8))
    pools = [PagePool.over(*(t.clone() for t in pool._planes)) for _ in range(2)]
    order = torch.randperm(pool.num_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return kc, vc, pools, table, torch.tensor(lens, dtype=torch.int32, device=DEV), g


def _same(a, b):
    for x, y in zip(a._planes, b._planes):  # as bytes: unwritten norms may be NaN
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("D,bits", [(64, 2), (64, 3), (64, 4), (128, 2), (128, 3), (128, 4)])
@pytest.mark.parametrize("T,Hq,Hkv,dtype", [(1, 4, 2, torch.bfloat16), (1, 3, 3, torch.float16), (7, 8, 2, torch.float32),
                                           (33, 4, 1, torch.bfloat16), (64, 2, 2, torch.float16)])
def test_step_equals_its_parts(D, bits, T, Hq, Hkv, dtype):
    print("case:", D, bits, T, Hq, Hkv, dtype, flush=True)
    lens = [0, 31, 200, 63, 64]
    B = len(lens)
    kc, vc, (one, two), table, lengths, g = _setup(D, bits, B, Hkv, T, lens, 32, T)
    k, v, q = (torch.randn(B, T, h, D, device=DEV, generator=g).to(dtype).transpose(1, 2) for h in (Hkv, Hkv, Hq))
    # cached rows, so that attention has something to see
    ck, cv = kc.compress(torch.randn(B, Hkv, 200, D, device=DEV, generator=g)), vc.compress(
        torch.randn(B, Hkv, 200, D, device=DEV, generator=g))
    for pool in (one, two):
        pool.write(1, ck, cv, table, torch.zeros_like(lengths))
    two.write(1, kc.compress(k), vc.compress(v), table, lengths)
    par = torch.tensor([[i - 1 - (i + b) % 2 if i else -1 for i in range(T)] for b in range(B)], dtype=torch.int32, device=DEV)
    for parents in (None, par):
        want = tree_attention(q, kc, vc, two, 1, table, lengths, parents)
        out = append_tree_attention(k, v, q, kc, vc, one, 1, table, lengths, parents)
        assert out.dtype == dtype and torch.equal(out, want)
        _same(one, two)


def test_missing_pages_and_negative_lengths_are_left_alone():
    kc, vc, (one, two), table, lengths, g = _setup(128, 3, 4, 2, 5, [30, 62, 64, 10], 32, 3)
    table[0, 1] = -1  # positions 32..34 of sequence 0
    table[1, 2] = one.num_pages  # its positions 64..66
    lengths[3] = -1
    k, v = torch.randn(4, 2, 5, 128, device=DEV, generator=g), torch.randn(4, 2, 5, 128, device=DEV, generator=g)
    q = torch.randn(4, 4, 5, 128, device=DEV, generator=g)
    two.write(0, kc.compress(k), vc.compress(v), table, lengths)
    before = [t.clone() for t in one._planes]
    append_tree_attention(k, v, q, kc, vc, one, 0, table, lengths)
    _same(one, two)
    for t, s in zip(one._planes, before):
        assert torch.equal(t[1].view(torch.uint8), s[1].view(torch.uint8))  # the other layer
    # a start behind the table, and mixed types
    lengths[:] = torch.tensor([30, 200, 64, 126], device=DEV)
    two.write(0, kc.compress(k), vc.compress(v), table, lengths)
    append_tree_attention(k, v.double(), q.half(), kc, vc, one, 0, table, lengths)
    _same(one, two)
    empty = append_tree_attention(k[:0], v[:0], q[:0], kc, vc, one, 0, table[:0], lengths[:0])
    assert empty.shape == (0, 5, 4, 128)


def test_captured_steps():
    """A decoding loop as a graph: lengths advance on the device between the replays."""
    kc, vc, (one, two), table, lengths, g = _setup(64, 3, 2, 2, 40, [20, 50], 32, 4)
    k, v, q = (torch.empty(2, h, 1, 64, device=DEV) for h in (2, 2, 4))
    ck, cv = kc.compress(torch.randn(2, 2, 50, 64, device=DEV, generator=g)), vc.compress(
        torch.randn(2, 2, 50, 64, device=DEV, generator=g))
    for pool in (one, two):
        pool.write(0, ck, cv, table, torch.zeros_like(lengths))
    length2 = lengths.clone()

    def step():
        out = append_tree_attention(k, v, q, kc, vc, one, 0, table, lengths)
        lengths.add_(1)
        return out

    keep = [t.clone() for t in one._planes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t, s in zip(one._planes, keep):
        t.copy_(s)
    lengths.copy_(length2)
    for i in range(20):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
        graph.replay()
        want = append_tree_attention(k, v, q, kc, vc, two, 0, table, length2)
        length2 += 1
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lengths, length2), i
    _same(one, two)


@pytest.mark.parametrize("bits,pages", [(3, 96000), (4, 70000)])
def test_pages_past_4_gib(bits, pages):
    """The last pages of a pool whose planes pass 2^32 bytes: the same outputs as in a small pool."""
    print("case:", bits, pages, flush=True)
    kc = TurboQuantCompressorV2(128, bits, seed=42, device=DEV)
    vc = TurboQuantCompressorMSE(128, bits, seed=10042, device=DEV)
    page, Hkv = 128, 8
    big, small = PagePool(pages, page, Hkv, 128, bits, device=DEV), PagePool(8, page, Hkv, 128, bits, device=DEV)
    assert big.planes(0)["vcodes"].numel() > 2 ** 32
    table = torch.tensor([[3, 0, 5, -1], [1, 7, 2, 6]], dtype=torch.int32, device=DEV)
    far = torch.where(table < 0, table, table + (pages - 8))
    g = torch.Generator(device=DEV).manual_seed(8)
    lengths = torch.tensor([250, 300], dtype=torch.int32, device=DEV)
    ck, cv = (c.compress(torch.randn(2, Hkv, 300, 128, device=DEV, generator=g)) for c in (kc, vc))
    for pool, t in ((big, far), (small, table)):
        pool.write(0, ck, cv, t, torch.zeros_like(lengths))
    for Hq, T in ((8, 1), (32, 1), (16, 5), (64, 40)):  # every form
        k, v, q = (torch.randn(2, h, T, 128, device=DEV, generator=g) for h in (Hkv, Hkv, Hq))
        wide = torch.full((2, 4096), -1, dtype=torch.int32, device=DEV)
        for pad in (False, True):
            out = []
            for pool, t in ((big, far), (small, table)):
                if pad:
                    w = wide.clone()
                    w[:, :4] = t
                    t = w
                out.append(append_tree_attention(k, v, q, kc, vc, pool, 0, t, lengths))
            assert torch.equal(*out) and torch.isfinite(out[0]).all()
    for name, t in big.planes(0).items():
        assert torch.equal(t[pages - 8:].view(torch.uint8), small.planes(0)[name].view(torch.uint8)), name


@pytest.mark.parametrize("kt,vt,qt", [(torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float16, torch.float32),
                                      (torch.float16, torch.float16, torch.bfloat16), (torch.bfloat16, torch.float32, torch.bfloat16),
                                      (torch.float16, torch.bfloat16, torch.float32), (torch.float32, torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 9)])
def test_mixed_types_lose_nothing(kt, vt, qt, D, T):
    """Rows and outputs bit for bit those of the separate operators, each on its own type."""
    print("case:", kt, vt, qt, D, T, flush=True)
    kc, vc, (one, two), table, lengths, g = _setup(D, 3, 3, 2, T, [0, 31, 200], 32, 5)
    k, v, q = (torch.randn(3, T, h, D, device=DEV, generator=g).to(t).transpose(1, 2) for h, t in ((2, kt), (2, vt), (4, qt)))
    two.write(1, kc.compress(k), vc.compress(v), table, lengths)
    want = tree_attention(q, kc, vc, two, 1, table, lengths)
    out = append_tree_attention(k, v, q, kc, vc, one, 1, table, lengths)
    assert out.dtype == qt and torch.isfinite(out[0]).all()
    assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))  # positions behind a prefix hold random rows
    _same(one, two)
    empty = append_tree_attention(k[:0], v[:0], q[:0], kc, vc, one, 1, table[:0], lengths[:0])
    assert empty.shape == (0, T, 4, D) and empty.dtype == qt
