"""Pages of a compressed cache on the GPU: bytes end where they should and nowhere else.

Every operator is compared with plain indexing on the host, byte for byte over the whole pool.
"""

import pytest
import torch

from turboquant_pytorch import PagePool
from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("kcodes", "ksigns", "krn", "kvn", "vcodes", "vvn")


def _pool(N, P, H, D, bits, layers, seed=0):
    pool = PagePool(N, P, H, D, bits, layers=layers, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for i in range(layers):
        for t in pool.planes(i).values():
            if t.dtype == torch.uint8:
                t.copy_(torch.randint(0, 256, t.shape, device=DEV, generator=g, dtype=torch.uint8))
            else:
                t.copy_(torch.randn(t.shape, device=DEV, generator=g))
    return pool


def _host(pool):
    return [{n: t.cpu().clone() for n, t in pool.planes(i).items()} for i in range(pool.layers)]


def _same(pool, host):
    for i, planes in enumerate(host):
        for n, t in planes.items():
            assert torch.equal(pool.planes(i)[n].cpu(), t), (i, n)


def _rows(B, H, S, D, bits, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(2, B, H, S, D, device=DEV, generator=g)
    return (TurboQuantCompressorV2(D, bits, 42, DEV).compress(x[0]), TurboQuantCompressorMSE(D, bits, 7, DEV).compress(x[1]))


def _named(ck, cv, B, H, S):
    flat = (ck["packed_key_indices"], ck["packed_qjl_signs"], ck["residual_norm"], ck["vec_norms"], cv["packed_indices"],
            cv["vec_norms"])
    return {n: (t.reshape(B, H, S, -1) if t.dtype == torch.uint8 else t.reshape(B, H, S)).cpu()
            for n, t in zip(NAMES, flat)}


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# head dims whose rows are whole 16, 8, 4, 2 and 1 byte pieces
@pytest.mark.parametrize("D,bits", [(128, 3), (64, 2), (64, 4), (96, 3), (80, 3), (40, 2), (24, 3), (8, 2), (256, 4)])
@pytest.mark.parametrize("S,P", [(1, 32), (33, 32), (70, 64)])
def test_write_and_read(D, bits, S, P):
    print("case:", D, bits, S, P, flush=True)
    B, H, N = 4, 3, 14
    pool = _pool(N, P, H, D, bits, 2)
    host = _host(pool)
    ck, cv = _rows(B, H, S, D, bits, S)
    new = _named(ck, cv, B, H, S)
    table = _i32(5, 0, 9, -1, 3, 7, 1, 11, 2, N, 4, 6, 8, 10, 12, 13).reshape(4, 4)
    start = _i32(P - 1, 0, 5, -1)  # across a page's end; one sequence's second page is not in the pool; one waits
    pool.write(1, ck, cv, table, start)
    for b in range(B):
        for s in range(S):
            pos = int(start[b]) + s
            if int(start[b]) < 0 or pos // P >= 4:
                continue
            page = int(table[b, pos // P])
            if 0 <= page < N:
                for n in NAMES:
                    host[1][n][page, :, pos % P] = new[n][b, :, s]
    _same(pool, host)
    lengths = _i32(P + 3, 2, 0, -4)
    k, v = pool.read(1, table, lengths, S)
    got = _named(k, v, B, H, S)
    assert k["shape"] == (B, H, S, D)
    for b in range(B):
        for s in range(S):
            page = int(table[b, s // P]) if s // P < 4 else -1
            for n in NAMES:
                want = host[1][n][page, :, s % P] if s < int(lengths[b]) and 0 <= page < N else torch.zeros_like(got[n][b, :, s])
                assert torch.equal(got[n][b, :, s], want), (b, s, n)
    _same(pool, host)


def test_copy_pages_of_every_layer():
    pool = _pool(9, 32, 2, 80, 3, 3, seed=2)
    host = _host(pool)
    pool.copy(_i32(4, 0, 8, 2, -1), _i32(1, 3, 9, -3, 5))  # the last three pairs name pages that are not there
    for planes in host:
        for t in planes.values():
            t[1], t[3] = t[4].clone(), t[0].clone()
    _same(pool, host)
    pool.copy(_i32(), _i32())
    _same(pool, host)


@pytest.mark.parametrize("D,bits,P", [(128, 3, 32), (64, 2, 64), (24, 3, 32), (256, 8, 32)])
def test_keep_moves_overlapping_rows(D, bits, P):
    print("case:", D, bits, P, flush=True)
    H, T = 2, 8
    pool = _pool(12, P, H, D, bits, 3, seed=3)
    host = _host(pool)
    table = _i32(3, 5, 7, 9, 0, 2, 11, 1, 4, 6, -1, 8, 10, 3).reshape(7, 2)
    table[6, 0], table[6, 1] = 3, -1  # shared with sequence 0, which does not move rows there
    lengths = _i32(P - 3, 10, 0, P - 2, 20, 5, 0)
    path = torch.tensor([[0, 1, 3, 4, 7, -1, -1, -1], [0, 2, 4, 6, 7, -1, -1, -1], [0, 1, 2, -1, -1, -1, -1, -1],
                         [0, 3, 5, -1, -1, -1, -1, -1], [0, 5, -1, -1, -1, -1, -1, -1], [0, 9, 3, 2, -1, -1, -1, -1],
                         [0, -1, -1, -1, -1, -1, -1, -1]], dtype=torch.int32, device=DEV)
    count = _i32(5, 5, 3, 3, 2, 4, 1)
    lengths[4] = -1
    new = pool.keep(table, lengths, path, count)
    assert new.tolist() == [P + 2, 15, 3, P + 1, -1, 9, 1]
    old = [{n: t.clone() for n, t in planes.items()} for planes in host]
    for b in range(7):
        for i in range(int(count[b])):
            k, at = int(path[b, i]), int(lengths[b])
            if at < 0 or not 0 <= k < T or (at + k) // P > 1 or (at + i) // P > 1:
                continue
            src, dst = int(table[b, (at + k) // P]), int(table[b, (at + i) // P])
            if 0 <= src < 12 and 0 <= dst < 12:
                for l in range(3):
                    for n in NAMES:
                        host[l][n][dst, :, (at + i) % P] = old[l][n][src, :, (at + k) % P]
    _same(pool, host)


def test_replays_of_a_captured_keep():
    """write + keep captured together; the tables' contents change between the replays."""
    D, bits, P, B, H, T = 64, 3, 32, 3, 2, 6
    pool = _pool(10, P, H, D, bits, 1, seed=5)
    ck, cv = _rows(B, H, T, D, bits, 1)
    table = torch.randperm(9, device=DEV).to(torch.int32).reshape(3, 3)
    lengths, count = _i32(30, 0, 7), _i32(3, 1, 4)
    path = _i32(0, 2, 5, -1, -1, -1, 0, -1, -1, -1, -1, -1, 0, 1, 3, 5, -1, -1).reshape(3, 6)

    def step():
        pool.write(0, ck, cv, table, lengths)
        return pool.keep(table, lengths, path, count)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = step()
    for rep in range(4):
        lengths.copy_(_i32(rep * 9, 40 + rep, 0))
        table.copy_(torch.randperm(9, device=DEV).to(torch.int32).reshape(3, 3))
        before = _host(pool)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, lens = _host(pool), new.clone()
        for n in NAMES:
            pool.planes(0)[n].copy_(before[0][n])
        want = step()
        assert torch.equal(lens, want)
        _same(pool, got)


def test_a_pool_past_4_gib():
    """Rows of the last page of a plane beyond 2^32 bytes."""
    N, P, H, D = 46000, 256, 8, 128
    pool = PagePool(N, P, H, D, 3, device=DEV)
    assert pool.planes(0)["vcodes"].numel() > 1 << 32
    ck, cv = _rows(1, H, 40, D, 3, 9)
    table = _i32(N - 1, N - 2).reshape(1, 2)
    pool.write(0, ck, cv, table, _i32(230))
    k, v = pool.read(0, table, _i32(270), 270)
    got, new = _named(k, v, 1, H, 270), _named(ck, cv, 1, H, 40)
    for n in NAMES:
        assert torch.equal(got[n][:, :, 230:], new[n]) and not got[n][:, :, :230].any(), n
    pool.copy(_i32(N - 2), _i32(0))
    pl = pool.planes(0)
    for n in NAMES:
        assert torch.equal(pl[n][0], pl[n][N - 2]) and pl[n][0].any(), n


def test_tables_of_no_pages():
    """Sequences without a page yet: reads are zeros, writes go nowhere, lengths still advance."""
    print("case: no pages", flush=True)
    pool = PagePool(4, 32, 2, 64, 3, layers=2, device=DEV)
    for t in pool._planes:
        t.view(torch.uint8).fill_(0x55)
    keep = [t.clone() for t in pool._planes]
    table = torch.empty(3, 0, dtype=torch.int32, device=DEV)
    at = torch.tensor([0, 7, -1], dtype=torch.int32, device=DEV)
    ck, cv = pool.read(1, table, at, 9)
    for t in (ck["packed_key_indices"], ck["packed_qjl_signs"], ck["residual_norm"], ck["vec_norms"], cv["packed_indices"],
              cv["vec_norms"]):
        assert not t.any()
    pool.write(1, ck, cv, table, at)
    path = torch.tensor([[0, 1], [0, -1], [0, 1]], dtype=torch.int32, device=DEV)
    assert pool.keep(table, at, path, torch.tensor([2, 1, 2], dtype=torch.int32, device=DEV)).tolist() == [2, 8, -1]
    torch.cuda.synchronize()
    for t, k in zip(pool._planes, keep):
        assert torch.equal(t.view(torch.uint8), k.view(torch.uint8))
