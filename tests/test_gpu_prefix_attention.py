"""Attention of sequences that share a long prefix, against float64.

The oracle is that of tree attention (tests/test_gpu_tree_attention.py), which knows nothing of groups: every sequence
over its own table row.  Its tolerance holds here as it is: the roundings of a weight and of a value are
the same, and a column's records are joined in float32 as a sequence's parts are there.
"""

import pytest
import torch

from test_gpu_tree_attention import _check, _compressors, _tree
from turboquant_pytorch import PagePool, append_prefix_attention, prefix_attention, prefix_groups, tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(D, bits, Hq, Hkv, T, sizes, shared, own, page, seed=0):
    """Groups of `sizes` sequences with `shared` positions in common and own[b] (a negative one: no sequence) behind
    them.  Whole pages of the shared positions are the same pages; a page that they end in is
    each sequence's own, with the same rows.  Rows that belong to nobody hold random codes and NaN norms."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    kc, vc = _compressors(D, bits)
    first = [s for n, s in zip(sizes, shared) for _ in range(n)]
    group = [i for i, n in enumerate(sizes) for _ in range(n)]
    B = len(first)
    lens = [s + n if n >= 0 else -1 for s, n in zip(first, own)]
    need = [max(0, -(-(n + T) // page)) for n in lens]
    heads = [s // page for s in shared]
    N = sum(heads) + sum(max(0, n - heads[i]) for n, i in zip(need, group)) + 3
    pool = PagePool(N, page, Hkv, D, bits, layers=2, device=DEV)
    for t in pool.planes(1).values():
        if t.dtype == torch.uint8:
            t.copy_(torch.randint(0, 256, t.shape, device=DEV, generator=g, dtype=torch.uint8))
        else:
            t.fill_(float("nan"))
    order = torch.randperm(N, generator=g, device=DEV).to(torch.int32)
    at, prompts = 0, []
    for h in heads:
        prompts.append(order[at:at + h])
        at += h
    width = max(need + heads) + 1
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    for b, (n, i) in enumerate(zip(need, group)):
        table[b, :heads[i]] = prompts[i]
        if n > heads[i]:
            table[b, heads[i]:n] = order[at:at + n - heads[i]]
            at += n - heads[i]
    text = [(torch.randn(1, Hkv, s, D, device=DEV, generator=g), torch.randn(1, Hkv, s, D, device=DEV, generator=g)) for s in shared]
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    for b in range(B):
        if own[b] < 0 and shared[group[b]] == 0:
            continue
        n = max(0, own[b] + T) if own[b] >= 0 else 0
        k, v = (torch.cat([t, (1 + b % 3) * torch.randn(1, Hkv, n, D, device=DEV, generator=g)], 2) for t in text[group[b]])
        if own[b] < 0:  # only whole pages, which the others have too
            k, v = k[:, :, :heads[group[b]] * page], v[:, :, :heads[group[b]] * page]
        if k.shape[2]:
            pool.write(1, kc.compress(k), vc.compress(v), table[b:b + 1].contiguous(), zero)
    q = torch.randn(B, Hq, T, D, device=DEV, generator=g)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return kc, vc, pool, table, lengths, prefix_groups(sizes, shared), q


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (1, 3, 3), (5, 4, 2), (16, 8, 2), (33, 2, 1)])
def test_groups_of_a_ragged_batch(D, bits, T, Hq, Hkv):
    print("case:", D, bits, T, Hq, Hkv, flush=True)
    st = _setup(D, bits, Hq, Hkv, T, [3, 1, 4, 2, 1], [96, 0, 200, 33, 640], [0, 31, 500, 1, 0, 64, 3, 200, 5, 6, 7], 32, seed=T)
    kc, vc, pool, table, lengths, groups, q = st
    par = _tree(T, len(q), T)
    for parents in (par, None):
        out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, parents, out_dtype=torch.float32)
        _check(out, kc, vc, pool, table, lengths, q, parents)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_types_pages_and_strides(dtype, page):
    print("case:", dtype, page, flush=True)
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, 8, 2, 3, [4, 2], [700, 256], [5, 100, 0, 31, 40, 7], page, seed=3)
    par = _tree(3, 6, 5)
    q = q.to(dtype).transpose(1, 2).contiguous().transpose(1, 2)  # as a projection leaves it
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par)
    assert out.dtype == dtype
    _check(out, kc, vc, pool, table, lengths, q, par)


@pytest.mark.parametrize("T,Hq,Hkv,n,page", [(1, 8, 2, 20000, 64), (3, 6, 3, 9024, 32), (7, 8, 1, 5000, 128)])
def test_long_prefixes(T, Hq, Hkv, n, page):
    print("case:", T, Hq, Hkv, n, page, flush=True)
    own = [0, 800, 33, 1, 2000, 64, 5]
    kc, vc, pool, table, lengths, groups, q = _setup(64, 3, Hq, Hkv, T, [7], [n], own, page, seed=12)
    par = _tree(T, 7, 2)
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, scale=0.2, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par, scale=0.2)


@pytest.mark.parametrize("T,Hq,Hkv", [(1, 2, 1), (1, 16, 16), (3, 6, 3), (6, 12, 3)])
def test_more_sequences_than_lanes(T, Hq, Hkv):
    """Groups that go past the 64th and the 128th sequence, and many small ones."""
    print("case:", T, Hq, Hkv, flush=True)
    sizes, shared = [3, 100, 40, 1, 2, 2, 2, 30], [64, 160, 0, 32, 96, 31, 128, 512]
    own = [(7 * b) % 90 - (b % 11 == 5) * 100 for b in range(sum(sizes))]  # some are no sequences
    kc, vc, pool, table, lengths, groups, q = _setup(64, 3, Hq, Hkv, T, sizes, shared, own, 32, seed=21)
    par = _tree(T, len(q), 4)
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    some = torch.tensor([0, 1, 2, 3, 4, 5, 60, 62, 63, 64, 65, 102, 103, 127, 128, 130, 143, 144, 145, 146, 149, 150, 179], device=DEV)
    assert (lengths[some] < 0).any()
    _check(out[some], kc, vc, pool, table[some], lengths[some], q[some], par[some])


def test_ids_that_end_begin_again_and_mean_nothing():
    """A group is a run of equal entries; the same id further on is another run, and -1 or a share of zero or of a
    negative number is none."""
    T, sizes, shared = 2, [6], [128]
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, 4, 2, T, sizes, shared, [3, 40, 0, 9, 80, 1], 32, seed=5)
    for rows in ([[0, 128]] * 6, [[7, 128], [7, 128], [3, 128], [7, 128], [7, 128], [7, 96]],
                 [[-1, 128]] * 6, [[0, 0], [0, 128], [0, 128], [0, 64], [0, 64], [0, -5]],
                 [[1, 100], [1, 100], [1, 31], [1, 31], [2 ** 31 - 1, 33], [-(2 ** 31), 33]]):
        g = torch.tensor(rows, dtype=torch.int32, device=DEV)
        out = prefix_attention(q, kc, vc, pool, 1, table, lengths, g, out_dtype=torch.float32)
        _check(out, kc, vc, pool, table, lengths, q, None)


def test_sequences_that_do_not_run_and_pages_that_are_not_there():
    T = 4
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, 4, 2, T, [5, 2], [160, 64], [70, -1, 100, 40, 3, 9, 30], 32, seed=6)
    lengths[2] = table.shape[1] * 32 - 3  # one position too many
    lengths[3] = 159  # shorter than what it shares
    table[:5, 1] = -1  # pages of the prompt that are gone
    table[:5, 3] = pool.num_pages + 7
    table[6, 2] = -5
    par = _tree(T, 7, 8, pads=False)
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    assert (out[3] == 0).all()
    lengths[3] = -1  # for the oracle, which has no groups
    _check(out, kc, vc, pool, table, lengths, q, par)
    # the first of a group is no sequence any more, the others go on
    lengths[0] = -1
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)
    # a share that no table row holds leaves nothing to attend
    groups[:, 1] = table.shape[1] * 32 + 1
    assert (prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par) == 0).all()
    # every page of a group gone
    groups[:, 1] = 64
    table[5:] = -1
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    assert (out[5:] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 1e30, 6e4])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (3, 8, 2)])
def test_a_sequence_of_any_queries_changes_nothing_for_the_others(bad, T, Hq, Hkv):
    """Bit for bit: also a row that is no sequence, whose queries were never written."""
    print("case:", bad, T, Hq, Hkv, flush=True)
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, Hq, Hkv, T, [6], [320], [5, 60, -1, 3, 0, 9], 32, seed=9)
    clean = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, out_dtype=torch.float32)
    rest = [0, 1, 3, 5]
    q[2], q[4] = bad, -bad
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, out_dtype=torch.float32)
    assert torch.equal(out[rest], clean[rest]) and (out[2] == 0).all()


def test_nodes_without_a_place():
    T = 6
    kc, vc, pool, table, lengths, groups, q = _setup(64, 4, 4, 2, T, [3], [96], [5, 60, 0], 32, seed=10)
    par = torch.tensor([[-1, 0, 9, 1, -2, 0], [-1] * 6, [-2] * 6], dtype=torch.int32, device=DEV)
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)
    assert (out[0, [2, 4]] == 0).all() and (out[2] == 0).all()
    one = torch.tensor([-1, 0, -2, 0, 1, 5], dtype=torch.int32, device=DEV)  # one tree for all
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, one, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, one)


@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (6, 12, 2)])
def test_large_norms_of_a_shared_row(T, Hq, Hkv):
    """Norms at the end of f16 and zero in a row that everybody sees."""
    kc, vc, pool, table, lengths, groups, q = _setup(64, 3, Hq, Hkv, T, [4], [96], [5, 60, 0, 33], 32, seed=11)
    page, pl = int(table[0, 1]), pool.planes(1)
    for val in (6e4, 0.0, 2.0 ** -24):
        pl["vvn"][page, :, 5] = val
        out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, out_dtype=torch.float32)
        _check(out, kc, vc, pool, table, lengths, q, None)


@pytest.mark.parametrize("D,bits", [(64, 2), (128, 3), (128, 4)])
@pytest.mark.parametrize("T,Hq,Hkv,dtype", [(1, 4, 2, torch.bfloat16), (7, 8, 2, torch.float32), (20, 4, 2, torch.float16)])
def test_step_equals_its_parts(D, bits, T, Hq, Hkv, dtype):
    """append_prefix_attention: the rows it writes and its attention, bit for bit."""
    print("case:", D, bits, T, Hq, Hkv, dtype, flush=True)
    kc, vc, pool, table, lengths, groups, q = _setup(D, bits, Hq, Hkv, T, [4, 1], [128, 0], [5, 60, -1, 33, 7], 32, seed=T)
    g = torch.Generator(device=DEV).manual_seed(T)
    k, v, q = (torch.randn(5, T, h, D, device=DEV, generator=g).to(dtype).transpose(1, 2) for h in (Hkv, Hkv, Hq))
    two = PagePool.over(*(t.clone() for t in pool._planes))
    out = append_prefix_attention(k, v, q, kc, vc, pool, 1, table, lengths, groups)
    two.write(1, kc.compress(k), vc.compress(v), table, lengths)
    assert torch.equal(out, prefix_attention(q, kc, vc, two, 1, table, lengths, groups)) and out.dtype == dtype
    for x, y in zip(pool._planes, two._planes):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # keys of another type than the queries
    mixed = append_prefix_attention(k.float(), v.float(), q, kc, vc, pool, 1, table, lengths, groups)
    assert torch.equal(mixed, out)


def test_graph_replays_with_other_lengths_and_groups():
    T = 2
    kc, vc, pool, table, lengths, groups, q = _setup(64, 3, 4, 2, T, [4, 2], [256, 96], [30, 100, 5, 64, 13, 50], 32, seed=14)
    par = _tree(T, 6, 1, pads=False)
    args = (q, kc, vc, pool, 1, table, lengths, groups, par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prefix_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prefix_attention(*args)
    full = lengths.clone()
    for rep, (less, share) in enumerate([(0, [256, 96]), (3, [256, 64]), (5, [0, 96]), (1, [200, 90]), (4, [128, 0])]):
        lengths.copy_(full - less)
        groups.copy_(prefix_groups([4, 2], share))
        if rep == 2:
            lengths[1] = -1
        q.normal_()
        torch.cuda.synchronize()
        want = prefix_attention(*args).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep
        _check(out, kc, vc, pool, table, lengths, q, par)


def test_other_streams_and_two_calls_at_once():
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, 8, 2, 3, [5], [640], [6, 90, 0, 31, 7], 64, seed=15)
    want = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(prefix_attention(q, kc, vc, pool, 1, table, lengths, groups))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


def test_an_empty_batch_and_one_sequence():
    kc, vc, pool, table, lengths, groups, q = _setup(64, 3, 4, 2, 1, [1], [64], [0], 32, seed=16)
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, None)
    alone = tree_attention(q, kc, vc, pool, 1, table, lengths, out_dtype=torch.float32)
    assert (out - alone).norm() <= 16 * 2.0 ** -10 * alone.norm()  # as tests/test_gpu_tree_attention.py derives it
    none = prefix_attention(q[:0], kc, vc, pool, 1, table[:0], lengths[:0], groups[:0])
    assert none.shape == (0, 1, 4, 64)


@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (3, 8, 2), (20, 4, 2)])
def test_a_group_that_begins_with_idle_rows(T, Hq, Hkv):
    """Padding rows of a batch: no length, and pages that are not theirs or none."""
    print("case:", T, Hq, Hkv, flush=True)
    own = [-1, -1, 40, -1, 3, 200, -1, -1, -1, 7, -1]
    kc, vc, pool, table, lengths, groups, q = _setup(128, 3, Hq, Hkv, T, [7, 1, 3], [500, 64, 160], own, 64, seed=17)
    table[[0, 6, 7, 8]] = -1
    table[1] = torch.arange(table.shape[1], dtype=torch.int32, device=DEV) % pool.num_pages  # another's rows
    par = _tree(T, len(q), 3)
    for parents in (par, None):
        out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, parents, out_dtype=torch.float32)
        _check(out, kc, vc, pool, table, lengths, q, parents)
    lengths[:7] = -1  # a whole group
    out = prefix_attention(q, kc, vc, pool, 1, table, lengths, groups, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)
