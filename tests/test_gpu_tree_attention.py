"""Attention of drafted tokens over pages of a compressed cache, against float64.

The oracle reads the same packed rows and the device's prepared queries (f16 q_rot, f32 q_proj:
tests/test_gpu_kernels.py checks those) and works in float64 on the CPU.

Tolerance, per output row (b, i, h), derived before the first run: with weights p_j, the row's
error is measured in the 2-norm against  W = sum_j p_j vnv_j ||Cv[codes_j]||  (Pi_v is orthogonal).
  P as f16 operand: 2^-11 of each term; value centroids as f16: 2^-11; their product's cross term below 2^-20
  scores: f32 sums of d products, each term's partial sums off by at most d 2^-24 of the sum of
    absolute products A_j (q_proj as hi + lo adds 2^-22 of its part): ds = (d + 8) 2^-24 max_j A_j in natural-log
    units; a weight is off by at most 2 ds + 2^-20 (exp2 and the sums, f32)
  keys whose weight is below 2^-31 of the heaviest vanish: N 2^-30
  Pi_v as f16 hi + lo, f32 sums: d 2^-22
and the output's own rounding, eps / 2 of its type times the row's norm.
"""

import math

import pytest
import torch

from oracle import tq_oracle as O
from turboquant_pytorch import PagePool, tree_attention
from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2
from turboquant_pytorch.drafts import tree_attention_from_prepared

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _compressors(D, bits):
    return (TurboQuantCompressorV2(D, bits, seed=42, device=DEV),
            TurboQuantCompressorMSE(D, bits, seed=10042, device=DEV))


def _setup(D, bits, B, Hq, Hkv, T, lens, page, seed=0, garbage=True, spare=3):
    """A pool with each sequence's rows scattered over its pages; every row that belongs to nobody
    holds random codes and NaN norms."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    kc, vc = _compressors(D, bits)
    need = [max(0, -(-(n + T) // page)) for n in lens]
    N = sum(need) + spare
    pool = PagePool(N, page, Hkv, D, bits, layers=2, device=DEV)
    if garbage:
        for name, t in pool.planes(1).items():
            if t.dtype == torch.uint8:
                t.copy_(torch.randint(0, 256, t.shape, device=DEV, generator=g, dtype=torch.uint8))
            else:
                t.fill_(float("nan"))
    order = torch.randperm(N, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B, max(need + [1]) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    S = max([n + T for n in lens] + [1])
    k = torch.randn(B, Hkv, S, D, device=DEV, generator=g)
    v = torch.randn(B, Hkv, S, D, device=DEV, generator=g) * (1 + torch.rand(B, Hkv, S, 1, device=DEV, generator=g))
    for b, n in enumerate(lens):
        if n < 0:
            continue
        ck, cv = kc.compress(k[b:b + 1, :, :n + T]), vc.compress(v[b:b + 1, :, :n + T])
        pool.write(1, ck, cv, table[b:b + 1].contiguous(), torch.zeros(1, dtype=torch.int32, device=DEV))
    q = torch.randn(B, Hq, T, D, device=DEV, generator=g)
    return kc, vc, pool, table, lengths, q


def _tree(T, B, seed, pads=True):
    g = torch.Generator().manual_seed(seed)
    par = torch.empty(B, T, dtype=torch.int32)
    for b in range(B):
        for i in range(T):
            par[b, i] = int(torch.randint(max(-1, i - 5), i, (1,), generator=g)) if i else -1
    if pads and T > 3:
        par[-1, T - 2:] = torch.tensor([-2, T + 5])
    return par.to(DEV)


def _seen(par, T):
    """[T, T] bool from one sequence's parents, node by node."""
    out = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        p = i - 1 if par is None else int(par[i])
        if -1 <= p < i:
            if p >= 0:
                out[i] = out[p]
            out[i, i] = True
    return out


def _check(out, kc, vc, pool, table, lengths, q, par, scale=None, layer=1):
    B, Hq, T, D = q.shape
    P, H, bits = pool.page_size, pool.num_kv_heads, pool.bits
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    coeff = math.sqrt(math.pi / 2) / D
    q_rot, q_proj = (t.double().cpu() for t in kc.prepare_queries(q))
    pl = {n: t.cpu() for n, t in pool.planes(layer).items()}
    ck, cv = kc.centroids.half().double().cpu(), vc.centroids.double().cpu()
    pi_v = vc.Pi.double().cpu()
    tab, lens = table.cpu(), lengths.cpu().tolist()
    got = out.double().cpu()
    assert out.shape == (B, T, Hq, D) and torch.isfinite(got).all()
    eps = torch.finfo(out.dtype).eps / 2
    for b in range(B):
        n = lens[b]
        if n < 0 or n + T > table.shape[1] * P:
            assert (got[b] == 0).all()
            continue
        pos = torch.arange(n + T)
        page = tab[b, pos // P].long()
        have = (page >= 0) & (page < pool.num_pages)
        pos, page = pos[have], page[have]
        tree = _seen(None if par is None else (par if par.dim() == 1 else par[b]).cpu(), T)
        sees = torch.cat([tree.any(1, keepdim=True).expand(T, n), tree], 1)[:, have]
        for h in range(H):
            rows = {k: t[page, h, pos % P] for k, t in pl.items()}
            code = torch.from_numpy(O.unpack_bits(rows["kcodes"].numpy(), bits - 1, D)).long()
            sign = 2.0 * torch.from_numpy(O.unpack_bits(rows["ksigns"].numpy(), 1, D)).double() - 1
            vcode = torch.from_numpy(O.unpack_bits(rows["vcodes"].numpy(), bits, D)).long()
            keys, rn, kn = ck[code], rows["krn"].double(), rows["kvn"].double()
            vals = cv[vcode]
            for gq in range(G):
                qr, qp = q_rot[b, h * G + gq], q_proj[b, h * G + gq]
                s = scale * ((qr @ keys.T) * kn + coeff * (qp @ sign.T) * rn)
                big = scale * ((qr.abs() @ keys.abs().T) * kn + coeff * (qp.abs() @ sign.abs().T) * rn)
                for i in range(T):
                    m = sees[i]
                    row = got[b, i, h * G + gq]
                    if not m.any():
                        assert (row == 0).all(), (b, i, h)
                        continue
                    p = torch.softmax(s[i, m], 0)
                    vn = rows["vvn"].double()[m]
                    ref = ((p * vn) @ vals[m]) @ pi_v
                    W = float((p * vn * vals[m].norm(dim=1)).sum())
                    ds = (D + 8) * 2.0 ** -24 * float(big[i, m].max())
                    tol = 2.0 ** -10 + 2 * ds + 2.0 ** -20 + int(m.sum()) * 2.0 ** -30 + D * 2.0 ** -22
                    err = float((row - ref).norm())
                    assert err <= tol * W + eps * float(ref.norm()) * 1.01, (b, i, h, gq, err, tol * W)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 2), (1, 3, 3), (5, 4, 2), (9, 6, 2), (16, 8, 2), (33, 2, 1)])
def test_trees_ragged_batch(D, bits, T, Hq, Hkv):
    print("case:", D, bits, T, Hq, Hkv, flush=True)
    lens = [0, 31, 500, 1]
    st = _setup(D, bits, len(lens), Hq, Hkv, T, lens, 32, seed=T)
    kc, vc, pool, table, lengths, q = st
    par = _tree(T, len(lens), T)
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_types_pages_and_strides(dtype, page):
    print("case:", dtype, page, flush=True)
    lens = [257, 64, 3]
    kc, vc, pool, table, lengths, q = _setup(128, 3, 3, 8, 2, 7, lens, page, seed=3)
    par = _tree(7, 3, 5)
    q = q.to(dtype).transpose(1, 2).contiguous().transpose(1, 2)  # as a projection leaves it
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par)
    assert out.dtype == dtype
    _check(out, kc, vc, pool, table, lengths, q, par)


def test_shared_tree_chain_and_scale():
    kc, vc, pool, table, lengths, q = _setup(64, 3, 2, 4, 2, 6, [100, 37], 64, seed=4)
    par = torch.tensor([-1, 0, 0, 1, -1, 4], dtype=torch.int32, device=DEV)  # two trees in one
    _check(tree_attention(q, kc, vc, pool, 1, table, lengths, par, scale=0.3, out_dtype=torch.float32), kc, vc, pool,
           table, lengths, q, par, scale=0.3)
    chain = tree_attention(q, kc, vc, pool, 1, table, lengths, out_dtype=torch.float32)
    _check(chain, kc, vc, pool, table, lengths, q, None)
    same = tree_attention(q, kc, vc, pool, 1, table, lengths, torch.arange(-1, 5, dtype=torch.int32, device=DEV),
                          out_dtype=torch.float32)
    assert torch.equal(chain, same)
    prepared = tree_attention_from_prepared(*kc.prepare_queries(q), kc, vc, pool, 1, table, lengths)
    assert torch.equal(chain, prepared)


def test_sequences_that_do_not_run_and_pages_that_are_not_there():
    """Negative and overlong lengths give zeros; positions without a page are not attended."""
    lens = [70, -1, 100, 40]
    kc, vc, pool, table, lengths, q = _setup(128, 3, 4, 4, 2, 4, lens, 32, seed=6)
    lengths[2] = table.shape[1] * 32 - 3  # one position too many
    table[0, 1] = -1
    table[3, 0] = pool.num_pages + 7
    par = _tree(4, 4, 8, pads=False)
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)
    # nothing at all to attend: every page of a sequence gone
    table[3] = -1
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    assert (out[3] == 0).all()


def test_masked_rows_may_hold_anything():
    """Infinite and NaN norms in a node's row reach only the nodes that see it."""
    T = 6
    kc, vc, pool, table, lengths, q = _setup(128, 3, 1, 4, 1, T, [45], 32, seed=9)
    par = torch.tensor([[-1, 0, 0, 1, 2, 2]], dtype=torch.int32, device=DEV)
    clean = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    pos = 45 + 1  # node 1: seen by 1 and 3
    page, row = int(table[0, pos // 32]), pos % 32
    pl = pool.planes(1)
    for name, val in (("kvn", float("nan")), ("krn", float("inf")), ("vvn", float("nan")), ("vvn", float("inf"))):
        keep = pl[name][page, 0, row].clone()
        pl[name][page, 0, row] = val
        out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
        rest = [0, 2, 4, 5]
        # an infinite norm raises the common scale of the value weights: f16 weights at 2^-16 of it
        assert torch.isfinite(out[:, rest]).all(), name
        assert (out[:, rest] - clean[:, rest]).norm() <= 2.0 ** -8 * clean[:, rest].norm(), name
        assert not torch.isfinite(out[:, [1, 3]]).all(), name
        pl[name][page, 0, row] = keep
    # a node without a place is seen by nobody, whatever its row holds
    par[0, 5] = -2
    pos = 45 + 5
    for name in ("kvn", "krn", "vvn"):
        pl[name][int(table[0, pos // 32]), 0, pos % 32] = float("inf")
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    assert torch.equal(out[:, :5], clean[:, :5]) and (out[:, 5] == 0).all()


def test_a_query_of_nan_stays_its_own():
    kc, vc, pool, table, lengths, q = _setup(64, 3, 1, 4, 2, 3, [50], 32, seed=10)
    clean = tree_attention(q, kc, vc, pool, 1, table, lengths, out_dtype=torch.float32)
    q[0, 1, 1] = float("nan")
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, out_dtype=torch.float32)
    assert torch.isnan(out[0, 1, 1]).all()
    hurt = torch.isnan(out).any(-1)
    assert int(hurt.sum()) == 1 and torch.equal(out[~hurt], clean[~hurt])


@pytest.mark.parametrize("n,T,page", [(20000, 1, 64), (9001, 13, 128)])
def test_long_and_many_sequences(n, T, page):
    """Unequal lengths over more sequences than a wave has lanes."""
    print("case:", n, T, flush=True)
    lens = [n, 0, 777] + [5 + 3 * i for i in range(70)]
    kc, vc, pool, table, lengths, q = _setup(64, 3, len(lens), 2, 1, T, lens, page, seed=12)
    par = _tree(T, len(lens), 2)
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)


def _widen(table, width):
    """The table with empty entries up to `width` pages: room for long sequences, which two column tiles serve."""
    return torch.cat([table, torch.full((table.shape[0], width - table.shape[1]), -1, dtype=table.dtype, device=DEV)], 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [2, 3, 4])
@pytest.mark.parametrize("T,Hq,Hkv", [(9, 6, 3), (17, 2, 2), (16, 8, 2), (33, 3, 1)])
def test_two_column_tiles(D, bits, T, Hq, Hkv):
    """More than 16 columns under tables of 2^17 positions and more; a page in the middle is missing."""
    print("case:", D, bits, T, Hq, Hkv, flush=True)
    lens = [0, 31, 900, 1, 200]
    kc, vc, pool, table, lengths, q = _setup(D, bits, len(lens), Hq, Hkv, T, lens, 32, seed=T)
    table = _widen(table, 4096)
    table[2, 5] = pool.num_pages + 3
    par = _tree(T, len(lens), T)
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)


@pytest.mark.parametrize("bits", [2, 3, 4])
def test_many_parts_of_a_block(bits):
    """Stretches that cover several sequences, at each number of column tiles."""
    print("case:", bits, flush=True)
    lens = [3 + (37 * i) % 400 for i in range(300)]
    for T, Hq, Hkv in ((1, 2, 1), (1, 16, 16), (3, 6, 3), (6, 12, 3)):
        kc, vc, pool, table, lengths, q = _setup(64, bits, len(lens), Hq, Hkv, T, lens, 32, seed=21)
        if Hq // Hkv * T > 16:
            table = _widen(table, 512)
        par = _tree(T, len(lens), 4)
        out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
        some = torch.tensor([0, 1, 63, 64, 150, 298, 299], device=DEV)
        _check(out[some], kc, vc, pool, table[some], lengths[some], q[some], par[some])


@pytest.mark.parametrize("T,Hq,Hkv,wide", [(1, 4, 1, 0), (4, 6, 2, 0), (12, 6, 2, 0), (12, 6, 2, 4096)])
def test_a_query_that_is_not_finite_spoils_itself_only(T, Hq, Hkv, wide):
    print("case:", T, Hq, Hkv, wide, flush=True)
    kc, vc, pool, table, lengths, q = _setup(128, 3, 2, Hq, Hkv, T, [400, 37], 32, seed=15)
    if wide:
        table = _widen(table, wide)
    q_rot, q_proj = kc.prepare_queries(q)
    clean = tree_attention_from_prepared(q_rot, q_proj, kc, vc, pool, 1, table, lengths)
    for bad in (float("inf"), float("nan")):
        r, p = q_rot.clone(), q_proj.clone()
        r[0, 1, T - 1, ::2] = bad
        r[0, 1, T - 1, 1::2] = -bad
        p[0, 1, T - 1] = bad
        out = tree_attention_from_prepared(r, p, kc, vc, pool, 1, table, lengths)
        hurt = torch.zeros(out.shape[:3], dtype=torch.bool, device=DEV)
        hurt[0, T - 1, 1] = True
        assert torch.isnan(out[hurt]).all()
        # the others' queries may be scaled by another power of two, which rounds their low parts only
        assert (out[~hurt] - clean[~hurt]).norm() <= 2.0 ** -16 * clean[~hurt].norm()


def test_agrees_with_the_cache_of_one_length():
    """A chain over pages against compressed_attention over contiguous planes of the same rows."""
    from turboquant_pytorch import compressed_attention

    kc, vc, pool, table, lengths, q = _setup(128, 3, 2, 8, 2, 4, [300, 300], 64, seed=13)
    ck, cv = pool.read(1, table, lengths + 4, 304)
    a = compressed_attention(q, kc, vc, ck, cv, causal=True, out_dtype=torch.float32)
    b = tree_attention(q, kc, vc, pool, 1, table, lengths, out_dtype=torch.float32)
    # both sides round P and the value centroids to f16: 2 (2^-10) of the row's weighted norms, which
    # for these random values are below 8 times the norm of their mean
    assert (a - b).norm() <= 16 * 2.0 ** -10 * a.norm()


def test_graph_replays_with_other_lengths():
    """Captured once; lengths, trees and tables change between the replays, eager work in between."""
    T = 5
    kc, vc, pool, table, lengths, q = _setup(64, 3, 3, 4, 2, T, [300, 200, 100], 32, seed=14)
    par = _tree(T, 3, 1, pads=False)
    args = (q, kc, vc, pool, 1, table, lengths, par)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_attention(*args)
    for rep, lens in enumerate([[300, 200, 100], [1, 0, 99], [-1, 150, 33], [300, -1, 2]]):
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        par.copy_(_tree(T, 3, rep + 20, pads=rep == 2))
        q.normal_()
        torch.cuda.synchronize()
        want = tree_attention(*args).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep


def test_another_stream():
    kc, vc, pool, table, lengths, q = _setup(128, 3, 2, 8, 2, 3, [600, 90], 64, seed=15)
    want = tree_attention(q, kc, vc, pool, 1, table, lengths)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s in (s1, s2, s1, s2):
        with torch.cuda.stream(s):
            got.append(tree_attention(q, kc, vc, pool, 1, table, lengths))
    torch.cuda.synchronize()
    for o in got:
        assert torch.equal(o, want)


@pytest.mark.parametrize("bits", [2, 3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hq,Hkv", [(2, 4, 2), (2, 2, 2), (3, 2, 2), (4, 3, 3)])
def test_few_drafted_tokens_per_head(D, bits, T, Hq, Hkv):
    """Up to 4 columns per kv head from several nodes: speculation with few query heads per kv head."""
    print("case:", D, bits, T, Hq, Hkv, flush=True)
    lens = [0, 31, 500, 1, 64]
    kc, vc, pool, table, lengths, q = _setup(D, bits, len(lens), Hq, Hkv, T, lens, 32, seed=30 + T)
    for par in (None, _tree(T, len(lens), T), torch.tensor([-1] + [0] * (T - 1), dtype=torch.int32, device=DEV)):
        out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
        _check(out, kc, vc, pool, table, lengths, q, par)


# planes, one column tile, two column tiles
FORMS = [(1, 4, 2, 0), (4, 2, 2, 0), (5, 4, 2, 0), (16, 4, 2, 4096)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,Hq,Hkv,wide", FORMS)
def test_large_norms_of_keys_that_weigh_nothing(D, T, Hq, Hkv, wide):
    """Every slab of 32 keys holds a key of weight 1 and value norm 2^-6, one of weight e^-100 and norm 6e4,
    and 30 of weight 2^-15.2 and norm 1, whose values point one way: 5% of the row's weighted norms.  Each of those
    contributions is 2^-9 of the largest one, far above the 2^-30 that the bound leaves out."""
    print("case:", D, T, Hq, Hkv, wide, flush=True)
    n = 4096
    kc, vc, pool, table, lengths, q = _setup(D, 3, 1, Hq, Hkv, T, [n], 32, seed=40)
    if wide:
        table = _widen(table, wide)
    G = Hq // Hkv
    q = q[:, ::G, :1].repeat_interleave(G, 1).expand(1, Hq, T, D).contiguous()  # a kv head's columns are alike
    q_rot = kc.prepare_queries(q)[0][0, ::G, 0].double()  # [Hkv, D]
    top = float(kc.centroids.half().max())
    codes = torch.where(q_rot < 0, 3, 0).to(torch.uint8)  # <q_rot, C[codes]> = -top sum |q_rot| (symmetric codebook)
    unit = top * q_rot.abs().sum(-1) / math.sqrt(D)  # minus a score, per unit of key norm
    pl = pool.planes(1)
    pl["krn"].zero_()
    pl["kvn"].copy_((15.2 * math.log(2) / unit)[None, :, None].expand(pl["kvn"].shape))
    pl["kvn"][:, :, 3] = 0
    pl["kvn"][:, :, 7] = (100 / unit)[None].half()
    pl["vvn"].fill_(1)
    pl["vvn"][:, :, 3] = 2.0 ** -6
    pl["vvn"][:, :, 7] = 6e4
    packed = torch.from_numpy(O.pack_bits(codes.cpu().numpy(), 2)).to(DEV)
    pl["kcodes"].copy_(packed[None, :, None].expand(pl["kcodes"].shape))
    pl["vcodes"].fill_(255)
    pl["vcodes"][:, :, 3] = 0
    par = _tree(T, 1, 3, pads=False)
    out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    _check(out, kc, vc, pool, table, lengths, q, par)


@pytest.mark.parametrize("T,Hq,Hkv,wide", [(4, 2, 2, 0), (6, 4, 2, 0), (16, 4, 2, 4096)])
def test_norms_of_a_row_do_not_reach_the_nodes_that_do_not_see_it(T, Hq, Hkv, wide):
    """Bit for bit: a sibling's value norm, however large, changes nothing for the other branches."""
    print("case:", T, Hq, Hkv, wide, flush=True)
    kc, vc, pool, table, lengths, q = _setup(128, 3, 1, Hq, Hkv, T, [45], 32, seed=41)
    if wide:
        table = _widen(table, wide)
    par = torch.tensor([[-1, 0, 0, 1] + [2] * (T - 4)], dtype=torch.int32, device=DEV)
    clean = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
    rest = [i for i in range(T) if i not in (1, 3)]
    pos = 45 + 1  # node 1: seen by 1 and 3
    row = pool.planes(1)["vvn"][int(table[0, pos // 32]), :, pos % 32]
    for val in (6e4, 100.0, float("inf"), float("nan"), 0.0):
        row.fill_(val)
        out = tree_attention(q, kc, vc, pool, 1, table, lengths, par, out_dtype=torch.float32)
        assert torch.equal(out[:, rest], clean[:, rest]), val
        if math.isfinite(val):
            _check(out, kc, vc, pool, table, lengths, q, par)
