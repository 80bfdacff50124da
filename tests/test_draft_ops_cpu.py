"""Argument checks of the page, tree-attention and verification operators, on the CPU.

Meta tensors drive the checks that each operator shares with its Meta kernel; the C entry points
refuse before any launch.  No GPU is touched.
"""

import ctypes

import pytest
import torch

from turboquant_pytorch import PagePool, _native, tree_attention, verify_drafts
from turboquant_pytorch._ops import ops

M = "meta"
L, N, H, P, D, BITS, B, W, T, S, V = 3, 9, 2, 64, 128, 3, 4, 5, 6, 70, 1000
F16, F32, U8, I32, I64 = torch.float16, torch.float32, torch.uint8, torch.int32, torch.int64


def _e(*shape, dtype=F32, device=M):
    return torch.empty(*shape, dtype=dtype, device=device)


def _planes(*lead):
    return dict(pk=_e(*lead, 32, dtype=U8), ps=_e(*lead, 16, dtype=U8), prn=_e(*lead, dtype=F16), pkn=_e(*lead, dtype=F16),
                pv=_e(*lead, 48, dtype=U8), pvn=_e(*lead, dtype=F16))


def _refuses(fn, args, bad, match):
    a = dict(args)
    a.update(bad)
    with pytest.raises(RuntimeError, match=match):
        fn(*a.values())


def _write_args():
    n = (B, H, S)
    return dict(kc=_e(*n, 32, dtype=U8), ks=_e(*n, 16, dtype=U8), rn=_e(*n, dtype=F16), kn=_e(*n, dtype=F16),
                vc=_e(*n, 48, dtype=U8), vn=_e(*n, dtype=F16), **_planes(N, H, P), table=_e(B, W, dtype=I32),
                start=_e(B, dtype=I32), S=S)


def _read_args():
    return dict(**_planes(N, H, P), table=_e(B, W, dtype=I32), lengths=_e(B, dtype=I32), S=S)


POOL = [
    (dict(pkn=_e(N, H, 48, dtype=F16)), "power of two"),
    (dict(pkn=_e(N, H, 16, dtype=F16)), "power of two"),
    (dict(pkn=_e(N, H, P)), "must be Half"),
    (dict(pk=_e(N, H, P, 31, dtype=U8)), "no codes of one head_dim"),
    (dict(pv=_e(N, H + 1, P, 48, dtype=U8)), "geometry"),
    (dict(pv=_e(N, H, P, 96, dtype=U8)[..., ::2]), "contiguous"),
    (dict(ps=_e(N, H, P, 16, dtype=torch.int8)), "must be Byte"),
    (dict(prn=_e(N, H, P // 2, dtype=F16)), "kernels read|geometry"),
    (dict(pvn=_e(N, H, P, dtype=F16, device="cpu")), "expected meta"),
    (dict(table=_e(B, W, dtype=I64)), "int32"),
    (dict(table=_e(B * W, dtype=I32)), "block_table must be"),
    (dict(table=_e(W, B, dtype=I32).t()), "contiguous"),
]


@pytest.mark.parametrize("bad,match", POOL + [
    (dict(start=_e(B + 1, dtype=I32)), "start must be"),
    (dict(kc=_e(B, H, S, 31, dtype=U8)), "rows must hold 32"),
    (dict(vn=_e(B, H, S + 1, dtype=F16)), "expected"),
    (dict(kn=_e(B, H, S - 1, dtype=F16)), "kernels read"),
    (dict(S=-1), "row count"),
])
def test_page_write_refuses(bad, match):
    ops().page_write(*_write_args().values())
    _refuses(ops().page_write, _write_args(), bad, match)


@pytest.mark.parametrize("bad,match", POOL + [(dict(lengths=_e(B, dtype=I64)), "int32")])
def test_page_read_refuses(bad, match):
    out = ops().page_read(*_read_args().values())
    assert [tuple(t.shape) for t in out] == [(B, H, S, 32), (B, H, S, 16), (B, H, S), (B, H, S), (B, H, S, 48), (B, H, S)]
    _refuses(ops().page_read, _read_args(), bad, match)


def test_page_copy_and_keep_check_every_layer():
    pl = _planes(L, N, H, P)
    idx = _e(7, dtype=I32)
    ops().page_copy(*pl.values(), idx, idx)
    for bad, match in ((dict(src=_e(7, dtype=I64)), "int32"), (dict(dst=_e(6, dtype=I32)), "dst must be"),
                       (dict(pkn=_e(N, H, P, dtype=F16)), "norm planes must be"),
                       (dict(pk=_e(L + 1, N, H, P, 32, dtype=U8)), "geometry")):
        _refuses(ops().page_copy, dict(pl, src=idx, dst=idx), bad, match)
    keep = dict(pl, table=_e(B, W, dtype=I32), lengths=_e(B, dtype=I32), path=_e(B, T, dtype=I32), count=_e(B, dtype=I32))
    out = ops().page_keep(*keep.values())
    assert out.shape == (B,) and out.dtype == I32
    for bad, match in ((dict(path=_e(B, 65, dtype=I32)), "1 to 64"), (dict(path=_e(B, T, dtype=I64)), "int32"),
                       (dict(count=_e(B - 1, dtype=I32)), "count must be"), (dict(lengths=_e(1, dtype=I32)), "lengths must be")):
        _refuses(ops().page_keep, keep, bad, match)


def _tree_args(raw):
    q = dict(q=_e(B, 8, T, D, dtype=torch.bfloat16), pi=_e(2, D, D, dtype=F16), se=_e(D, D, dtype=F16)) if raw else \
        dict(q=_e(B, 8, T, D, dtype=F16), qp=_e(B, 8, T, D))
    p = _planes(N, H, P)
    return dict(**q, pk=p["pk"], ps=p["ps"], prn=p["prn"], pkn=p["pkn"], kcent=_e(4, dtype=F16), bits=BITS, pv=p["pv"],
                pvn=p["pvn"], vcent=_e(8), vpit=_e(2, D, D, dtype=F16), table=_e(B, W, dtype=I32),
                lengths=_e(B, dtype=I32), parents=None, coeff=0.01, scale=0.09, out=torch.bfloat16)


@pytest.mark.parametrize("raw", [True, False])
@pytest.mark.parametrize("bad,match", POOL + [
    (dict(bits=4), "the pool holds"),
    (dict(bits=5), "the pool holds"),
    (dict(kcent=_e(3, dtype=F16)), "key centroids"),
    (dict(vcent=_e(8, dtype=F16)), "must be Float"),
    (dict(vpit=_e(D, D, dtype=F16)), "Pi_v"),
    (dict(table=_e(B + 1, W, dtype=I32)), "block_table has"),
    (dict(table=_e(B, 0, dtype=I32)), "must hold"),
    (dict(lengths=_e(B, 1, dtype=I32)), "lengths must be"),
    (dict(parents=_e(T + 1, dtype=I32)), "parents must be"),
    (dict(parents=_e(B, T, dtype=I64)), "int32"),
    (dict(parents=_e(1, T, dtype=I32)), "parents must be"),
    (dict(out=torch.int32), "out_dtype"),
])
def test_tree_attention_refuses(raw, bad, match):
    fn = ops().tree_attend if raw else ops().tree_attention
    for par in (None, _e(T, dtype=I32), _e(B, T, dtype=I32)):
        out = fn(*dict(_tree_args(raw), parents=par).values())
        assert out.shape == (B, T, 8, D) and out.dtype == torch.bfloat16
    _refuses(fn, _tree_args(raw), bad, match)


@pytest.mark.parametrize("shape,match", [((B, 8, 65, D), "1 to 64"), ((B, 8, 0, D), "1 to 64"), ((B, 7, T, D), "multiple"),
                                         ((B, 8, T, 64), "the pool holds"), ((B, 8, T, 96), "head_dim 96"),
                                         ((8, T, D), "must be \\[B, Hq, T, D\\]")])
def test_tree_attention_refuses_queries(shape, match):
    _refuses(ops().tree_attend, _tree_args(True), dict(q=_e(*shape)), match)


def test_tree_attention_python_checks():
    from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2

    pool = PagePool(N, P, H, D, 3, device=M)
    kc, vc = TurboQuantCompressorV2(D, 3, 1), TurboQuantCompressorMSE(D, 4, 2)
    with pytest.raises(ValueError, match="one bit width"):
        tree_attention(_e(B, 8, T, D), kc, vc, pool, 0, _e(B, W, dtype=I32), _e(B, dtype=I32))


def _verify_args():
    return dict(tokens=_e(B, T, dtype=I64), p=_e(B, T, V), u=_e(B, T), parents=None, draft=None)


@pytest.mark.parametrize("bad,match", [
    (dict(tokens=_e(B, T, dtype=I32)), "int64"),
    (dict(tokens=_e(T, B, dtype=I64).t()), "contiguous"),
    (dict(tokens=_e(B, T - 1, dtype=I64)), "tokens must be"),
    (dict(p=_e(B, T, V, dtype=torch.float64)), "target_probs must be"),
    (dict(p=_e(B, V, T).transpose(1, 2)), "contiguous along"),
    (dict(p=_e(B * T, V)), "target_probs must be"),
    (dict(u=_e(B, T, dtype=torch.float64)), "uniforms"),
    (dict(u=_e(B, T - 1)), "uniforms"),
    (dict(u=_e(B, T, device="cpu")), "expected meta"),
    (dict(parents=_e(B, T - 1, dtype=I32)), "parents must be"),
    (dict(parents=_e(T, dtype=I64)), "int32"),
    (dict(draft=_e(B, T, V)), "draft_probs must be"),
    (dict(draft=_e(B, T - 1, V, dtype=F16)), "draft_probs must be"),
    (dict(parents=_e(T, dtype=I32), draft=_e(B, T - 1, V)), "chain"),
])
def test_verify_refuses(bad, match):
    for par, draft in ((None, None), (_e(T, dtype=I32), None), (_e(B, T, dtype=I32), None), (None, _e(B, T - 1, V))):
        path, count, nxt = verify_drafts(_e(B, T, dtype=I64), _e(B, T, V), _e(B, T), par, draft)
        assert (path.shape, path.dtype, count.shape, count.dtype, nxt.shape, nxt.dtype) == ((B, T), I32, (B,), I32, (B,), I64)
    _refuses(ops().verify_drafts, _verify_args(), bad, match)
    with pytest.raises(RuntimeError, match="1 to 64"):
        verify_drafts(_e(B, 65, dtype=I64), _e(B, 65, V), _e(B, 65))


def test_no_cpu_path():
    with pytest.raises((RuntimeError, NotImplementedError)):
        verify_drafts(torch.zeros(1, 1, dtype=I64), torch.ones(1, 1, 4), torch.zeros(1, 1))


def test_pool_geometry():
    pool = PagePool(N, P, H, 80, 4, layers=L, device="cpu")
    assert (pool.layers, pool.num_pages, pool.num_kv_heads, pool.page_size, pool.head_dim, pool.bits) == (L, N, H, P, 80, 4)
    assert {n: tuple(t.shape) for n, t in pool.planes(1).items()} == {
        "kcodes": (N, H, P, 30), "ksigns": (N, H, P, 10), "krn": (N, H, P), "kvn": (N, H, P), "vcodes": (N, H, P, 40),
        "vvn": (N, H, P)}
    assert pool.nbytes() == L * N * H * P * (30 + 10 + 4 + 40 + 2)
    again = PagePool.over(*pool._planes)
    assert (again.layers, again.bits, again.head_dim) == (L, 4, 80)
    for bad in (dict(page_size=48), dict(page_size=16), dict(bits=1), dict(head_dim=100), dict(num_pages=0)):
        with pytest.raises(ValueError):
            PagePool(**{**dict(num_pages=N, page_size=P, num_kv_heads=H, head_dim=D, bits=3, device="cpu"), **bad})
    ck = {"packed_key_indices": None, "shape": (B, H + 1, S, 80)}
    with pytest.raises(ValueError, match="do not go into"):
        pool.write(0, ck, {"packed_indices": None, "shape": (B, H + 1, S, 80)}, _e(B, W, dtype=I32), _e(B, dtype=I32))
    with pytest.raises(ValueError, match="packed"):
        pool.write(0, {}, {}, _e(B, W, dtype=I32), _e(B, dtype=I32))


def test_c_entries_refuse():
    lib = _native.lib()
    six = (ctypes.c_void_p * 6)(*[16 * (i + 1) for i in range(6)])
    none = None
    rows = lambda **k: [six, six, 1, H, 4, k.get("d", 64), 2, k.get("vb", 3), 5, k.get("P", 64), 16, 2, k.get("W", 2), 16, none]  # noqa: E731
    for fn in (lib.tq_page_write, lib.tq_page_read):
        for kw, msg in ((dict(d=100), b"head_dim 100"), (dict(P=48), b"power of two"), (dict(P=16), b"power of two"),
                        (dict(vb=9), b"bits"), (dict(W=3), b"bad shape")):
            assert fn(*rows(**kw)) == -1 and msg in lib.tq_last_error()
        assert fn(none, none, 1, H, 4, 64, 2, 3, 5, 64, none, 0, 0, none, none) == -1
        assert fn(none, none, 0, H, 4, 64, 2, 3, 5, 64, none, 0, 0, none, none) == 0  # nothing to do
    odd = (ctypes.c_void_p * 6)(*[16 * (i + 1) + 8 for i in range(6)])
    assert lib.tq_page_copy(odd, 1, H, 64, 2, 3, 5, 64, 16, 16, 1, none) == -1 and b"16-byte" in lib.tq_last_error()
    assert lib.tq_page_copy(none, 1, H, 64, 2, 3, 5, 64, none, none, 0, none) == 0
    assert lib.tq_page_keep(six, 1, 1, H, 65, 64, 2, 3, 5, 64, 16, 2, 2, 16, 16, 16, 16, none) == -1
    assert b"at most 64" in lib.tq_last_error()
    tree = lambda T=2, d=64, bits=3, P=64, W=2: lib.tq_tree_attention(  # noqa: E731
        *[16] * 7, bits, *[16] * 4, 5, P, 16, W, W, 16, none, 0, 1, 4, 2, T, d, 0.1, 0.1, 16, 0, 0, 0, 0, none, 0, none)
    assert tree(d=96) == -2 and tree(bits=5) == -2
    assert tree(T=65) == -1 and tree(P=16) == -1 and tree(W=0) == -1 and tree(W=1 << 20) == -1
    assert lib.tq_tree_workspace_size(1, 4, 2, 65, 2, 64, 64, 3) == 0
    assert lib.tq_verify_drafts(none, none, 0, 0, 0, none, 0, 0, none, none, 0, 1, 65, 10, none, none, none, none, 0, none) == -1
    assert lib.tq_verify_drafts(16, 16, 0, 0, 0, 16, 0, 0, 16, 16, 0, 1, 2, 10, 16, 16, 16, 16, 99, none) == -1
    assert b"chain" in lib.tq_last_error()
    assert lib.tq_verify_drafts(16, 16, 0, 0, 0, none, 0, 0, 16, 16, 0, 1, 2, 10, 16, 16, 16, 16, 1, none) == -1
    assert b"workspace" in lib.tq_last_error()


def _append_args():
    t = dict(_tree_args(True))
    head = dict(k=_e(B, H, T, D, dtype=torch.bfloat16), v=_e(B, H, T, D, dtype=torch.bfloat16), q=t.pop("q"),
                pi=t.pop("pi"), ks=_e(2, D, D, dtype=F16), kc=_e(4), kb=_e(3), vpi=_e(2, D, D, dtype=F16), vb=_e(7),
                se=t.pop("se"))
    return {**head, **t}


@pytest.mark.parametrize("bad,match", POOL + [
    (dict(k=_e(B, H, T + 1, D)), "k and v must be"),
    (dict(v=_e(B, H, T, D // 2)), "k and v must be"),
    (dict(k=_e(B, H + 1, T, D), v=_e(B, H + 1, T, D)), "k and v must be"),
    (dict(ks=_e(D, D, dtype=F16)), "key split S_eff"),
    (dict(kc=_e(3)), "key centroids"),
    (dict(kb=_e(2)), "key boundaries"),
    (dict(vpi=_e(2, D, D)), "value split Pi"),
    (dict(vb=_e(6)), "value boundaries"),
    (dict(se=_e(2, D, dtype=F16)), "f16 S_eff"),
    (dict(q=_e(B, 8, 65, D)), "1 to 64"),
    (dict(bits=4), "the pool holds"),
    (dict(parents=_e(T + 1, dtype=I32)), "parents must be"),
    (dict(lengths=_e(B + 1, dtype=I32)), "lengths must be"),
    (dict(out=torch.int32), "out_dtype"),
])
def test_page_attend_refuses(bad, match):
    out = ops().page_attend(*_append_args().values())
    assert out.shape == (B, T, 8, D) and out.dtype == torch.bfloat16
    _refuses(ops().page_attend, _append_args(), bad, match)


def test_page_append_c_entry_refuses():
    lib = _native.lib()
    six = (ctypes.c_void_p * 6)(*[16 * (i + 1) for i in range(6)])
    odd = (ctypes.c_void_p * 6)(*[16 * (i + 1) + 4 for i in range(6)])
    none = None

    def call(pool=six, dt=0, B=1, H=2, S=3, d=64, bits=3, n=5, P=64, W=2, k=16, q=16, qr=16):
        return lib.tq_page_append(k, 16, dt, B, H, S, d, *[0] * 6, *[16] * 6, bits, pool, n, P, 16, W, W, 16, q, 4, 0, 0, 0,
                                  16, qr, 16, none)

    assert call(d=96) == -2 and call(bits=5) == -2 and call(bits=1) == -2
    for kw, msg in ((dict(dt=7), b"dtype"), (dict(P=48), b"power of two"), (dict(P=16), b"power of two"), (dict(n=0), b"bad pool"),
                    (dict(S=-1), b"bad shape"), (dict(H=0), b"bad shape"), (dict(k=none), b"null"), (dict(pool=odd), b"16-byte"),
                    (dict(qr=4), b"q_rot"), (dict(B=1 << 20, H=1 << 10, S=64), b"2^31")):
        assert call(**kw) == -1 and msg in lib.tq_last_error(), kw
    assert call(B=0, k=none) == 0 and call(S=0, k=none) == 0


def test_more_sequences_than_a_grid_takes_are_refused_before_a_row_is_written():
    n = 65536
    big = dict(table=_e(n, W, dtype=I32), lengths=_e(n, dtype=I32))
    for args, fn in ((_append_args(), ops().page_attend), (_tree_args(True), ops().tree_attend)):
        new = {k: _e(n, *args[k].shape[1:], dtype=args[k].dtype) for k in ("k", "v", "q") if k in args}
        _refuses(fn, args, {**new, **big}, "at most 65535 sequences")
